"""The recurrence and the rotary positions without a GPU: what their entry points refuse, the table, and the oracle against closed forms."""
import ctypes as C
import math
import os

import pytest
import torch

from oracle import sequence_ref as R


@pytest.fixture(scope="module")
def lib():
    from dest3d_amd import _lib as L
    if not os.path.exists(L.LIB_PATH):
        from dest3d_amd.build import build
        build(verbose=False)
    return L.load()


FAKE = 0x1000   # (an address that nothing reads: all of these calls are refused before a launch)


def test_no_cpu_path(lib):
    from dest3d_amd import gated_scan, gated_scan_step, qk_norm_rotary, rotary, rotary_table
    x, A = torch.zeros(1, 4, 8), torch.full((8,), -1.0)
    q, w, tab = torch.zeros(1, 4, 2, 8), torch.ones(8), rotary_table(4, 8, device="cpu")
    for call in (lambda: gated_scan(x, x, A), lambda: gated_scan_step(x[0], x[0], A, torch.zeros(4, 8)), lambda: rotary(q, None, tab),
                 lambda: qk_norm_rotary(q, None, w, None, tab)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()
    with pytest.raises(ValueError):
        qk_norm_rotary(q, q, w, None, tab)
    with pytest.raises(ValueError):
        qk_norm_rotary(q, None, None, None, tab)


def _scan(lib, **kw):
    from dest3d_amd import _lib as L
    a = L.GatedScanArgs()
    a.batch, a.seqlen, a.channels, a.x, a.gate, a.A, a.y = 2, 100, 8, FAKE, FAKE, FAKE, FAKE
    for k, v in kw.items():
        if isinstance(v, tuple):
            for i, e in enumerate(v):
                getattr(a, k)[i] = e
        else:
            setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,code,text", [
    (dict(batch=0), -2, "batch=0"), (dict(seqlen=-1), -2, "seqlen=-1"), (dict(channels=0), -2, "channels=0"), (dict(seqlen=2 ** 31 - 1), -2, ""),
    (dict(batch=2 ** 30, seqlen=2 ** 30), -2, "too many"), (dict(batch=2 ** 22, seqlen=1), -2, "too many"), (dict(dtype=2), -4, "dtype"), (dict(flags=8), -5, "flags"), (dict(x=None), -1, ""), (dict(gate=None), -1, ""),
    (dict(A=None), -1, ""), (dict(y=None), -1, "y is NULL"), (dict(x_stride=(-1, 8)), -3, "stride"), (dict(gate_stride=(0, -8)), -3, "stride"),
    (dict(in_gate=FAKE, in_gate_stride=(-8, 8)), -3, "stride"), (dict(seq_idx=FAKE, seq_idx_stride=(4, -1)), -3, "stride")])
def test_scan_refuses(lib, kw, code, text):
    a = _scan(lib, **kw)
    assert lib.issm_gated_scan_fwd(C.byref(a)) == code and text in lib.issm_last_error().decode()


def test_scan_backward_refuses(lib):
    a = _scan(lib)
    assert lib.issm_gated_scan_bwd(C.byref(a)) == -1 and b"saved" in lib.issm_last_error()
    a.saved, a.din_gate = FAKE, FAKE
    assert lib.issm_gated_scan_bwd(C.byref(a)) == -1 and b"in_gate" in lib.issm_last_error()
    a.din_gate, a.dA = None, FAKE
    assert lib.issm_gated_scan_bwd(C.byref(a)) == -6
    need = C.c_size_t()
    assert lib.issm_gated_scan_workspace_bytes(C.byref(a), 1, C.byref(need)) == 0 and need.value >= 2 * 8 * 4
    a.workspace, a.workspace_bytes = FAKE, need.value - 1
    assert lib.issm_gated_scan_bwd(C.byref(a)) == -6
    assert lib.issm_gated_scan_saved_bytes(C.byref(a), C.byref(need)) == 0 and need.value % (2 * 8 * 4) == 0
    for f in (lib.issm_gated_scan_fwd, lib.issm_gated_scan_bwd, lib.issm_gated_scan_step, lib.issm_rotary, lib.issm_rotary_norm_fwd, lib.issm_rotary_norm_bwd):
        assert f(None) == -1


@pytest.mark.parametrize("kw,code", [
    (dict(rows=0), -2), (dict(channels=0), -2), (dict(slots=0), -2), (dict(slots=1), -2), (dict(dtype=3), -4), (dict(flags=2), -5), (dict(state=None), -1),
    (dict(y=None), -1), (dict(state_stride=7), -3), (dict(x_stride=-1), -3), (dict(rows=2 ** 23, slots=2 ** 23), -2)])
def test_step_refuses(lib, kw, code):
    from dest3d_amd import _lib as L
    a = L.GatedScanStepArgs()
    a.rows, a.channels, a.slots, a.x, a.gate, a.A, a.state, a.y, a.state_stride = 2, 8, 4, FAKE, FAKE, FAKE, FAKE, FAKE, 8
    for k, v in kw.items():
        setattr(a, k, v)
    assert lib.issm_gated_scan_step(C.byref(a)) == code


@pytest.mark.parametrize("kw,code", [
    (dict(batch=0), -2), (dict(seqlen=0), -2), (dict(headdim=0), -2), (dict(heads=(0, 0)), -2), (dict(heads=(-1, 2)), -2), (dict(rot=0), -2), (dict(rot=7), -2),
    (dict(rot=10), -2), (dict(headdim=1026), -5), (dict(batch=2 ** 16, seqlen=2 ** 15), -2), (dict(heads=(2 ** 19, 0), batch=64, seqlen=64), -2), (dict(dtype=2), -4),
    (dict(weight_dtype=-1), -4), (dict(flags=4), -5), (dict(x=(None, None)), -1), (dict(y=(None, None)), -1), (dict(table=None), -1), (dict(table_rows=0), -2),
    (dict(table_rows=4), -2), (dict(positions=FAKE, positions_stride=(-1, 1)), -3)])
def test_rotary_refuses(lib, kw, code):
    from dest3d_amd import _lib as L
    a = L.RotaryArgs()
    a.batch, a.seqlen, a.headdim, a.rot, a.table, a.table_rows = 1, 5, 8, 8, FAKE, 5
    a.heads[0], a.x[0], a.y[0], a.w[0] = 2, FAKE, FAKE, FAKE
    for k, v in kw.items():
        if isinstance(v, tuple):
            for i, e in enumerate(v):
                getattr(a, k)[i] = e
        else:
            setattr(a, k, v)
    assert lib.issm_rotary(C.byref(a)) == code and lib.issm_rotary_norm_fwd(C.byref(a)) == code
    if code in (-2, -4, -5):
        need = C.c_size_t()
        assert kw.get("table_rows") is not None or lib.issm_rotary_norm_bwd_bytes(C.byref(a), C.byref(need)) == code


def test_rotary_backward_refuses(lib):
    from dest3d_amd import _lib as L
    a = L.RotaryArgs()
    a.batch, a.seqlen, a.headdim, a.rot, a.table, a.table_rows = 1, 5, 8, 8, FAKE, 5
    a.heads[0], a.x[0], a.dx[0], a.w[0] = 2, FAKE, FAKE, FAKE
    assert lib.issm_rotary_norm_bwd(C.byref(a)) == -1 and b"dy" in lib.issm_last_error()
    a.dy[0] = FAKE
    assert lib.issm_rotary_norm_bwd(C.byref(a)) == -6
    a.flags = 2
    assert lib.issm_rotary_norm_bwd(C.byref(a)) == -5 and lib.issm_rotary_norm_fwd(C.byref(a)) in (-1, -5)


def test_table():
    from dest3d_amd import rotary_table
    t = rotary_table(100, 8, base=100.0, device="cpu")
    assert t.shape == (100, 8) and t.dtype == torch.float32
    for p, j in ((0, 0), (7, 1), (99, 3)):
        a = p * 100.0 ** (-2 * j / 8)
        assert abs(t[p, j].item() - math.cos(a)) <= 2 ** -24 and abs(t[p, 4 + j].item() - math.sin(a)) <= 2 ** -24
    # far positions: the angle in 64 bits, so that the sine is right to fp32's last place
    far = rotary_table(300001, 2, device="cpu")[300000]
    assert abs(far[0].item() - math.cos(300000.0)) <= 2 ** -24 and abs(far[1].item() - math.sin(300000.0)) <= 2 ** -24
    angle = lambda t: torch.atan2(t[1, t.shape[1] // 2:].double(), t[1, :t.shape[1] // 2].double())  # noqa: E731
    plain = angle(rotary_table(2, 64, device="cpu"))
    torch.testing.assert_close(angle(rotary_table(2, 64, scaling="linear", factor=4.0, device="cpu")), plain / 4, rtol=1e-5, atol=1e-7)
    base = angle(rotary_table(2, 64, scaling="base", factor=4.0, device="cpu"))
    assert abs(base[0] - plain[0]) < 1e-6 and abs(base[-1] / plain[-1] - 0.25) < 1e-5 and (base <= plain + 1e-7).all()
    parts = rotary_table(2, 64, scaling="parts", factor=4.0, original_length=4096, device="cpu")
    size = 0.1 * math.log(4.0) + 1.0
    torch.testing.assert_close((parts[1, :32].double() ** 2 + parts[1, 32:].double() ** 2).sqrt(), torch.full((32,), size).double(), rtol=1e-6, atol=0)
    ratio = angle(parts) / plain
    turns = 4096 * plain / (2 * math.pi)
    assert (ratio[turns > 40] - 1).abs().max() < 1e-5 and (ratio[turns < 0.7] - 0.25).abs().max() < 1e-4 and (ratio.diff() <= 1e-5).all()
    assert torch.equal(rotary_table(9, 6, scaling="parts", factor=1.0, original_length=9, device="cpu"), rotary_table(9, 6, device="cpu"))
    for kw in (dict(length=0, dim=4), dict(length=4, dim=3), dict(length=4, dim=0), dict(length=4, dim=4, base=1.0), dict(length=4, dim=4, factor=0.5),
               dict(length=4, dim=4, scaling="other"), dict(length=4, dim=4, scaling="parts"), dict(length=4, dim=4, scaling="parts", original_length=9, beta_slow=64.0)):
        with pytest.raises(ValueError):
            rotary_table(device="cpu", **kw)


def test_oracle():
    """Constant gates: a geometric sum; and a rotation as a product of complex numbers."""
    L, A = 30, torch.tensor([-0.7], dtype=torch.float64)
    x, gate = torch.ones(1, L, 1, dtype=torch.float64), torch.full((1, L, 1), 0.3, dtype=torch.float64)
    y, last = R.gated_scan(x, gate, A, initial_states=torch.full((1, 1), 2.0, dtype=torch.float64))
    a = torch.exp(A * torch.sigmoid(torch.tensor(0.3, dtype=torch.float64)))
    t = torch.arange(1, L + 1)
    want = 2 * a ** t + torch.sqrt(1 - a * a) * (1 - a ** t) / (1 - a)
    torch.testing.assert_close(y[0, :, 0], want, rtol=1e-12, atol=0)
    assert last == y[0, -1]
    back, first = R.gated_scan(x, gate, A, initial_states=torch.full((1, 1), 2.0, dtype=torch.float64), reverse=True)
    assert torch.equal(back.flip(1), y) and first == last
    ids = torch.tensor([[0] * 10 + [1] * 20])
    cut, _ = R.gated_scan(x, gate, A, seq_idx=ids)
    alone, _ = R.gated_scan(x[:, 10:], gate[:, 10:], A)
    assert torch.equal(cut[:, 10:], alone)
    v = torch.randn(1, 5, 2, 6, dtype=torch.float64)
    angle = torch.rand(5, 3, dtype=torch.float64)
    tab = torch.cat([angle.cos(), angle.sin()], 1)
    for inter in (False, True):
        w = R.rotary(v, tab, interleaved=inter)
        one, two = (slice(0, 6, 2), slice(1, 6, 2)) if inter else (slice(0, 3), slice(3, 6))
        z = torch.complex(v[..., one], v[..., two]) * torch.polar(torch.ones_like(angle), angle)[None, :, None]
        torch.testing.assert_close(torch.complex(w[..., one], w[..., two]), z)


@pytest.mark.parametrize("batch,seqlen,channels", [(8192, 1, 4096), (65535, 1, 4032), (600, 4096, 64), (513, 100000, 7), (3, 100, 64), (1, 1, 1)])
def test_workspace_of_walked_rows(lib, batch, seqlen, channels):
    """Rows that a workgroup walks ask for nothing forward, and backward for a row of dA's sums each; shared ones for less than the data."""
    a, need = _scan(lib, batch=batch, seqlen=seqlen, channels=channels), C.c_size_t()
    assert lib.issm_gated_scan_workspace_bytes(C.byref(a), 0, C.byref(need)) == 0 and need.value == 0
    assert lib.issm_gated_scan_workspace_bytes(C.byref(a), 1, C.byref(need)) == 0
    if (batch, seqlen) != (3, 100):   # (one tile forward, two backward: shared)
        assert batch * channels * 4 <= need.value < batch * channels * 4 + 256


@pytest.mark.parametrize("batch,seqlen,channels", [(1, 131072, 2048), (8, 4096, 2048), (2, 1000, 288), (511, 113, 64)])
def test_workspace_of_shared_rows(lib, batch, seqlen, channels):
    """8 bytes a channel for 112 tokens, backward for 56, and there 4 for dA's sums; beside them what five tiles take, and the tickets."""
    a, need, size = _scan(lib, batch=batch, seqlen=seqlen, channels=channels), C.c_size_t(), batch * seqlen * channels
    rows = batch * -(-channels // 64)
    for back, share in ((0, 8 / 112), (1, 12 / 56)):
        assert lib.issm_gated_scan_workspace_bytes(C.byref(a), back, C.byref(need)) == 0
        assert 0 < need.value < share * size * 1.15 + rows * (128 + 5 * 512 + 256)   # (288 channels take the words of 320)


def test_documented_sizes(lib):
    """The last sizes that the header allows, and the first ones behind them."""
    from dest3d_amd import _lib as L
    need = C.c_size_t()
    for sizes, ok in ((dict(batch=2 ** 16 - 1, seqlen=1, channels=4096), True), (dict(batch=2 ** 16, seqlen=1, channels=4096), False),
                      (dict(batch=2 ** 22 - 1, seqlen=4 * 28, channels=1), True), (dict(batch=2 ** 22 - 1, seqlen=4 * 28 + 1, channels=1), False),
                      (dict(batch=1, seqlen=2 ** 24 * 28 - 28, channels=64), True), (dict(batch=1, seqlen=2 ** 24 * 28 - 27, channels=64), False),
                      (dict(batch=1, seqlen=28, channels=64 * (2 ** 22 - 1)), True), (dict(batch=1, seqlen=28, channels=64 * (2 ** 22 - 1) + 1), False)):
        rc = lib.issm_gated_scan_workspace_bytes(C.byref(_scan(lib, **sizes)), 1, C.byref(need))
        assert rc == (0 if ok else -2), sizes
    a = L.RotaryArgs()
    a.headdim, a.rot, a.heads[0], a.heads[1] = 64, 64, 3, 1
    for batch, seqlen, ok in ((1, 2 ** 29 - 1, True), (1, 2 ** 29, False), (2 ** 15, 2 ** 14, False)):
        a.batch, a.seqlen = batch, seqlen
        assert lib.issm_rotary_norm_bwd_bytes(C.byref(a), C.byref(need)) == (0 if ok else -2)
    for heads, ok in (((2 ** 20 - 1, 1), True), ((2 ** 20, 1), False)):
        a.batch, a.seqlen, a.heads[0], a.heads[1] = 1, 2, *heads
        assert lib.issm_rotary_norm_bwd_bytes(C.byref(a), C.byref(need)) == (0 if ok else -2)
