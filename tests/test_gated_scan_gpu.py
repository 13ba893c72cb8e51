"""gated_scan and gated_scan_step against the recurrence token by token in float64 (oracle/sequence_ref.py)."""
import pytest
import torch

from oracle import sequence_ref as R

pytestmark = pytest.mark.gpu

# A step of the recurrence rounds its decay and its state once each in fp32, 2^-24 of the state at most, and takes beta from a reciprocal, a
# series and a root of about two places each.  The tests' decays remember at most some 60 tokens on average (A <= -0.03 at a gate of 1/2), so that
# a state is off by 60 * 2 * 2^-24 = 7e-6 of itself if all errors agree; gradients go through two such recurrences.
FP32 = dict(y=1e-5, grad=2e-5)
# bf16 results are rounded once on top: half of a step of 2^-7, off by at most 2^-8 of each value and so of their norm (a single value close
# above a power of two reaches it)
STEP = 2.0 ** -8


def make(B, L, C, dtype, seed=0, in_gate=True, initial=True, packed=0, A_lo=-1.0):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    d = dict(x=n(B, L, C).to(dtype), gate=n(B, L, C).to(dtype), A=A_lo + (-0.03 - A_lo) * torch.rand(C, generator=g),
             in_gate=n(B, L, C).to(dtype) if in_gate else None, initial_states=n(B, C) if initial else None, seq_idx=None)
    if packed:
        ids = torch.zeros(B, L, dtype=torch.long)
        for b in range(B):
            for c in torch.randint(0, L, (packed,), generator=g).tolist():
                ids[b, c:] += 1
        ids[0] -= ids[0, 0].clone()    # one row that takes its initial states
        d["seq_idx"] = ids
    return d, n(B, L, C).to(dtype), n(B, C)


LEAVES = ("x", "gate", "A", "in_gate", "initial_states")


def run(d, dy, dlast, **kw):
    from dest3d_amd import gated_scan
    g = {k: None if v is None else v.cuda() for k, v in d.items()}
    for k in LEAVES:
        if g[k] is not None:
            g[k].requires_grad_()
    y, last = gated_scan(**g, return_final_states=True, **kw)
    names = [k for k in LEAVES if g[k] is not None]
    grads = torch.autograd.grad((y, last), [g[k] for k in names], (dy.cuda(), dlast.cuda()))
    return dict(y=y.detach(), last=last.detach(), **{"d" + k: v for k, v in zip(names, grads)})


def ref(d, dy, dlast, **kw):
    r = {k: v if v is None or k == "seq_idx" else v.double().requires_grad_() for k, v in d.items()}
    y, last = R.gated_scan(**r, **kw)
    names = [k for k in LEAVES if r[k] is not None]
    grads = torch.autograd.grad((y, last), [r[k] for k in names], (dy.double(), dlast.double()), allow_unused=True)
    return dict(y=y.detach(), last=last.detach(), **{"d" + k: torch.zeros_like(r[k]) if v is None else v for k, v in zip(names, grads)})


def check(got, want):
    for k, w in want.items():
        v = got[k].double().cpu()
        assert v.shape == w.shape and torch.isfinite(v).all(), k
        lim = FP32["grad" if k.startswith("d") else "y"] + (STEP if got[k].dtype == torch.bfloat16 else 0.0)
        off, size = (v - w).norm().item(), w.norm().item()
        assert off <= lim * size + 1e-30, (k, off / max(size, 1e-300), lim)


SIZES = [(1, 1, 1), (2, 1, 5), (3, 2, 3), (1, 127, 4), (2, 128, 64), (3, 129, 65), (2, 300, 70), (1, 513, 130), (2, 1000, 288), (1, 2049, 67)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,L,C", SIZES)
def test_forward_and_gradients(B, L, C, dtype):
    case = make(B, L, C, dtype, seed=L + C)
    check(run(*case), ref(*case))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("in_gate,normalize,initial,packed,reverse", [
    (False, True, True, 0, False), (True, False, True, 0, False), (False, False, False, 0, False), (True, True, False, 5, False),
    (True, True, True, 9, True), (False, False, True, 4, True), (False, True, True, 3, False), (True, False, False, 12, False),
    (True, True, True, 0, True)])
def test_forms(in_gate, normalize, initial, packed, reverse, dtype):
    for B, L, C in ((2, 333, 40), (2, 37, 2)):
        case = make(B, L, C, dtype, seed=packed, in_gate=in_gate, initial=initial, packed=packed)
        check(run(*case, normalize=normalize, reverse=reverse), ref(*case, normalize=normalize, reverse=reverse))


def test_every_token_a_sequence_of_its_own():
    case = make(2, 300, 24, torch.float32)
    case[0]["seq_idx"] = torch.arange(300).expand(2, 300).clone()
    check(run(*case), ref(*case))
    case[0]["seq_idx"] = torch.arange(1, 301).expand(2, 300).clone()   # (and none that takes the initial states)
    got = run(*case)
    check(got, ref(*case))
    assert not got["dinitial_states"].any()


def test_one_sequence_by_name_is_no_packing():
    d, dy, dlast = make(2, 300, 24, torch.float32)
    plain = run(d, dy, dlast)
    named = run(dict(d, seq_idx=torch.zeros(2, 300, dtype=torch.int32)), dy, dlast)
    assert all(torch.equal(plain[k], named[k]) for k in plain)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides(dtype):
    """Slices of one projection at odd offsets, rows in another order, repeated inputs: as their contiguous copies, bit for bit."""
    from dest3d_amd import gated_scan
    g = torch.Generator().manual_seed(3)
    B, L, C = 2, 260, 70
    wide = torch.randn(L, B, 3 * C + 5, generator=g).to(dtype).cuda()
    x, gate, in_gate = (wide[..., 1 + i * (C + 1):1 + i * (C + 1) + C].transpose(0, 1) for i in range(3))
    A = -torch.rand(C, generator=g).cuda() - 0.03
    repeated = torch.randn(1, 1, C, generator=g).to(dtype).cuda().expand(B, L, C)
    ids = (torch.arange(L, dtype=torch.int32) // 50)[None].expand(B, L).cuda()
    for kw in (dict(gate=gate, in_gate=in_gate), dict(gate=repeated, in_gate=in_gate), dict(gate=gate, in_gate=repeated)):
        for reverse in (False, True):
            a = gated_scan(x, A=A, seq_idx=ids, reverse=reverse, **kw)
            b = gated_scan(x.contiguous(), A=A, seq_idx=ids.contiguous(), reverse=reverse, **{k: v.contiguous() for k, v in kw.items()})
            assert torch.equal(a, b)
    # a gradient that is repeated, and those of a repeated input and of channels that are not contiguous
    xr = torch.randn(B, 1, C, generator=g).to(dtype).cuda().requires_grad_()
    xt = torch.randn(B, C, L, generator=g).to(dtype).cuda().requires_grad_()
    gated_scan(xr.expand(B, L, C) + xt.transpose(1, 2), gate, A).sum().backward()
    full = (xr.detach().expand(B, L, C) + xt.detach().transpose(1, 2)).contiguous().requires_grad_()
    gated_scan(full, gate, A).backward(torch.ones_like(full))
    assert torch.equal(xt.grad, full.grad.transpose(1, 2))
    assert torch.equal(xr.grad, full.grad.sum(1, keepdim=True))


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("reverse", [False, True])
def test_nothing_passes_a_cut(bad, reverse):
    """A sequence whose inputs, states or gradients are no numbers leaves its neighbours' results and gradients as they were."""
    d, dy, dlast = make(2, 300, 24, torch.float32)
    ids = torch.zeros(2, 300, dtype=torch.int32)
    ids[:, 90:170], ids[:, 170:] = 1, 2
    d["seq_idx"] = ids
    clean = run(d, dy, dlast, reverse=reverse)
    for where in ("x", "gate", "in_gate", "dy"):
        e, ey = {k: None if v is None else v.clone() for k, v in d.items()}, dy.clone()
        (ey if where == "dy" else e[where])[:, 120] = bad
        got = run(e, ey, dlast, reverse=reverse)
        keep = torch.ones(300, dtype=torch.bool)
        keep[90:170] = False
        for k in ("y", "dx", "dgate", "din_gate"):
            assert torch.equal(got[k][:, keep], clean[k][:, keep]), (where, k)
        assert torch.equal(got["last"], clean["last"]) and torch.equal(got["dinitial_states"], clean["dinitial_states"])
        if where == "x" and bad != bad:
            assert torch.isnan(got["y"][:, 120]).all()


def test_gates_at_their_ends():
    """Full and empty gates, infinite ones too, and channels that nothing decays in: values as the formula's limits, gradients finite."""
    B, L, C = 1, 140, 8
    d, dy, dlast = make(B, L, C, torch.float32)
    d["gate"][:, ::3] = 60.0
    d["gate"][:, 1::3] = -60.0
    d["gate"][:, 7], d["gate"][:, 8] = -float("inf"), float("inf")
    d["in_gate"][:, ::5] = -200.0
    want = ref(dict(d, gate=d["gate"].clamp(-300, 300)), dy, dlast)
    got = run(d, dy, dlast)
    # where beta is 0 (sigmoid(-300) = 5e-131 rounds to it in fp32) the oracle in float64 still has a number, below 1e-60
    check(got, want)
    d["A"][:4] = 0.0
    got = run(d, dy, dlast)
    assert all(torch.isfinite(v).all() for v in got.values())
    want = d["initial_states"][:, None, :4].expand(B, L, 4)
    assert torch.equal(got["y"][..., :4].cpu(), want)
    assert not got["dgate"][..., :4].any()
    # a state that stays: dA is what the decays' own part gives, sum c_t h_{t-1} r_t, and nothing through beta, whose derivative has no value there
    c = dy[..., :4].double().flip(1).cumsum(1).flip(1) + dlast[:, None, :4].double()
    terms = c * want.double() * torch.sigmoid(d["gate"][..., :4].double())
    assert ((got["dA"][:4].double().cpu() - terms.sum((0, 1))).abs() <= FP32["grad"] * terms.abs().sum((0, 1))).all()


def test_decays_of_all_sizes():
    """From nothing to far beyond fp32's range, on both sides of the series' end, over a length that a decay next to one remembers whole."""
    B, L, C = 1, 600, 16
    d, dy, dlast = make(B, L, C, torch.float32)
    d["A"] = -torch.logspace(-6, 4, C)
    d["gate"] = torch.randn(B, L, C, generator=torch.Generator().manual_seed(1))
    got, want = run(d, dy, dlast), ref(d, dy, dlast)
    for c in range(C):   # each channel by itself: 600 steps of 2^-24 twice, if all errors agree, in a gradient twice that
        for k in want:
            if k == "dA":
                continue   # (its terms cancel in channels that remember all: below, by its own terms' size)
            v, w = got[k][..., c].double().cpu(), want[k][..., c]
            assert (v - w).norm() <= (1.5e-4 if k.startswith("d") else 7.2e-5) * w.norm() + 1e-30, (c, k)
    r = {k: v if v is None or k == "seq_idx" else v.double() for k, v in d.items()}
    A = r["A"][None].expand(L, C).clone().requires_grad_()   # a parameter for each token: the terms of dA
    y, last = R.gated_scan(r["x"], r["gate"], A[None], r["in_gate"], r["initial_states"])
    (terms,) = torch.autograd.grad((y, last), (A,), (dy.double(), dlast.double()))
    assert ((got["dA"].double().cpu() - want["dA"]).abs() <= 1.5e-4 * terms.abs().sum(0) + 1e-30).all()


def test_gradients_by_differences():
    from dest3d_amd import gated_scan
    d, dy, dlast = make(2, 150, 9, torch.float32, packed=2)
    got = run(d, dy, dlast)
    g = {k: None if v is None else v.cuda() for k, v in d.items()}

    def loss(**kw):
        y, last = gated_scan(**{**g, **kw}, return_final_states=True)
        return (y.double() * dy.cuda().double()).sum() + (last.double() * dlast.cuda().double()).sum()

    gen = torch.Generator().manual_seed(5)
    for k in LEAVES:
        v = torch.randn(g[k].shape, generator=gen).cuda()
        if k == "A":
            v = v * 0.02      # (A stays below 0)
        v = torch.sign((got["d" + k] * v).sum()) * v + 0.3 * got["d" + k] / got["d" + k].abs().max() * v.abs().mean()   # (a direction with a slope)
        e = 2.0 ** -6
        slope = (loss(**{k: g[k] + e * v}) - loss(**{k: g[k] - e * v})).item() / (2 * e)
        want = (got["d" + k].double() * v.double()).sum().item()
        # the third derivative's share, e^2 / 6 of a function of exponentials of unit scale, and fp32 results' 1e-5 of the loss's terms over 2 e
        assert abs(slope - want) <= 2e-2 * abs(want), (k, slope, want)


def test_other_types():
    from dest3d_amd import gated_scan
    d, dy, dlast = make(2, 100, 12, torch.float32)
    g = {k: None if v is None else v.cuda() for k, v in d.items()}
    base = gated_scan(**g)
    for t in (torch.float16, torch.float64):
        e = {k: v if v is None else v.to(t) for k, v in g.items()}
        y, last = gated_scan(**e, return_final_states=True)
        assert y.dtype == t and last.dtype == torch.float32
        torch.testing.assert_close(y.float(), base, rtol=2e-2, atol=2e-2) if t == torch.float16 else torch.testing.assert_close(y.float(), base, rtol=0, atol=0)
    x = g["x"].to(torch.bfloat16).requires_grad_()
    gate, A = g["gate"].requires_grad_(), g["A"].to(torch.float64).requires_grad_()
    y = gated_scan(x, gate, A)
    y.float().sum().backward()
    assert (y.dtype, x.grad.dtype, gate.grad.dtype, A.grad.dtype) == (torch.bfloat16, torch.bfloat16, torch.float32, torch.float64)


def test_no_tokens_and_no_rows():
    from dest3d_amd import gated_scan, gated_scan_step
    for B, L, C in ((2, 0, 5), (0, 4, 5), (2, 4, 0)):
        x = torch.zeros(B, L, C, device="cuda", requires_grad=True)
        A, h0 = torch.full((C,), -1.0, device="cuda", requires_grad=True), torch.randn(B, C, device="cuda", requires_grad=True)
        y, last = gated_scan(x, x, A, initial_states=h0, return_final_states=True)
        assert y.shape == x.shape and last.shape == (B, C)
        if L == 0:
            assert torch.equal(last, h0)
        w = torch.randn(B, C, device="cuda")
        (y.sum() + (last * w).sum()).backward()
        assert x.grad.shape == x.shape and not A.grad.any()
        if L == 0:
            assert torch.equal(h0.grad, w)
        assert torch.equal(gated_scan(x.detach(), x.detach(), A.detach(), return_final_states=True)[1], h0 * 0)
    x = torch.zeros(0, 5, device="cuda")
    assert gated_scan_step(x, x, torch.full((5,), -1.0, device="cuda"), torch.zeros(0, 5, device="cuda")).shape == (0, 5)


def test_parts_of_the_gradients():
    """Only what is asked for, and with either gradient of the results absent: as in the whole, bit for bit."""
    from dest3d_amd import gated_scan
    d, dy, dlast = make(2, 140, 20, torch.bfloat16)
    whole = run(d, dy, torch.zeros_like(dlast))
    for k in LEAVES:
        g = {n: None if v is None else v.cuda() for n, v in d.items()}
        g[k].requires_grad_()
        (grad,) = torch.autograd.grad(gated_scan(**g), (g[k],), (dy.cuda(),))
        assert torch.equal(grad, whole["d" + k]), k
    g = {n: None if v is None else v.cuda() for n, v in d.items()}
    g["x"].requires_grad_()
    _, last = gated_scan(**g, return_final_states=True)
    (grad,) = torch.autograd.grad(last, (g["x"],), (dlast.cuda(),))
    assert torch.equal(grad, run(d, torch.zeros_like(dy), dlast)["dx"])


def test_same_bits_twice_and_without_gradients():
    from dest3d_amd import gated_scan
    d, dy, dlast = make(3, 700, 100, torch.bfloat16, packed=3)
    a, b = run(d, dy, dlast), run(d, dy, dlast)
    assert all(torch.equal(a[k], b[k]) for k in a)
    with torch.no_grad():
        y, last = gated_scan(**{k: None if v is None else v.cuda() for k, v in d.items()}, return_final_states=True)
    assert torch.equal(y, a["y"]) and torch.equal(last, a["last"])


def test_streams():
    """Two calls at once, on streams of their own."""
    from dest3d_amd import gated_scan
    cases = [make(2, 3000, 96, torch.float32, seed=s) for s in (1, 2)]
    want = [run(*c) for c in cases]
    g = [{k: None if v is None else v.cuda() for k, v in c[0].items()} for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[] for _ in cases]
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(gated_scan(**g[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]["y"]) for i in range(2) for y in got[i])


def test_captured():
    """Forward and backward in a graph, replayed on other inputs with eager work between the replays; two graphs at once."""
    from dest3d_amd import gated_scan
    graphs = []
    for seed, L in ((1, 700), (2, 90)):
        d, dy, dlast = make(2, L, 72, torch.float32, seed=seed)
        g = {k: None if v is None else v.cuda() for k, v in d.items()}
        for k in LEAVES:
            g[k].requires_grad_()
        dyg = dy.cuda()

        def step(g=g, dyg=dyg):
            y = gated_scan(**g)
            return [y.detach(), *torch.autograd.grad(y, [g[k] for k in LEAVES], (dyg,))]

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, g, step, out))
    for turn in range(3):
        for graph, g, step, out in graphs:
            with torch.no_grad():
                for k in LEAVES:
                    g[k].add_(0.01 * turn * torch.randn_like(g[k])) if k != "A" else g[k].mul_(1.01)
            want = step()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_backward_reads_its_inputs_as_they_were():
    from dest3d_amd import gated_scan
    d, dy, _ = make(1, 50, 8, torch.float32)
    g = {k: None if v is None else v.cuda() for k, v in d.items()}
    x = g["x"].requires_grad_() * 1.0
    y = gated_scan(x, g["gate"], g["A"])
    x.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward(dy.cuda())
    x = g["x"].detach().requires_grad_()
    with pytest.raises(RuntimeError, match="first derivatives only"):
        torch.autograd.grad(gated_scan(x, g["gate"], g["A"]).sum(), x, create_graph=True)


# ------------------------------------------------------------------------------------------------------------ one token
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,C,in_gate,normalize", [(1, 1, True, True), (3, 7, False, True), (5, 288, True, False), (2, 1030, True, True), (70, 64, False, False)])
def test_step_by_step_is_the_scan(rows, C, in_gate, normalize, dtype):
    from dest3d_amd import gated_scan_step
    d, _, _ = make(rows, 6, C, dtype, seed=C, in_gate=in_gate)
    want, last = R.gated_scan(**{k: v if v is None else v.double() for k, v in d.items()}, normalize=normalize)
    g = {k: None if v is None else v.cuda() for k, v in d.items()}
    state = g["initial_states"].clone()
    for t in range(6):
        y = gated_scan_step(g["x"][:, t], g["gate"][:, t], g["A"], state, in_gate=None if g["in_gate"] is None else g["in_gate"][:, t], normalize=normalize)
        lim = 1e-5 + (STEP if dtype == torch.bfloat16 else 0.0)
        assert y.dtype == dtype and ((y.double().cpu() - want[:, t]).abs() <= lim * want[:, t].abs() + 1e-5).all()
    assert ((state.double().cpu() - last).abs() <= 1e-5 * last.abs() + 1e-5).all()


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_step_in_a_pool(index):
    """Slots in any order, rows without one, one slot several times, and a pool whose slots lie apart."""
    from dest3d_amd import gated_scan_step
    rows, C, slots = 150, 37, 40
    d, _, _ = make(1, rows, C, torch.float32)
    g = {k: None if v is None else v[0].cuda() if v.dim() > 1 else v.cuda() for k, v in d.items()}
    gen = torch.Generator().manual_seed(2)
    wide = torch.randn(slots, C + 11, generator=gen).cuda()
    before = wide.clone()
    at = torch.randint(-2, slots + 3, (rows,), generator=gen)
    at[5], at[6], at[149] = 7, 7, 7
    if index == torch.int64:
        at[9] = 2 ** 32 + 3    # (no slot, whatever its low half says)
    y = gated_scan_step(g["x"], g["gate"], g["A"], wide[:, 3:3 + C], in_gate=g["in_gate"], state_indices=at.to(index).cuda())
    state = before[:, 3:3 + C].double().cpu()
    for r in range(rows):
        s = int(at[r])
        if not 0 <= s < slots:
            assert not y[r].any()
            continue
        one = lambda t: t[r].double().cpu()[None, None]  # noqa: E731
        h, _ = R.gated_scan(one(g["x"]), one(g["gate"]), g["A"].double().cpu(), one(g["in_gate"]), state[s][None].clone())
        state[s] = h[0, 0]
        assert ((y[r].double().cpu() - h[0, 0]).abs() <= 2e-5).all(), r
    assert ((wide[:, 3:3 + C].double().cpu() - state).abs() <= 2e-5).all()
    assert torch.equal(wide[:, :3], before[:, :3]) and torch.equal(wide[:, 3 + C:], before[:, 3 + C:])
    touched = torch.zeros(slots, dtype=torch.bool)
    touched[at[(at >= 0) & (at < slots)]] = True
    assert torch.equal(wide[~touched.cuda()], before[~touched.cuda()])


def test_step_tells_what_saved_its_state_and_is_captured():
    from dest3d_amd import gated_scan_step
    d, _, _ = make(1, 4, 8, torch.float32)
    g = {k: None if v is None else v[0].cuda() if v.dim() > 1 else v.cuda() for k, v in d.items()}
    state = torch.randn(4, 8, device="cuda")
    version = state._version
    w = torch.ones(4, 8, device="cuda", requires_grad=True)
    kept = (w * state).sum()
    gated_scan_step(g["x"], g["gate"], g["A"], state)
    assert state._version > version
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        kept.backward()
    at = torch.tensor([2, 0, -1, 3], device="cuda")
    y0 = gated_scan_step(g["x"], g["gate"], g["A"], state.clone(), state_indices=at)
    graph = torch.cuda.CUDAGraph()
    start = state.clone()
    with torch.cuda.graph(graph):
        y = gated_scan_step(g["x"], g["gate"], g["A"], state, state_indices=at)
    for _ in range(3):
        state.copy_(start)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, y0)
    with torch.inference_mode():
        gated_scan_step(g["x"], g["gate"], g["A"], torch.zeros(4, 8, device="cuda"))


# ------------------------------------------------------------------------------------------- ways through the kernels
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,L,C,packed,reverse", [(520, 130, 8, 0, False), (520, 57, 8, 3, True), (300, 113, 72, 2, False), (515, 1, 4, 0, False), (530, 56, 7, 2, False)])
def test_rows_that_fill_the_gpu(B, L, C, packed, reverse, dtype):
    """Many rows, one workgroup each from the first tile to the last; an odd width takes the other addresses."""
    case = make(B, L, C, dtype, seed=L, packed=packed)
    check(run(*case, reverse=reverse), ref(*case, reverse=reverse))


@pytest.mark.parametrize("L", [55, 56, 57, 111, 112, 113, 223, 224, 225, 448, 449])
@pytest.mark.parametrize("C", [62, 64, 66])
def test_ends_of_tiles(L, C):
    """Lengths and widths to both sides of what a tile takes, forward and backward."""
    case = make(2, L, C, torch.bfloat16, seed=L, packed=1)
    check(run(*case), ref(*case))


def test_long_rows():
    """20000 tokens through some 180 tiles of 112 and 360 of 56, on many workgroups, twice: the oracle's values, and the same bits."""
    case = make(2, 20000, 6, torch.float32, packed=2)
    got = run(*case)
    check(got, ref(*case))
    again = run(*case)
    assert all(torch.equal(got[k], again[k]) for k in got)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_same_values_by_all_addresses(dtype):
    """Rows at odd places and rows too far apart for 32 bits: what aligned rows give, bit for bit, states and their gradients too."""
    from dest3d_amd import gated_scan
    B, L, C = 2, 150, 64
    d, dy, dlast = make(B, L, C, dtype)
    g = {k: None if v is None else v.cuda() for k, v in d.items()}
    want = run(d, dy, dlast)

    def moved(t, token, start):
        wide = torch.empty(start + B * L * token, dtype=dtype, device="cuda")
        v = wide.as_strided((B, L, C), (L * token, token, 1), start)
        v.copy_(t)
        return v

    for token, start in ((C + 3, 1), (C + 2, 0), (5_000_000, 0) if dtype == torch.bfloat16 else (C + 1, 3)):
        x = moved(g["x"], token, start).requires_grad_()
        gate = moved(g["gate"], C + 2, 2).requires_grad_()
        y, last = gated_scan(x, gate, g["A"], in_gate=g["in_gate"], initial_states=g["initial_states"], return_final_states=True)
        dx, dgate = torch.autograd.grad((y, last), (x, gate), (dy.cuda(), dlast.cuda()))
        assert torch.equal(y, want["y"]) and torch.equal(last, want["last"]) and torch.equal(dx, want["dx"]) and torch.equal(dgate, want["dgate"])
        del x, gate


def test_offsets_beyond_32_bits():
    """Tokens, rows and slots more than 2^31 elements apart."""
    from dest3d_amd import gated_scan, gated_scan_step
    far = 2 ** 31 + 64
    wide = torch.empty(far + 4096, dtype=torch.bfloat16, device="cuda")
    A = -torch.rand(64, device="cuda") - 0.03
    for strides in ((0, far), (far, 64)):
        n = (1, 2) if strides[0] == 0 else (2, 2)
        x = wide.as_strided((*n, 64), (*strides, 1))
        x.copy_(torch.randn(*n, 64))
        gate = torch.randn(*n, 64, device="cuda").bfloat16()
        assert torch.equal(gated_scan(x, gate, A), gated_scan(x.contiguous(), gate, A))
        assert torch.equal(gated_scan(x, gate, A, reverse=True), gated_scan(x.contiguous(), gate, A, reverse=True))
    pool = torch.empty(far + 4096, dtype=torch.float32, device="cuda").as_strided((2, 64), (far, 1))
    pool.copy_(torch.randn(2, 64))
    small, at = pool.contiguous(), torch.tensor([1, 0], device="cuda")
    x = torch.randn(2, 64, device="cuda")
    assert torch.equal(gated_scan_step(x, x, A, pool, state_indices=at), gated_scan_step(x, x, A, small, state_indices=at))
    assert torch.equal(pool, small)


def test_refusals():
    from dest3d_amd import gated_scan, gated_scan_step
    x, A = torch.zeros(2, 5, 8, device="cuda"), torch.full((8,), -1.0, device="cuda")
    ids = torch.zeros(2, 5, dtype=torch.int32, device="cuda")
    for kw in (dict(x=x[0]), dict(gate=x[:, :4]), dict(in_gate=x[..., :4]), dict(A=A[:4]), dict(A=A[None]), dict(initial_states=x[:, 0, :4]), dict(seq_idx=ids[:, :4])):
        with pytest.raises(ValueError):
            gated_scan(**{**dict(x=x, gate=x, A=A), **kw})
    for kw in (dict(x=x.long()), dict(gate=x.int()), dict(A=A.long()), dict(seq_idx=ids.float()), dict(initial_states=ids[:, :1].expand(2, 8))):
        with pytest.raises(TypeError):
            gated_scan(**{**dict(x=x, gate=x, A=A), **kw})
    for kw in (dict(gate=x.cpu()), dict(A=A.cpu()), dict(seq_idx=ids.cpu())):
        with pytest.raises(RuntimeError, match="all operands must be on"):
            gated_scan(**{**dict(x=x, gate=x, A=A), **kw})
    t, s = x[:, 0], torch.zeros(3, 8, device="cuda")
    at = torch.tensor([0, 2], device="cuda")
    for kw in (dict(x=x), dict(gate=t[:1]), dict(A=A[:4]), dict(state=s[:, :4]), dict(state_indices=at[:1]), dict(state_indices=None)):
        with pytest.raises(ValueError):
            gated_scan_step(**{**dict(x=t, gate=t, A=A, state=s, state_indices=at), **kw})
    for kw in (dict(state=s.double()), dict(state=s.bfloat16()), dict(state_indices=at.float()), dict(state_indices=at.to(torch.int16))):
        with pytest.raises(TypeError):
            gated_scan_step(**{**dict(x=t, gate=t, A=A, state=s, state_indices=at), **kw})
    for state in (s[:1].expand(3, 8), torch.zeros(8, 3, device="cuda").t()):     # slots that overlap, channels apart
        with pytest.raises(AssertionError):
            gated_scan_step(t, t, A, state, state_indices=at)
    with pytest.raises(RuntimeError, match="no backward"):
        gated_scan_step(t.clone().requires_grad_(), t, A, s, state_indices=at)
    with torch.no_grad():
        gated_scan_step(t.clone().requires_grad_(), t, A, s, state_indices=at)


def test_modes():
    """Inference mode, lazy negations, and forward derivatives, which there are none of."""
    from dest3d_amd import gated_scan, qk_norm_rotary, rotary, rotary_table
    d, _, _ = make(2, 60, 8, torch.float32)
    g = {k: None if v is None else v.cuda() for k, v in d.items()}
    want = gated_scan(**g)
    q, w, tab = torch.randn(1, 9, 2, 32, device="cuda"), torch.rand(32, device="cuda"), rotary_table(9, 32)
    turned = rotary(q, None, tab)
    with torch.inference_mode():
        assert torch.equal(gated_scan(**g), want) and torch.equal(rotary(q, None, tab), turned)
    lazy = torch.complex(g["x"], -g["x"]).conj().imag
    assert lazy.is_neg() and torch.equal(gated_scan(**{**g, "x": lazy}), want)
    lazy = torch.complex(q, -q).conj().imag
    assert lazy.is_neg() and torch.equal(rotary(lazy, None, tab), turned)
    import torch.autograd.forward_ad as fwAD
    with fwAD.dual_level():
        for call in (lambda: gated_scan(fwAD.make_dual(g["x"], g["x"]), g["gate"], g["A"]), lambda: rotary(fwAD.make_dual(q, q), None, tab),
                     lambda: qk_norm_rotary(fwAD.make_dual(q, q), None, w, None, tab)):
            with pytest.raises(RuntimeError):
                call()


@pytest.mark.parametrize("dtype,index,C", [(torch.float32, torch.int64, 5), (torch.bfloat16, torch.int32, 8)])
def test_step_of_many_rows(dtype, index, C):
    """More rows than a launch looks over: those of one slot still in their order, whichever launch they are in."""
    from dest3d_amd import gated_scan_step
    rows, slots = 4099, 1500
    d, _, _ = make(1, rows, C, dtype)
    x, gate, in_gate, A = d["x"][0], d["gate"][0], d["in_gate"][0], d["A"]
    wide = torch.cat([x, gate, in_gate], 1).cuda()      # rows that lie apart
    gen = torch.Generator().manual_seed(5)
    at = torch.randint(-1, slots, (rows,), generator=gen)
    at[[0, 2047, 2048, 4096, 4098]] = 11
    pool = torch.randn(slots, C, generator=gen)
    got = pool.cuda()
    y = gated_scan_step(wide[:, :C], wide[:, C:2 * C], A.cuda(), got, in_gate=wide[:, 2 * C:], state_indices=at.to(index).cuda())
    state, want = pool.double(), torch.zeros(rows, C, dtype=torch.float64)
    turn = torch.zeros(rows, dtype=torch.long)           # a row's place among those of its slot
    seen = {}
    for r, s in enumerate(at.tolist()):
        turn[r] = seen[s] = seen.get(s, -1) + 1
    for n in range(int(turn.max()) + 1):
        r = ((turn == n) & (at >= 0)).nonzero()[:, 0]
        h, _ = R.gated_scan(x[r][:, None].double(), gate[r][:, None].double(), A.double(), in_gate[r][:, None].double(), state[at[r]])
        state[at[r]] = want[r] = h[:, 0]
    # (a value's states are off by 7e-6 of their size, about 1 to 4 here; bf16 by half a step on top)
    assert ((y.double().cpu() - want).abs() <= 3e-5 + (STEP * want.abs() if dtype == torch.bfloat16 else 0.0)).all()
    assert ((got.double().cpu() - state).abs() <= 3e-5).all() and not y[at.cuda() < 0].any()


@pytest.mark.parametrize("wide", [("gate",), ("in_gate",), ("x",), ("gate", "in_gate")])
def test_operands_of_two_types(wide):
    """An operand in float32 beside others in bfloat16 is not rounded to theirs: what is returned in float32 is as exact as if all were."""
    from dest3d_amd import gated_scan_step
    d, dy, dlast = make(2, 150, 20, torch.bfloat16, seed=3)
    for k in wide:
        d[k] = torch.randn(2, 150, 20, generator=torch.Generator().manual_seed(len(k)))
    check(run(d, dy.to(d["x"].dtype), dlast), ref(d, dy, dlast))
    one = {k: d[k][:, 0] for k in ("x", "gate", "in_gate")}
    pool = d["initial_states"].cuda()
    gated_scan_step(one["x"].cuda(), one["gate"].cuda(), d["A"].cuda(), pool, in_gate=one["in_gate"].cuda())
    want, _ = R.gated_scan(*(one[k][:, None].double() for k in ("x", "gate")), d["A"].double(), one["in_gate"][:, None].double(), d["initial_states"].double())
    assert (pool.double().cpu() - want[:, 0]).norm() <= FP32["y"] * want.norm()


def test_step_refuses_its_state_as_an_input():
    from dest3d_amd import gated_scan_step
    pool, x, A = torch.randn(4, 8, device="cuda"), torch.randn(4, 8, device="cuda"), torch.full((8,), -1.0, device="cuda")
    before = pool.clone()
    for kw in (dict(x=pool), dict(gate=pool), dict(in_gate=pool), dict(A=pool[1]), dict(x=pool[1:], gate=x[1:], state=pool[:3])):
        with pytest.raises(AssertionError, match="share no memory"):
            gated_scan_step(**{**dict(x=x, gate=x, A=A, state=pool), **kw})
    assert torch.equal(pool, before)
    both = torch.randn(8, 8, device="cuda")    # (halves of one allocation are no overlap)
    want = both[4:].clone()
    y = gated_scan_step(both[:4], x, A, both[4:])
    assert torch.equal(y, gated_scan_step(both[:4].clone(), x, A, want)) and torch.equal(both[4:], want)


def test_kept_graphs_checkpoints_and_threads():
    """A graph run backwards twice, a call computed again in its backward, and calls from several threads give the same bits."""
    import threading
    from torch.utils.checkpoint import checkpoint
    from dest3d_amd import gated_scan
    d, dy, _ = make(2, 300, 64, torch.float32)
    g = {k: None if v is None else v.cuda() for k, v in d.items()}
    leaves = [g[k].requires_grad_() for k in LEAVES]
    dy = dy.cuda()

    def call(x, gate, A, in_gate, h0):
        return gated_scan(x, gate, A, in_gate, h0)

    y = call(*leaves)
    want = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(want, torch.autograd.grad(y, leaves, dy)))
    for reentrant in (False, True):
        for t in leaves:
            t.grad = None
        checkpoint(call, *leaves, use_reentrant=reentrant).backward(dy)
        assert all(torch.equal(a, t.grad) for a, t in zip(want, leaves))
    same = []

    def work():
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(5):
                got = torch.autograd.grad(call(*leaves), leaves, dy)
                torch.cuda.current_stream().synchronize()
                same.append(all(torch.equal(a, b) for a, b in zip(want, got)))

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work) for _ in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert same == [True] * 15


@pytest.mark.parametrize("B,L,C,dtype,packed", [
    (8, 6800, 66, torch.float32, 2), (7, 11000, 33, torch.float32, 0), (3, 15000, 130, torch.bfloat16, 3), (170, 240, 131, torch.float32, 2),
    (513, 60, 34, torch.float32, 2), (260, 130, 70, torch.bfloat16, 0), (511, 300, 7, torch.bfloat16, 2), (5, 20, 33, torch.float32, 0)])
def test_widths_that_share_cache_lines(B, L, C, dtype, packed):
    """Rows in the order in which an XCD takes those side by side: numbers of rows that are multiples of eight and not, shared and walked.  The same
    channels in rows of whole cache lines, which go in the other order, have the same bits; short ones are compared with the oracle too."""
    d, dy, dlast = make(B, L, C, dtype, packed=packed)
    got = run(d, dy, dlast)
    more = -C % 64

    def pad(k, t):
        return t if t is None or k == "seq_idx" else torch.nn.functional.pad(t, (0, more), value=-0.5 if k == "A" else 0.0)

    whole = run({k: pad(k, v) for k, v in d.items()}, pad("dy", dy), pad("dlast", dlast))
    for k, v in got.items():
        assert torch.isfinite(v).all() and torch.equal(v, whole[k][..., :C]), k
    if L <= 130:
        check(got, ref(d, dy, dlast))


# ------------------------------------------------------------------------------------------------ states that grow
def grown(got, want, lim):
    """Each channel by itself: the largest would hide the others."""
    for k, w in want.items():
        v = got[k].double().cpu()
        assert v.shape == w.shape and torch.isfinite(w).all() and torch.isfinite(v).all(), k
        over = tuple(range(w.dim() - 1))
        off, size = torch.linalg.vector_norm(v - w, dim=over), torch.linalg.vector_norm(w, dim=over)
        bar = (2 if k.startswith("d") else 1) * lim + (STEP if got[k].dtype == torch.bfloat16 else 0.0)
        assert (off <= bar * size + 1e-30).all(), (k, (off / size.clamp_min(1e-300)).max().item(), bar)


# One step's decay is off by 2^-24 times 6 l (the sigmoid's four roundings, the product's and the exponent's in base 2) and 2 (exponential and state), l = A r
def step_error(l):
    return (6 * l + 2) * 2.0 ** -24


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,L,C,packed,reverse", [(2, 300, 24, False, False), (2, 1500, 6, False, True), (1, 100, 5, False, False), (3, 1200, 7, True, False),
                                                  (520, 200, 8, False, False), (520, 130, 7, True, True)])
def test_states_that_grow_behind_zeros(B, L, C, packed, reverse, dtype):
    """Positive A: inputs that are zero up to the last 20 tokens, gradients that are zero behind the first 20.  States and what they pass back are 0 over
    many tiles whose decays' product is far beyond fp32."""
    d, dy, dlast = make(B, L, C, dtype, seed=L, initial=False)
    d["gate"] = (0.3 * d["gate"].float()).to(dtype)
    d["A"] = 1.0 + 3.0 * torch.rand(C, generator=torch.Generator().manual_seed(L))
    first, last = (slice(0, 20), slice(L - 20, L)) if not reverse else (slice(L - 20, L), slice(0, 20))
    keep = torch.zeros(L, dtype=torch.bool)
    keep[last] = True
    d["x"][:, ~keep] = 0
    keep[:] = False
    keep[first] = True
    dy[:, ~keep] = 0
    if packed:   # (a cut among the zeros)
        d["seq_idx"] = torch.zeros(B, L, dtype=torch.int32)
        d["seq_idx"][:, L // 2:] = 1
    kw = dict(normalize=False, reverse=reverse)
    l = (d["A"] * torch.sigmoid(d["gate"].double())).max().item()
    got, want = run(d, dy, dlast * 0, **kw), ref(d, dy, dlast * 0, **kw)
    assert want["y"].abs().max() > 1e8 and want["dx"].abs().max() > 1e8
    grown(got, want, 20 * step_error(l))


@pytest.mark.parametrize("B,L,l,reverse", [(2, 130, 1.2, False), (2, 90, 1.7, False), (600, 90, 1.7, True), (1, 140, 1.1, True)])
def test_small_states_that_grow(B, L, l, reverse):
    """A state of 1e-36 that grows over a tile by more than fp32 holds, and a gradient that does, stay numbers."""
    C = 8
    d = dict(x=torch.zeros(B, L, C), gate=torch.zeros(B, L, C), A=torch.full((C,), 2 * l), in_gate=None, initial_states=torch.full((B, C), 1e-36), seq_idx=None)
    dy, dlast = torch.zeros(B, L, C), torch.full((B, C), 1e-36)
    kw = dict(normalize=False, reverse=reverse)
    got, want = run(d, dy, dlast, **kw), ref(d, dy, dlast, **kw)
    grown({k: got[k] for k in want if k != "dx"}, {k: want[k] for k in want if k != "dx"}, L * step_error(l))
    grown(dict(dx=got["dx"]), dict(dx=want["dx"]), L * step_error(l))


def test_growth_within_a_window():
    """Growth over 30 tokens among ones that change nothing (empty gates): all gradients, A's among them."""
    d, dy, dlast = make(2, 400, 12, torch.float32)
    d["A"] = 1.0 + 2.0 * torch.rand(12, generator=torch.Generator().manual_seed(4))
    keep = torch.zeros(400, dtype=torch.bool)
    keep[150:180] = True
    d["gate"][:, ~keep] = -200.0
    d["gate"][:, keep] *= 0.3
    l = (d["A"] * torch.sigmoid(d["gate"].double())).max().item()
    got, want = run(d, dy, dlast, normalize=False), ref(d, dy, dlast, normalize=False)
    # (30 steps that grow; 370 sums in which all terms stay, 2^-24 each)
    grown(got, want, 30 * step_error(l) + 370 * 2.0 ** -24)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,L,C,packed", [(2, 300, 24, False), (1, 1500, 7, True), (520, 200, 8, True), (520, 200, 7, False), (2, 100, 3, False)])
def test_steep_growth_of_zeros(B, L, C, packed, dtype):
    """Decays that four tokens multiply beyond fp32, each within it, on states and gradients of 0; smaller ones at both ends, where inputs and gradients are."""
    d, dy, dlast = make(B, L, C, dtype, seed=C, initial=False)
    g = torch.Generator().manual_seed(C)
    d["A"] = 20.0 + 70.0 * torch.rand(C, generator=g)
    gate = torch.full((B, L, C), 2.0)
    gate[:, :20], gate[:, -20:] = -4.0, -4.0
    d["gate"] = (gate + 0.1 * torch.rand(B, L, C, generator=g) - 0.1).to(dtype)
    d["x"][:, :-20] = 0
    dy[:, 20:] = 0
    if packed:
        d["seq_idx"] = torch.zeros(B, L, dtype=torch.int32)
        d["seq_idx"][:, L // 2:] = 1
    assert (d["A"] * torch.sigmoid(d["gate"].double())).max() < 88
    l = (d["A"] * torch.sigmoid(d["gate"][:, :20].double())).max().item()
    got, want = run(d, dy, dlast * 0, normalize=False), ref(d, dy, dlast * 0, normalize=False)
    # (a step as above, its sigmoid's exponent of 4 rounded too)
    grown(got, want, 20 * (step_error(l) + 4 * l * 2.0 ** -24))


def test_steep_growth_for_a_token():
    """A far above what all tokens together could take, behind gates that are nearly empty but for one."""
    d, dy, dlast = make(2, 300, 12, torch.float32, in_gate=False)
    d["A"] = torch.full((12,), 60.0)
    d["gate"] = -30.0 + 0.3 * d["gate"]
    d["gate"][:, 150] = 0.0
    d["x"], d["initial_states"] = d["x"].abs(), d["initial_states"].abs()
    got, want = run(d, dy.abs(), dlast.abs(), normalize=False), ref(d, dy.abs(), dlast.abs(), normalize=False)
    # (sums of positive terms: 300 roundings of a state or what it passes back, the step's, and a sigmoid's exponent of 32)
    grown(got, want, 300 * 2.0 ** -24 + step_error(30.0) + 32 * 2.0 ** -24)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,L,C", [(2, 56, 8), (2, 57, 8), (3, 100, 7), (2, 225, 64), (1, 1, 4), (520, 57, 8)])
def test_no_number_at_the_last_token(B, L, C, dtype):
    """An infinite state behind the row, or an infinite gradient of a last state that a cut keeps from the row: the gradient of A is that of the tokens
    in front, bit for bit, however far the row's last tile reaches."""
    d, dy, dlast = make(B, L, C, dtype)
    clean = run(d, dy, dlast, normalize=False)
    for bad in (float("inf"), -float("inf"), float("nan")):
        e = dict(d, x=d["x"].clone())
        e["x"][:, -1] = bad
        got = run(e, dy, dlast, normalize=False)
        assert not torch.isfinite(got["last"]).any() and torch.equal(got["dA"], clean["dA"]) and torch.equal(got["dx"], clean["dx"])
        cut = dict(d, seq_idx=torch.zeros(B, L, dtype=torch.int32))
        cut["seq_idx"][:, -1] = 1
        want = run(cut, dy, dlast, normalize=False)
        got = run(cut, dy, torch.full_like(dlast, bad), normalize=False)
        assert torch.isfinite(got["dA"]).all()
        for k in ("dA", "dinitial_states"):
            assert torch.equal(got[k], want[k]), k
        for k in ("dx", "dgate", "din_gate"):
            assert torch.equal(got[k][:, :-1], want[k][:, :-1]), k


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,L,C,packed", [(520, 130, 8, 0), (300, 113, 72, 2), (3, 100, 8, 0), (600, 1, 8, 0)])
def test_walked_rows_by_all_addresses(B, L, C, packed, dtype):
    """Rows that one workgroup walks, at odd places: what aligned ones give, bit for bit."""
    d, dy, dlast = make(B, L, C, dtype, packed=packed)
    want = run(d, dy, dlast)
    wide = torch.empty(B * L * (C + 3) + 1, dtype=dtype, device="cuda")
    odd = wide.as_strided((B, L, C), (L * (C + 3), C + 3, 1), 1)
    odd.copy_(d["x"])
    got = run(dict(d, x=odd), dy, dlast)
    assert all(torch.equal(got[k], want[k]) for k in want)


def test_memory_of_many_short_rows():
    """A call of single tokens takes its results, and in the backward a row of partial sums for each row, beside its inputs."""
    from dest3d_amd import gated_scan
    B, C = 4096, 2048
    for width in (C, C - 1):
        x = torch.randn(B, 1, width, device="cuda", dtype=torch.bfloat16)
        A = torch.full((width,), -1.0, device="cuda")
        size = x.numel() * 2
        gated_scan(x, x, A)
        torch.cuda.synchronize()
        start = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        y = gated_scan(x, x, A)
        assert torch.cuda.max_memory_allocated() - start <= size + (1 << 21)
        leaves = [x.detach().requires_grad_(), x.detach().clone().requires_grad_(), A.detach().requires_grad_()]
        y = gated_scan(*leaves)
        start = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        torch.autograd.grad(y, leaves, x)
        assert torch.cuda.max_memory_allocated() - start <= 4 * size + (1 << 21)   # two gradients in bf16, sums in fp32
        torch.autograd.grad(gated_scan(*leaves[:2], A), leaves[:2], x)


def test_initial_states_may_change_before_the_backward():
    """The backward does not read them: a buffer of states that the next call's take over is no error, and the gradients are the same."""
    from dest3d_amd import gated_scan
    for L in (90, 700, 0):
        d, dy, dlast = make(2, L, 24, torch.float32)
        g = {k: None if v is None else v.cuda() for k, v in d.items()}
        leaves = [g[k].requires_grad_() for k in ("x", "gate", "A", "in_gate")]
        want = torch.autograd.grad(gated_scan(**g, return_final_states=True), leaves, (dy.cuda(), dlast.cuda()), allow_unused=L == 0)
        y, last = gated_scan(**g, return_final_states=True)
        g["initial_states"].copy_(last.detach() + 1.0)
        got = torch.autograd.grad((y, last), leaves, (dy.cuda(), dlast.cuda()), allow_unused=L == 0)
        assert all(torch.equal(a, b) for a, b in zip(got, want) if a is not None)


def test_step_refuses_its_state_as_an_input_in_a_pool_with_gaps():
    """Slots that lie apart: an input that has a number of one of them is refused; what lies beside them, between them or was copied is not."""
    from dest3d_amd import gated_scan_step
    C, A, at = 8, torch.full((8,), -1.0, device="cuda"), torch.tensor([2, 0, 3, 1], device="cuda")
    wide = torch.randn(9, 24, device="cuda")
    before = wide.clone()
    state, x = wide[:4, 8:16], torch.randn(4, C, device="cuda")
    for bad in (wide[:4, 8:16], wide[:4, 3:11], wide[:4, 15:23], wide[3:7, 8:16], wide[:8:2, 8:16], wide[3].view(1, 24)[:, 8:16].expand(4, C),
                wide.flatten()[13:61].view(4, 12)[:, 3:11]):   # (rows 12 apart, at 16, 28, 40, 52: the second and the fourth)
        for kw in (dict(x=bad), dict(gate=bad), dict(in_gate=bad)):
            with pytest.raises(AssertionError, match="share no memory"):
                gated_scan_step(**{**dict(x=x, gate=x, A=A, state=state, state_indices=at), **kw})
    with pytest.raises(AssertionError, match="share no memory"):
        gated_scan_step(x, x, wide[3, 12:20], state, state_indices=at)
    with pytest.raises(AssertionError, match="share no memory"):
        gated_scan_step(x, x, A, state, state_indices=wide.view(torch.int32)[1, 10:14])
    assert torch.equal(wide, before)
    for good in (wide[:4, :8], wide[:4, 16:], wide[4:8, 8:16], wide[5:9, 8:16], wide[4:8, 8:16].bfloat16(), torch.as_strided(wide, (4, C), (48, 1), 16)):
        copy = wide[:4, 8:16].clone()
        want = gated_scan_step(good.clone(), x, A, copy, in_gate=good.clone(), state_indices=at)
        got = gated_scan_step(good, x, A, state, in_gate=good, state_indices=at)
        assert torch.equal(got, want) and torch.equal(state, copy)
    # channels apart: the kernel reads a copy, made before a state changes
    square = torch.randn(C, C, device="cuda")
    copy = square.clone()
    want = gated_scan_step(square.t().clone(), square.t().clone(), A, copy)
    assert torch.equal(gated_scan_step(square.t(), square.t(), A, square), want) and torch.equal(square, copy)
