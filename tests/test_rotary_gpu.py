"""rotary and qk_norm_rotary against their definitions in float64 (oracle/sequence_ref.py), and a run of them with the recurrence, the scan, the
convolution and the norm."""
import pytest
import torch

from oracle import sequence_ref as R

pytestmark = pytest.mark.gpu

# A rotation is two products and a sum, three roundings of 2^-24 of its pair's size; the norm adds a sum of D squares (its error of a few 2^-24
# halved by the root), a quotient, a root and two products; the backward a second sum.  bf16 results are rounded once, by half a step of 2^-8.
EPS32, STEP = 2.0 ** -24, 2.0 ** -8


def table(n, rot, seed=0):
    from dest3d_amd import rotary_table
    return rotary_table(n, rot, device="cpu")


def make(B, L, H, K, D, rot, dtype, seed=0, rows=None, positions="rows"):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g).to(dtype)  # noqa: E731
    rows = rows or max(L, 4) + 40
    d = dict(q=n(B, L, H, D), k=n(B, L, K, D) if K else None, wq=(1 + 0.3 * torch.randn(D, generator=g)).to(dtype),
             wk=(1 + 0.3 * torch.randn(D, generator=g)).to(dtype) if K else None, table=table(rows, rot), pos=None)
    if positions == "rows":
        d["pos"] = torch.randint(0, rows, (B, L), generator=g)
    elif positions == "shared":
        d["pos"] = torch.randint(0, rows, (L,), generator=g).to(torch.int32)
    return d, n(B, L, H, D), n(B, L, K, D) if K else None


def run(d, dq, dk, norm, interleaved):
    from dest3d_amd import qk_norm_rotary, rotary
    g = {k: None if v is None else v.cuda() for k, v in d.items()}
    names = [k for k in (("q", "k", "wq", "wk") if norm else ("q", "k")) if g[k] is not None]
    for k in names:
        g[k].requires_grad_()
    if norm:
        y = qk_norm_rotary(g["q"], g["k"], g["wq"], g["wk"], g["table"], positions=g["pos"], interleaved=interleaved)
    else:
        y = rotary(g["q"], g["k"], g["table"], positions=g["pos"], interleaved=interleaved)
    y = (y,) if d["k"] is None else y
    grads = torch.autograd.grad(y, [g[k] for k in names], [t.cuda() for t in (dq, dk) if t is not None])
    return {**dict(zip(("yq", "yk"), (t.detach() for t in y))), **{"d" + k: v for k, v in zip(names, grads)}}


def ref(d, dq, dk, norm, interleaved):
    r = {k: v if v is None or k == "pos" else v.double() for k, v in d.items()}
    names = [k for k in (("q", "k", "wq", "wk") if norm else ("q", "k")) if r[k] is not None]
    for k in names:
        r[k].requires_grad_()
    y = []
    for k in ("q", "k"):
        if r[k] is not None:
            y.append(R.norm_rotary(r[k], r["w" + k], r["table"], r["pos"], 1e-6, interleaved) if norm else R.rotary(r[k], r["table"], r["pos"], interleaved))
    grads = torch.autograd.grad(y, [r[k] for k in names], [t.double() for t in (dq, dk) if t is not None])
    return {**dict(zip(("yq", "yk"), (t.detach() for t in y))), **{"d" + k: v for k, v in zip(names, grads)}}


def check(got, want):
    assert set(got) == set(want)
    for k, w in want.items():
        v = got[k].double().cpu()
        assert v.shape == w.shape, k
        half = STEP if got[k].dtype == torch.bfloat16 else 0.0
        if k in ("dwq", "dwk"):
            # a sum over rows: each term off by 16 roundings, and the sums' own
            assert (v - w).norm() <= (64 * EPS32 + half) * w.norm() + 1e-30, (k, (v - w).norm() / w.norm())
            continue
        # element by element: half a step of the value, and 16 roundings of a pair's size, which a head's largest value bounds
        big = w.abs().amax(-1, keepdim=True)
        assert ((v - w).abs() <= half * w.abs() + 24 * EPS32 * big + 1e-30).all(), (k, ((v - w).abs() / big).max())


SIZES = [  # B, L, H, K, D, rot: every width of the kernels' accesses, heads of one pair to the widest
    (1, 1, 1, 1, 2, 2), (2, 3, 1, 0, 64, 64), (1, 5, 4, 2, 128, 128), (2, 7, 3, 1, 128, 64), (1, 9, 8, 8, 36, 24), (2, 33, 2, 1, 80, 80),
    (1, 11, 5, 2, 96, 32), (1, 6, 1, 1, 256, 256), (1, 4, 2, 1, 100, 20), (1, 3, 2, 2, 37, 10), (1, 3, 1, 1, 1024, 1024), (1, 2, 3, 1, 1023, 510),
    (1, 3, 2, 1, 516, 258), (1, 2, 1, 1, 600, 2), (3, 130, 6, 2, 64, 64), (1, 2, 1, 1, 3, 2), (2, 5, 2, 1, 72, 72), (1, 17, 1, 1, 512, 512)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,L,H,K,D,rot", SIZES)
def test_forward_and_gradients(B, L, H, K, D, rot, interleaved, dtype):
    for norm in (False, True):
        for positions in ("rows", "shared", None):
            case = make(B, L, H, K, D, rot, dtype, seed=D, positions=positions)
            check(run(*case, norm, interleaved), ref(*case, norm, interleaved))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("norm", [False, True])
def test_many_rows(norm, dtype):
    """More rows than the backward's workgroups take at once."""
    case = make(4, 1500, 6, 2, 64, 64, dtype)
    check(run(*case, norm, False), ref(*case, norm, False))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
def test_strides(interleaved, dtype):
    """Slices of one projection at odd offsets, heads before tokens, repeated heads: as their contiguous copies, bit for bit, gradients too."""
    from dest3d_amd import qk_norm_rotary, rotary
    g = torch.Generator().manual_seed(1)
    B, L, H, K, D = 2, 19, 6, 2, 64
    n = lambda *s: torch.randn(*s, generator=g).to(dtype).cuda()  # noqa: E731
    wide = n(B, L, (H + 2 * K) * D + 3)
    q = wide[..., 1:1 + H * D].unflatten(-1, (H, D))
    k = wide[..., 2 + H * D:2 + (H + K) * D].unflatten(-1, (K, D))
    tr = n(B, H, L, D).transpose(1, 2)
    rep = n(B, L, 1, D).expand(B, L, K, D)
    skew = n(B, L, D, K).transpose(2, 3)      # features not contiguous
    wq, wk, tab = n(D), n(D), table(64, 32).cuda()
    pos = torch.randint(0, 64, (L, B), generator=g).cuda().t()
    for a, b in ((q, k), (tr, rep), (tr, skew)):
        for f in (lambda x, y: rotary(x, y, tab, positions=pos, interleaved=interleaved),
                  lambda x, y: qk_norm_rotary(x, y, wq, wk, tab, positions=pos, interleaved=interleaved)):
            res = []
            for x, y in ((a, b), (a.contiguous(), b.contiguous())):
                x, y = x.detach().requires_grad_(), y.detach().requires_grad_()
                out = f(x, y)
                res.append((*out, *torch.autograd.grad(out, (x, y), (tr, rep))))
            assert all(torch.equal(s, t) for s, t in zip(*res))


def test_positions_outside_the_table():
    from dest3d_amd import qk_norm_rotary, rotary
    q = torch.randn(1, 6, 2, 16, device="cuda")
    w, tab = torch.ones(16, device="cuda"), table(8, 12).cuda()
    for t in (torch.int32, torch.int64):
        pos = torch.tensor([0, 8, -1, 7, 2 ** 31 - 1, -2 ** 31], dtype=t, device="cuda")
        if t == torch.int64:
            pos[4] = 2 ** 32     # (no position, whatever its low half says)
        inside = torch.tensor([True, False, False, True, False, False], device="cuda")
        for y in (rotary(q, None, tab, positions=pos), qk_norm_rotary(q, None, w, None, tab, positions=pos)):
            assert torch.isnan(y[:, ~inside, :, :12]).all() and torch.isfinite(y[:, inside]).all() and torch.isfinite(y[..., 12:]).all()


def test_heads_of_zeros_and_of_no_numbers():
    """A head of zeros has the norm's eps under its root; one that is no number leaves the others of its token as they are."""
    from dest3d_amd import qk_norm_rotary
    q = torch.randn(1, 3, 4, 32, device="cuda")
    w, tab = torch.ones(32, device="cuda"), table(8, 32).cuda()
    want = qk_norm_rotary(q, None, w, None, tab)
    q[0, 1, 1] = 0.0
    q[0, 1, 2, 5] = float("nan")
    q[0, 2, 0, 3] = float("inf")
    x = q.clone().requires_grad_()
    y = qk_norm_rotary(x, None, w, None, tab)
    (grad,) = torch.autograd.grad(y, x, torch.ones_like(y))
    keep = torch.ones(1, 3, 4, dtype=torch.bool)
    keep[0, 1, 1] = keep[0, 1, 2] = keep[0, 2, 0] = False
    assert torch.equal(y[keep], want[keep]) and torch.isfinite(grad[keep]).all()
    assert not y[0, 1, 1].any() and torch.isfinite(grad[0, 1, 1]).all()
    assert torch.isnan(y[0, 1, 2]).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_sizes_of_values(dtype):
    """Heads far from unit size: the squares' sum stays in fp32's range for values of 1e-15 to 1e15."""
    d, dq, dk = make(1, 8, 4, 2, 128, 128, dtype)
    d["q"] = d["q"] * torch.logspace(-15, 15, 8).to(dtype)[None, :, None, None]
    got, want = run(d, dq, dk, True, False), ref(d, dq, dk, True, False)
    for t in range(8):
        check({"y": got["yq"][:, t], "dx": got["dq"][:, t]}, {"y": want["yq"][:, t], "dx": want["dq"][:, t]})


def test_turns_back():
    """A rotation by the negated sines is its inverse, and lengths are kept."""
    from dest3d_amd import rotary
    q, tab = torch.randn(2, 50, 3, 64, device="cuda"), table(50, 64).cuda()
    y = rotary(q, None, tab)
    torch.testing.assert_close(y.norm(dim=-1), q.norm(dim=-1), rtol=1e-6, atol=0)
    back = rotary(y, None, torch.cat([tab[:, :32], -tab[:, 32:]], 1))
    torch.testing.assert_close(back, q, rtol=0, atol=1e-6)


def test_gradients_by_differences():
    from dest3d_amd import qk_norm_rotary
    d, dq, dk = make(2, 9, 3, 2, 24, 16, torch.float32)
    got = run(d, dq, dk, True, True)
    g = {k: None if v is None else v.cuda() for k, v in d.items()}

    def loss(**kw):
        a = {**g, **kw}
        y = qk_norm_rotary(a["q"], a["k"], a["wq"], a["wk"], a["table"], positions=a["pos"], interleaved=True)
        return sum((t.double() * u.cuda().double()).sum() for t, u in zip(y, (dq, dk)))

    for k in ("q", "k", "wq", "wk"):
        v, e = got["d" + k] / got["d" + k].norm(), 2.0 ** -5
        slope = (loss(**{k: g[k] + e * v}) - loss(**{k: g[k] - e * v})).item() / (2 * e)
        # along the gradient itself; e^2 / 6 of the third derivative, and 1e-6 of the loss's terms over 2 e
        assert abs(slope - got["d" + k].norm().item()) <= 5e-3 * got["d" + k].norm().item(), (k, slope)


def test_types_and_absent_gradients():
    from dest3d_amd import qk_norm_rotary, rotary
    tab = table(9, 32).cuda()
    q, k = torch.randn(1, 9, 2, 32, device="cuda"), torch.randn(1, 9, 1, 32, device="cuda")
    w = torch.rand(32, device="cuda") + 0.5
    base = qk_norm_rotary(q, k, w, w, tab)
    for t in (torch.float16, torch.float64):
        y = qk_norm_rotary(q.to(t), k.to(t), w.to(t), w, tab.to(torch.float64))
        assert y[0].dtype == y[1].dtype == t
        for a, b in zip(y, base):
            torch.testing.assert_close(a.float(), b, rtol=4e-3, atol=4e-3)
    # one side's gradient, one weight's, fp32 weights beside bf16 heads
    qb, kb = q.bfloat16().requires_grad_(), k.bfloat16().requires_grad_()
    wq, wk = w.clone().requires_grad_(), w.clone().requires_grad_()
    yq, yk = qk_norm_rotary(qb, kb, wq, wk, tab)
    whole = torch.autograd.grad((yq, yk), (qb, kb, wq, wk), (yq.detach(), yk.detach()), retain_graph=True)
    assert [t.dtype for t in whole] == [torch.bfloat16, torch.bfloat16, torch.float32, torch.float32]
    part = torch.autograd.grad(yk, (kb, wk), yk.detach(), retain_graph=True)
    assert torch.equal(part[0], whole[1]) and torch.equal(part[1], whole[3])
    (only,) = torch.autograd.grad(qk_norm_rotary(qb.detach(), kb.detach(), wq, w, tab)[0], wq, yq.detach())
    assert torch.equal(only, whole[2])
    (dk,) = torch.autograd.grad(rotary(qb, kb, tab)[1], kb, yk.detach())
    assert dk.shape == kb.shape
    # weights of two types: both in fp32
    y2 = qk_norm_rotary(q, k, w.bfloat16(), w, tab)
    assert torch.equal(y2[1], base[1]) and torch.equal(y2[0], qk_norm_rotary(q, k, w.bfloat16().float(), w, tab)[0])


def test_nothing_to_turn():
    from dest3d_amd import qk_norm_rotary, rotary
    tab, w = table(9, 32).cuda(), torch.ones(32, device="cuda", requires_grad=True)
    for B, L, H, K in ((0, 5, 2, 1), (2, 0, 2, 1), (2, 5, 0, 1), (2, 5, 2, 0)):
        q, k = (torch.randn(B, L, h, 32, device="cuda", requires_grad=True) for h in (H, K))
        y = rotary(q, k, tab)
        assert y[0].shape == q.shape and y[1].shape == k.shape
        y = qk_norm_rotary(q, k, w, w, tab)
        (y[0].sum() + y[1].sum()).backward()
        assert q.grad.shape == q.shape and k.grad.shape == k.shape and torch.isfinite(w.grad).all()
        w.grad = None


def test_captured_streams_and_same_bits():
    from dest3d_amd import qk_norm_rotary
    d, dq, dk = make(2, 200, 4, 2, 64, 48, torch.bfloat16)
    g = {k: None if v is None else v.cuda() for k, v in d.items()}
    names = ("q", "k", "wq", "wk")
    for k in names:
        g[k].requires_grad_()
    cot = (dq.cuda(), dk.cuda())

    def step():
        y = qk_norm_rotary(g["q"], g["k"], g["wq"], g["wk"], g["table"], positions=g["pos"])
        return [*(t.detach() for t in y), *torch.autograd.grad(y, [g[k] for k in names], cot)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, step()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for turn in range(3):
        with torch.no_grad():
            for k in names:
                g[k].add_(0.05 * turn)
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_inputs_as_they_were():
    from dest3d_amd import qk_norm_rotary, rotary
    tab = table(9, 32).cuda()
    q = torch.randn(1, 9, 2, 32, device="cuda", requires_grad=True)
    w = torch.ones(32, device="cuda")
    x = q * 1.0
    y = qk_norm_rotary(x, None, w, None, tab)
    x.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    x = q * 1.0
    y = rotary(x, None, tab)
    x.mul_(2.0)               # (which the rotation's backward does not read)
    y.sum().backward()
    with pytest.raises(RuntimeError, match="first derivatives only"):
        torch.autograd.grad(rotary(q, None, tab).sum(), q, create_graph=True)


# ------------------------------------------------------------------------------------------------------------- together
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_layer_of_them(dtype):
    """Convolution, recurrence, turned and normalised C and B, the scan, the gated norm: a mixing layer on packed rows, forward and backward."""
    from dest3d_amd import ISSM_chunk_scan_combined, gated_scan, qk_norm_rotary, rmsnorm_fn, rotary_table
    from dest3d_amd.dwconv import dwconv_silu
    from oracle import issm_ref
    g = torch.Generator().manual_seed(0)
    B, L, H, P, N = 2, 140, 4, 16, 64
    C = H * P
    n = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    p = dict(u=n(B, L, C).to(dtype), cw=0.4 * n(C, 1, 7), cb=0.1 * n(C), gate=n(B, L, C).to(dtype), in_gate=n(B, L, C).to(dtype),
             Ag=-torch.rand(C, generator=g) - 0.05, Cq=n(B, L, 1, N).to(dtype), Bk=n(B, L, 1, N).to(dtype), wq=1 + 0.2 * n(N), wk=1 + 0.2 * n(N),
             dt=n(B, L, H, N).to(dtype), A=-torch.rand(H, N, generator=g) - 0.1, z=n(B, L, C).to(dtype), wn=1 + 0.2 * n(C))
    ids = torch.zeros(B, L, dtype=torch.long)
    ids[0, 50:], ids[1, 90:] = 1, 1
    pos = torch.stack([torch.cat([torch.arange(c), torch.arange(L - c)]) for c in (50, 90)])
    cot = n(B, L, C)
    tab = rotary_table(L, N, device="cpu")

    d = {k: v.cuda().requires_grad_() for k, v in p.items()}
    (x,) = dwconv_silu(d["u"], [d["cw"]], [d["cb"]])
    h = gated_scan(x, d["gate"], d["Ag"], in_gate=d["in_gate"], seq_idx=ids.cuda())
    c, b = qk_norm_rotary(d["Cq"], d["Bk"], d["wq"], d["wk"], tab.cuda(), positions=pos.cuda())
    y = ISSM_chunk_scan_combined(h.view(B, L, H, P), d["dt"], d["A"], b, c, 64, seq_idx=ids.cuda(), dt_softplus=True)
    out = rmsnorm_fn(y.reshape(B, L, C), d["wn"], None, z=d["z"], norm_before_gate=False)
    grads = torch.autograd.grad(out, list(d.values()), cot.to(dtype).cuda())

    r = {k: v.double().requires_grad_() for k, v in p.items()}
    xr = torch.nn.functional.silu(torch.nn.functional.conv1d(r["u"].transpose(1, 2), r["cw"], r["cb"], padding=3, groups=C)).transpose(1, 2)
    hr, _ = R.gated_scan(xr, r["gate"], r["Ag"], r["in_gate"], seq_idx=ids)
    cr, br = (R.norm_rotary(r[a], r[w], tab.double(), pos, 1e-6) for a, w in (("Cq", "wq"), ("Bk", "wk")))
    ys = []
    for i, cut in enumerate((50, 90)):
        parts = [issm_ref.issm_scan_sequential(hr[i:i + 1, s].reshape(1, -1, H, P), r["dt"][i:i + 1, s], r["A"], br[i:i + 1, s], cr[i:i + 1, s], dt_softplus=True)[0]
                 for s in (slice(0, cut), slice(cut, L))]
        ys.append(torch.cat(parts, 1))
    v = torch.cat(ys).reshape(B, L, C) * torch.nn.functional.silu(r["z"])
    outr = v / torch.sqrt((v * v).mean(-1, keepdim=True) + 1e-6) * r["wn"]
    want = torch.autograd.grad(outr, list(r.values()), cot.to(dtype).double())
    # the scan's own bars: products of 16 bits in fp32 (1e-4, gradients 1e-3), operands rounded to bf16 in bf16 (2e-2, 5e-2)
    lim = (1e-4, 1e-3) if dtype == torch.float32 else (2e-2, 5e-2)
    rel = lambda a, b: ((a.double().cpu() - b).norm() / b.norm()).item()  # noqa: E731
    assert rel(out.detach(), outr.detach()) <= lim[0]
    for k, a, b_ in zip(d, grads, want):
        assert a.dtype == d[k].dtype and rel(a, b_) <= lim[1], (k, rel(a, b_))


def test_offsets_beyond_32_bits_and_many_tokens():
    from dest3d_amd import qk_norm_rotary, rotary
    far, tab, w = 2 ** 31 + 64, table(9, 64).cuda(), torch.ones(64, device="cuda")
    wide = torch.empty(far + 4096, dtype=torch.bfloat16, device="cuda")
    for shape, strides in (((1, 1, 2, 64), (0, 0, far, 1)), ((1, 2, 1, 64), (0, far, 64, 1)), ((2, 1, 1, 64), (far, 64, 64, 1))):
        q = wide.as_strided(shape, strides)
        q.copy_(torch.randn(shape))
        assert torch.equal(rotary(q, None, tab), rotary(q.contiguous(), None, tab))
        a, b = (t.detach().requires_grad_() for t in (q, q.contiguous()))
        grads = [torch.autograd.grad(qk_norm_rotary(t, None, w, None, tab), t, b.detach())[0] for t in (a, b)]
        assert torch.equal(*grads)
    # enough tokens of one head for several of them a wave
    case = make(3, 30000, 1, 1, 16, 16, torch.float32, rows=30000)
    for norm in (False, True):
        check(run(*case, norm, True), ref(*case, norm, True))


def test_refusals():
    from dest3d_amd import qk_norm_rotary, rotary
    q, k, tab, w = torch.zeros(2, 5, 4, 16, device="cuda"), torch.zeros(2, 5, 2, 16, device="cuda"), table(5, 16).cuda(), torch.ones(16, device="cuda")
    pos = torch.zeros(2, 5, dtype=torch.int32, device="cuda")
    for kw in (dict(q=q[0]), dict(k=k[:1]), dict(k=k[:, :4]), dict(k=k[..., :8]), dict(table=tab[:, :7]), dict(table=table(5, 18).cuda()), dict(table=tab[0]), dict(table=tab[:4]),
               dict(positions=pos[:, :4]), dict(positions=pos[:1]), dict(positions=pos[..., None]), dict(table=tab[:0], positions=pos)):
        with pytest.raises(ValueError):
            rotary(**{**dict(q=q, k=k, table=tab), **kw})
    for kw in (dict(q=q.long()), dict(k=k.int()), dict(table=tab.long()), dict(positions=pos.float()), dict(positions=pos.to(torch.int16))):
        with pytest.raises(TypeError):
            rotary(**{**dict(q=q, k=k, table=tab), **kw})
    for kw in (dict(k=k.cpu()), dict(table=tab.cpu()), dict(positions=pos.cpu())):
        with pytest.raises(RuntimeError, match="all operands must be on"):
            rotary(**{**dict(q=q, k=k, table=tab), **kw})
    with pytest.raises(AssertionError, match="no gradient"):
        rotary(q, k, tab.clone().requires_grad_())
    with pytest.raises(RuntimeError, match="1024"):
        rotary(torch.zeros(1, 1, 1, 1026, device="cuda"), None, tab)
    for kw in (dict(q_weight=w[:8]), dict(k_weight=w[None])):
        with pytest.raises(ValueError):
            qk_norm_rotary(**{**dict(q=q, k=k, q_weight=w, k_weight=w, table=tab), **kw})
    with pytest.raises(TypeError):
        qk_norm_rotary(q, k, w.long(), w, tab)


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("wide", ["q", "k"])
def test_sides_of_two_types(wide, norm):
    """A side in float32 beside one in bfloat16 is not rounded to the other's type."""
    d, dq, dk = make(2, 30, 4, 2, 64, 48, torch.bfloat16)
    d[wide] = torch.randn(d[wide].shape, generator=torch.Generator().manual_seed(4))
    check(run(d, dq.to(d["q"].dtype), dk.to(d["k"].dtype), norm, False), ref(d, dq, dk, norm, False))

def test_table_without_forward_derivative():
    import torch.autograd.forward_ad as fwAD
    from dest3d_amd import rotary
    q, tab = torch.zeros(1, 5, 2, 16, device="cuda"), table(5, 16).cuda()
    with fwAD.dual_level(), pytest.raises(AssertionError, match="no gradient"):
        rotary(q, None, fwAD.make_dual(tab, tab))


@pytest.mark.parametrize("norm,tokens", [(False, 2 ** 26 + 2 ** 20 + 8), (True, 2 ** 27 + 8)])
def test_more_waves_than_a_launch_has(norm, tokens):
    """Heads of 66 features, a wave for each or for two of them: rows below 2^31, in more launches than one."""
    from dest3d_amd import qk_norm_rotary, rotary
    tab, w = table(8, 2).cuda(), torch.rand(66, device="cuda")
    x = torch.randn(66, device="cuda").bfloat16()
    call = (lambda q, **kw: qk_norm_rotary(q, None, w, None, tab, **kw)) if norm else (lambda q, **kw: rotary(q, None, tab, **kw))
    want = call(x.expand(1, 8, 1, 66))[0, :, 0]
    pos = torch.arange(8, device="cuda", dtype=torch.int32).repeat(tokens // 8)
    y = call(x.expand(1, tokens, 1, 66), positions=pos)
    assert not torch.equal(want[1], want[2])
    for part in y.view(tokens // 8, 8, 66).split(2 ** 20):
        assert (part == want).all()
