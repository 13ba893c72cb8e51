"""The work that the recurrence and the position rotation are measured on.

Four operators of ``dest3d_amd``:

* ``recurrence``  ``gated_scan``: a state of one number for each channel, decayed by a gate and fed by the input, over a whole sequence;
                  forward alone or forward + backward through autograd
* ``step``        ``gated_scan_step``: one token a row, the states kept in a pool
* ``qk``          ``qk_norm_rotary``: queries and keys normalised for each head and rotated by their positions, with or without gradients
* ``rotary``      ``rotary``: the rotation alone, in both layouts, of a whole head or its first features

With ``own`` false ``run`` computes the same in elementary tensor operations in 32 bits, rounded once at the end.  Every input is made on
the GPU from the seed."""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}
MOST_TRAIN, MOST_INFER, MOST_HEADS = 8 * 4096 * 2048, 131072 * 2048, 65536 * 20 * 128     # values of the largest listed cases


# ---------------------------------------------------------------------------------------------------------------- cases
def _recurrence(name, **kw):
    case = dict(name=name, kind="recurrence", train=False, dtype="bf16", batch=1, seqlen=1024, channels=2048, in_gate=True, normalize=True,
                packed=0, initial=True, reverse=False, fused=False)
    case.update(kw)
    return case


def _heads(name, kind, **kw):
    case = dict(name=name, kind=kind, train=False, dtype="bf16", batch=1, seqlen=1024, heads=16, kv_heads=4, headdim=128, rot=128,
                interleaved=False, rows=32768, ragged=False, fused=False, base=10000.0, stretch=1.0)
    case.update(kw)
    return case


def listed():
    return [
        # evaluation of two scenes of 1000 tokens at the decoder's width: no size fills a tile; latency
        _recurrence("recurrence_infer_small_fp32", dtype="fp32", batch=2, seqlen=1000, channels=288),
        # training on packed rows: sequences of different lengths in each, an odd width, fp32
        _recurrence("recurrence_train_packed_fp32", train=True, dtype="fp32", batch=4, seqlen=5001, channels=801, packed=7),
        # training of a layer of 2048 channels
        _recurrence("recurrence_train_bf16", train=True, batch=8, seqlen=4096),
        # a prompt of 131072 tokens, one row, the three inputs side by side as one projection leaves them
        _recurrence("recurrence_prefill_long_bf16", seqlen=131072, fused=True),
        # serving one sequence, token by token
        dict(name="step_one_bf16", kind="step", dtype="bf16", batch=1, channels=2048, slots=1, indexed=False, in_gate=True, normalize=True),
        # serving 512 sequences whose states are spread over a pool
        dict(name="step_pool_bf16", kind="step", dtype="bf16", batch=512, channels=4096, slots=1024, indexed=True, in_gate=True,
             normalize=True),
        # one token of each of 64 sequences at positions of their own, queries and keys as slices of one projection
        _heads("qk_decode_bf16", "qk", batch=64, seqlen=1, heads=32, kv_heads=8, ragged=True, fused=True),
        # a prompt of 16384 tokens
        _heads("qk_prefill_bf16", "qk", seqlen=16384, heads=32, kv_heads=8, fused=True),
        # the scan's C and B (queries and keys of 256 states, one group) in training, fp32
        _heads("qk_train_states_fp32", "qk", train=True, dtype="fp32", batch=8, heads=1, kv_heads=1, headdim=256, rot=256),
        # training with grouped heads
        _heads("qk_train_bf16", "qk", train=True, batch=4, seqlen=4096),
        # a context stretched to 65536 tokens, interleaved pairs, half of each head
        _heads("rotary_long_interleaved_bf16", "rotary", seqlen=65536, rot=64, interleaved=True, rows=65536, base=500000.0, stretch=4.0),
        # training with the detector's heads of 36 features, of which 24 are rotated
        _heads("rotary_train_odd_fp32", "rotary", train=True, dtype="fp32", batch=8, seqlen=1021, heads=8, kv_heads=8, headdim=36, rot=24),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_recurrence(rng):
    while True:
        case = _recurrence("", train=rng.random() < 0.5, dtype=rng.choice(("fp32", "bf16", "bf16")), batch=_log_int(rng, 1, 16),
                           seqlen=_log_int(rng, 1, 131072), in_gate=rng.random() < 0.8, normalize=rng.random() < 0.8,
                           packed=rng.choice((0, 0, 3, 12)), initial=rng.random() < 0.6, reverse=rng.random() < 0.2)
        # half of the widths are whole multiples of 64, the others are what they happen to be
        case["channels"] = 64 * _log_int(rng, 1, 64) if rng.random() < 0.5 else _log_int(rng, 48, 4096)
        case["fused"] = not case["train"] and rng.random() < 0.5
        size = case["batch"] * case["seqlen"] * case["channels"] * (2 if case["dtype"] == "fp32" else 1)
        if size <= (MOST_TRAIN if case["train"] else MOST_INFER):
            del case["name"]
            return case


def _draw_heads(rng, kind):
    while True:
        kv = rng.choice((1, 2, 4, 8))
        case = _heads("", kind, train=rng.random() < 0.5, dtype=rng.choice(("fp32", "bf16", "bf16")), batch=_log_int(rng, 1, 64),
                      seqlen=_log_int(rng, 1, 65536), kv_heads=kv, heads=kv * rng.choice((1, 2, 4)),
                      headdim=rng.choice((32, 36, 64, 64, 80, 96, 128, 128, 256, 2 * rng.randint(16, 128))), interleaved=rng.random() < 0.4,
                      rows=65536, ragged=rng.random() < 0.5, base=rng.choice((10000.0, 500000.0)), stretch=rng.choice((1.0, 1.0, 8.0)))
        case["rot"] = case["headdim"] if rng.random() < 0.6 else 2 * rng.randint(1, case["headdim"] // 2)
        case["fused"] = not case["train"] and rng.random() < 0.5
        size = case["batch"] * case["seqlen"] * (case["heads"] + kv) * case["headdim"] * (2 if case["dtype"] == "fp32" else 1)
        if size <= MOST_HEADS // (4 if case["train"] else 1):
            del case["name"]
            return case


def draw(rng):
    """The kinds in the proportion of the list."""
    pick = rng.random() * 12
    if pick < 4:
        return _draw_recurrence(rng)
    if pick < 6:
        batch = _log_int(rng, 1, 512)
        return dict(kind="step", dtype=rng.choice(("fp32", "bf16", "bf16")), batch=batch, channels=_log_int(rng, 48, 4096),
                    slots=batch + rng.randint(0, 512), indexed=rng.random() < 0.7, in_gate=rng.random() < 0.8, normalize=rng.random() < 0.8)
    return _draw_heads(rng, "qk" if pick < 10 else "rotary")


# --------------------------------------------------------------------------------------------------------------- inputs
class _Draws:
    """Seeded random tensors on the GPU."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(self, *sizes, dtype=torch.float32):
        return torch.randn(*sizes, generator=self.g, device="cuda", dtype=torch.float32).to(dtype)

    def uniform(self, *sizes, lo=0.0, hi=1.0):
        return lo + (hi - lo) * torch.rand(*sizes, generator=self.g, device="cuda", dtype=torch.float32)

    def whole(self, lo, hi, *sizes):
        return torch.randint(lo, hi, sizes, generator=self.g, device="cuda")


def _prepare_recurrence(case, d):
    B, L, C, t = case["batch"], case["seqlen"], case["channels"], DTYPES[case["dtype"]]
    state = dict(case=case)
    n = 3 if case["in_gate"] else 2
    if case["fused"]:
        wide = d.normal(B, L, n * C, dtype=t)
        parts = [wide[..., i * C:(i + 1) * C] for i in range(n)]
    else:
        parts = [d.normal(B, L, C, dtype=t) for _ in range(n)]
    state["x"], state["gate"] = parts[:2]
    state["in_gate"] = parts[2] if case["in_gate"] else None
    state["A"] = torch.log(d.uniform(C, lo=0.9, hi=0.999))           # a full gate leaves 0.9 to 0.999 of a state a token
    state["h0"] = d.normal(B, C) if case["initial"] else None
    state["ids"] = None
    if case["packed"]:                                               # cuts at random places; every row's first sequence has id 0
        cuts = d.whole(0, L, B, case["packed"])
        marks = torch.zeros(B, L, dtype=torch.int32, device="cuda").scatter_(1, cuts, 1)
        marks[:, 0] = 0
        state["ids"] = marks.cumsum(1).to(torch.int32)
    if case["train"]:
        state["dy"], state["dlast"] = d.normal(B, L, C, dtype=t), d.normal(B, C)
        state["leaves"] = [k for k in ("x", "gate", "in_gate", "A", "h0") if state[k] is not None]
        for k in state["leaves"]:
            state[k].requires_grad_()
    return state


def _prepare_step(case, d):
    B, C, t = case["batch"], case["channels"], DTYPES[case["dtype"]]
    state = dict(case=case, x=d.normal(B, C, dtype=t), gate=d.normal(B, C, dtype=t), in_gate=d.normal(B, C, dtype=t) if case["in_gate"] else None,
                 A=torch.log(d.uniform(C, lo=0.9, hi=0.999)), pool=d.normal(case["slots"], C), at=None)
    if case["indexed"]:                                              # slots in any order, each once
        state["at"] = torch.randperm(case["slots"], generator=d.g, device="cuda")[:B].to(torch.int32)
    else:
        state["pool"] = state["pool"][:B].contiguous()
    return state


def _prepare_heads(case, d):
    B, L, H, K, D, R, t = (case[k] for k in ("batch", "seqlen", "heads", "kv_heads", "headdim", "rot", "dtype"))
    t = DTYPES[t]
    state = dict(case=case)
    if case["fused"]:                                                # queries, keys and values of one projection
        wide = d.normal(B, L, H + 2 * K, D, dtype=t)
        state["q"], state["k"] = wide[:, :, :H], wide[:, :, H:H + K]
    else:
        state["q"], state["k"] = d.normal(B, L, H, D, dtype=t), d.normal(B, L, K, D, dtype=t)
    # a row for each position: the cosines of its R / 2 angles, then their sines; angles of far positions in 64 bits
    inverse = case["base"] ** (-torch.arange(0, R, 2, device="cuda", dtype=torch.float64) / R)
    angle = torch.arange(case["rows"], device="cuda", dtype=torch.float64)[:, None] / case["stretch"] * inverse
    state["table"] = torch.cat([angle.cos(), angle.sin()], 1).float()
    state["positions"] = None
    if case["ragged"] or L > case["rows"]:                           # every row goes on from a position of its own
        state["positions"] = (d.whole(0, max(1, case["rows"] - L + 1), B, 1) + torch.arange(L, device="cuda")).to(torch.int32)
    if case["kind"] == "qk":
        state["wq"], state["wk"] = (1.0 + 0.2 * d.normal(D)).to(t), (1.0 + 0.2 * d.normal(D)).to(t)
    if case["train"]:
        state["dq"], state["dk"] = d.normal(B, L, H, D, dtype=t), d.normal(B, L, K, D, dtype=t)
        state["leaves"] = [k for k in ("q", "k", "wq", "wk") if k in state]
        for k in state["leaves"]:
            state[k].requires_grad_()
    return state


def prepare(case, seed):
    d = _Draws(seed)
    return {"recurrence": _prepare_recurrence, "step": _prepare_step, "qk": _prepare_heads, "rotary": _prepare_heads}[case["kind"]](case, d)


# ------------------------------------------------------------------------------------------- the framework's own calls
def _own_recurrence(s):
    from dest3d_amd import gated_scan
    case = s["case"]
    y, last = gated_scan(s["x"], s["gate"], s["A"], in_gate=s["in_gate"], initial_states=s["h0"], seq_idx=s["ids"],
                         normalize=case["normalize"], reverse=case["reverse"], return_final_states=True)
    if not case["train"]:
        return {"y": y, "last": last}
    grads = torch.autograd.grad((y, last), [s[k] for k in s["leaves"]], (s["dy"], s["dlast"]))
    return {"y": y.detach(), "last": last.detach(), **{"d" + k: g for k, g in zip(s["leaves"], grads)}}


def _own_step(s):
    from dest3d_amd import gated_scan_step
    y = gated_scan_step(s["x"], s["gate"], s["A"], s["pool"], in_gate=s["in_gate"], state_indices=s["at"], normalize=s["case"]["normalize"])
    return {"y": y, "pool": s["pool"]}


def _own_heads(s):
    from dest3d_amd import qk_norm_rotary, rotary
    case = s["case"]
    if case["kind"] == "qk":
        q, k = qk_norm_rotary(s["q"], s["k"], s["wq"], s["wk"], s["table"], positions=s["positions"], eps=1e-6, interleaved=case["interleaved"])
    else:
        q, k = rotary(s["q"], s["k"], s["table"], positions=s["positions"], interleaved=case["interleaved"])
    if not case["train"]:
        return {"q": q, "k": k}
    grads = torch.autograd.grad((q, k), [s[n] for n in s["leaves"]], (s["dq"], s["dk"]))
    return {"q": q.detach(), "k": k.detach(), **{"d" + n: g for n, g in zip(s["leaves"], grads)}}


# ----------------------------------------------------------------------------------------------------------- plain form
def _doubled(a, b):
    """All states of h_t = a_t h_{t-1} + b_t along dimension 1, from nothing: after each of log2(L) turns every place has taken in twice as many
    tokens before it.  (A quotient of cumulative sums and products needs no turns, and leaves 32 bits within some hundred tokens.)"""
    h, a, step = b.clone(), a.clone(), 1
    while step < h.shape[1]:
        h[:, step:] = torch.addcmul(h[:, step:], a[:, step:], h[:, :-step])
        a[:, step:] = a[:, step:] * a[:, :-step]
        step *= 2
    return h


def _plain_gates(s):
    case = s["case"]
    x, r = s["x"].float(), torch.sigmoid(s["gate"].float())
    la = s["A"].float() * r
    beta = torch.sqrt(-torch.expm1(2 * la)) if case["normalize"] else torch.ones_like(la)
    si = torch.sigmoid(s["in_gate"].float()) if s["in_gate"] is not None else None
    u = x if si is None else si * x
    return x, r, la, beta, si, u


@torch.no_grad()
def _plain_recurrence(s):
    case = s["case"]
    walk = (lambda t: t.flip(1)) if case["reverse"] else (lambda t: t)
    x, r, la, beta, si, u = (None if t is None else walk(t) for t in _plain_gates(s))
    a, b = la.double().exp().float(), beta * u                       # (next to one, where a bias of the last place adds up over all that is remembered)
    keep = a
    if s["ids"] is not None:
        ids = walk(s["ids"])
        before = torch.cat([torch.zeros_like(ids[:, :1]), ids[:, :-1]], 1)
        keep = a * (ids == before)[..., None]
    first = b[:, :1] + (keep[:, :1] * s["h0"].float()[:, None] if s["h0"] is not None else 0.0)
    h = _doubled(keep, torch.cat([first, b[:, 1:]], 1))
    t = s["x"].dtype
    out = {"y": walk(h).to(t), "last": h[:, -1].clone()}
    if not case["train"]:
        return out
    # backwards: c_t = keep_t a_t (dy_t + c_{t+1}) is the same recurrence from the other end
    dy = walk(s["dy"].float())
    ahead = torch.cat([dy[:, :-1], dy[:, -1:] + s["dlast"][:, None]], 1)
    c = _doubled(keep.flip(1), (keep * ahead).flip(1)).flip(1)
    g = ahead
    g[:, :-1] += c[:, 1:]
    h0 = s["h0"].float() if s["h0"] is not None else torch.zeros_like(h[:, 0])
    dla = c * torch.cat([h0[:, None], h[:, :-1]], 1)
    if case["normalize"]:
        dla -= g * u * a * a / beta
    du = g * beta
    grads = {"x": du if si is None else du * si, "gate": dla * la * (1 - r), "A": (dla * r).sum((0, 1)), "h0": c[:, 0].clone()}
    if si is not None:
        grads["in_gate"] = du * x * si * (1 - si)
    for k in s["leaves"]:
        out["d" + k] = (walk(grads[k]) if grads[k].dim() == 3 else grads[k]).to(s[k].dtype)
    return out


@torch.no_grad()
def _plain_step(s):
    x, r, la, beta, si, u = _plain_gates(s)
    old = s["pool"] if s["at"] is None else s["pool"][s["at"].long()]
    h = la.exp() * old + beta * u
    if s["at"] is None:
        s["pool"].copy_(h)
    else:
        s["pool"][s["at"].long()] = h
    return {"y": h.to(s["x"].dtype), "pool": s["pool"]}


def _turn(v, cos, sin, interleaved):
    """v (B, L, H, D) rotated by (B | 1, L, 1, R / 2) cosines and sines."""
    half = cos.shape[-1]
    head, rest = v[..., :2 * half], v[..., 2 * half:]
    one, two = (head[..., 0::2], head[..., 1::2]) if interleaved else (head[..., :half], head[..., half:])
    new = (one * cos - two * sin, one * sin + two * cos)
    turned = torch.stack(new, -1).flatten(-2) if interleaved else torch.cat(new, -1)
    return torch.cat([turned, rest], -1)


def _angles(s):
    case = s["case"]
    rows = s["table"][:case["seqlen"]][None] if s["positions"] is None else s["table"][s["positions"].long()]
    cos, sin = rows.chunk(2, -1)
    return cos[:, :, None], sin[:, :, None]


@torch.no_grad()
def _plain_heads(s):
    case = s["case"]
    cos, sin = _angles(s)
    turn = case["interleaved"]
    out = {}
    for n in ("q", "k"):
        x = s[n].float()
        if case["kind"] == "qk":
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * s["w" + n].float()
        out[n] = _turn(x, cos, sin, turn).to(s[n].dtype)
    if not case["train"]:
        return out
    for n in ("q", "k"):
        dv = _turn(s["d" + n].float(), cos, -sin, turn)
        if case["kind"] == "qk":
            x = s[n].float()
            rstd = torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6)
            xh, dxh = x * rstd, dv * s["w" + n].float()
            out["dw" + n] = (dv * xh).sum((0, 1, 2)).to(s["w" + n].dtype)
            dv = rstd * (dxh - xh * (dxh * xh).mean(-1, keepdim=True))
        out["d" + n] = dv.to(s[n].dtype)
    return {k: out[k] for k in ["q", "k"] + ["d" + n for n in s["leaves"]]}


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"recurrence": _own_recurrence, "step": _own_step, "qk": _own_heads, "rotary": _own_heads}[kind](state)
    return {"recurrence": _plain_recurrence, "step": _plain_step, "qk": _plain_heads, "rotary": _plain_heads}[kind](state)


# ----------------------------------------------------------------------------------------------------------------- work
def work(case):
    """What a pass cannot do without: each input read once, each result written once (a backward pass reads the inputs again: they do not fit
    between the two), and the arithmetic of the formulas, an exponential or a root as one operation."""
    size = 2 if case["dtype"] == "bf16" else 4
    if case["kind"] in ("recurrence", "step"):
        n = case["batch"] * case["channels"]
        ins = 3 if case["in_gate"] else 2
        flops = 10 + (5 if case["in_gate"] else 0) + (4 if case["normalize"] else 0)
        if case["kind"] == "step":
            return {"bytes": n * ((ins + 1) * size + 8) + 4 * case["channels"], "flops": n * flops}
        e = n * case["seqlen"]
        total = {"bytes": e * (ins + 1) * size + 8 * n + 4 * case["channels"], "flops": e * flops}
        if case["packed"]:
            total["bytes"] += 4 * case["batch"] * case["seqlen"]
        if case["train"]:
            total["bytes"] += e * (2 * ins + 1) * size + 16 * n
            total["flops"] += e * (2 * flops + 10)
        return total
    tokens = case["batch"] * case["seqlen"]
    e = tokens * (case["heads"] + case["kv_heads"]) * case["headdim"]
    turned = tokens * (case["heads"] + case["kv_heads"]) * case["rot"]
    rows = 4 * case["rot"] * min(case["rows"], tokens if case["ragged"] else case["seqlen"])
    norm = case["kind"] == "qk"
    total = {"bytes": 2 * e * size + rows, "flops": 3 * turned + (4 * e if norm else 0)}
    if case["train"]:
        total["bytes"] += (3 if norm else 2) * e * size + rows
        total["flops"] += 3 * turned + (12 * e if norm else 0)
    return total


# ---------------------------------------------------------------------------------------------------------------- exact
def _exact_recurrence(case, s):
    """Token by token in 64 bits."""
    x, gate, A = s["x"].double(), s["gate"].double(), s["A"].double()
    L = case["seqlen"]
    r = 1 / (1 + torch.exp(-gate))
    la = r * A
    a = torch.exp(la)
    beta = torch.sqrt(-torch.expm1(2 * la)) if case["normalize"] else None
    si = 1 / (1 + torch.exp(-s["in_gate"].double())) if case["in_gate"] else None
    u = x * si if si is not None else x
    b = u * beta if beta is not None else u
    kept = a
    order = list(range(L))[::-1] if case["reverse"] else list(range(L))
    if s["ids"] is not None:
        cut = torch.zeros(case["batch"], L, dtype=torch.bool, device=x.device)
        along = s["ids"][:, order]
        cut[:, 0] = along[:, 0] != 0
        cut[:, 1:] = along[:, 1:] != along[:, :-1]
        kept = torch.where(cut[:, torch.tensor(order, device=x.device).argsort()][..., None], torch.zeros_like(a), a)
    h0 = s["h0"].double() if s["h0"] is not None else torch.zeros_like(x[:, 0])
    y, h = torch.empty_like(x), h0
    for t in order:
        h = torch.addcmul(b[:, t], kept[:, t], h, out=y[:, t])
    out = {"y": y, "last": h.clone()}
    if not case["train"]:
        return out
    dy, c = s["dy"].double(), s["dlast"].double()
    g, carried = torch.empty_like(x), torch.empty_like(x)
    for t in order[::-1]:
        torch.add(dy[:, t], c, out=g[:, t])
        c = torch.mul(kept[:, t], g[:, t], out=carried[:, t])
    before = torch.empty_like(y)
    before[:, order[0]] = h0
    before[:, order[1:]] = y[:, order[:-1]]
    dla = carried * before
    if beta is not None:
        dla = dla - g * u * torch.exp(2 * la) / beta
        du = g * beta
    else:
        du = g
    grads = {"gate": dla * la * (1 - r), "A": (dla * r).sum((0, 1)), "h0": c.clone(), "x": du * si if si is not None else du}
    if si is not None:
        grads["in_gate"] = du * x * si * (1 - si)
    return {**out, **{"d" + k: grads[k] for k in s["leaves"]}}


def _exact_step(case, s):
    r = 1 / (1 + torch.exp(-s["gate"].double()))
    la = r * s["A"].double()
    b = s["x"].double()
    if case["in_gate"]:
        b = b / (1 + torch.exp(-s["in_gate"].double()))
    if case["normalize"]:
        b = b * torch.sqrt(-torch.expm1(2 * la))
    pool = s["pool"].double()
    at = torch.arange(case["batch"], device=pool.device) if s["at"] is None else s["at"].long()
    y = torch.exp(la) * pool[at] + b
    pool[at] = y
    return {"y": y, "pool": pool}


def _exact_heads(case, s):
    """As complex numbers: pair j of a head times cos + i sin."""
    R = case["rot"]
    at = torch.arange(case["seqlen"], device="cuda")[None] if s["positions"] is None else s["positions"].long()
    z = torch.complex(s["table"][:, :R // 2].double(), s["table"][:, R // 2:].double())[at].unsqueeze(2)

    def turned(v, z):
        w = v.clone()
        one, two = (slice(0, R, 2), slice(1, R, 2)) if case["interleaved"] else (slice(0, R // 2), slice(R // 2, R))
        p = torch.complex(v[..., one], v[..., two]) * z
        w[..., one], w[..., two] = p.real, p.imag
        return w

    out = {}
    for n in ("q", "k"):
        x = s[n].detach().double()
        scale = 1.0
        if case["kind"] == "qk":
            rms = torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6)
            scale = s["w" + n].detach().double() / rms
        out[n] = turned(x * scale, z)
        if case["train"]:
            dv = turned(s["d" + n].double(), z.conj())
            if case["kind"] == "qk":
                out["dw" + n] = (dv * x / rms).sum((0, 1, 2))
                out["d" + n] = dv * scale - x * (dv * scale * x).mean(-1, keepdim=True) / rms.square()
            else:
                out["d" + n] = dv
    return {k: out[k] for k in ["q", "k"] + (["d" + n for n in s["leaves"]] if case["train"] else [])}


@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "recurrence":
        return _exact_recurrence(case, s)
    return _exact_step(case, s) if case["kind"] == "step" else _exact_heads(case, s)
