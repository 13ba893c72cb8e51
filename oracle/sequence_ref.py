"""The gated linear recurrence and the rotary positions from their definitions, token by token, in the type of the inputs (float64 in the
tests); differentiable."""
import torch


def gated_scan(x, gate, A, in_gate=None, initial_states=None, seq_idx=None, normalize=True, reverse=False):
    B, L, C = x.shape
    r = torch.sigmoid(gate)
    la = A * r
    u = x if in_gate is None else torch.sigmoid(in_gate) * x
    if normalize:
        u = u * torch.sqrt(-torch.expm1(2 * la))
    h = torch.zeros(B, C, dtype=x.dtype) if initial_states is None else initial_states
    before = torch.zeros(B, dtype=torch.long)
    ys = [None] * L
    for t in (range(L - 1, -1, -1) if reverse else range(L)):
        passed = la[:, t].exp() * h
        if seq_idx is not None:   # selected, not multiplied by 0: nothing passes, whatever it is
            passed = torch.where((seq_idx[:, t] == before)[:, None], passed, torch.zeros_like(passed))
            before = seq_idx[:, t]
        ys[t] = h = passed + u[:, t]
    return (torch.stack(ys, 1) if L else x.clone()), h


def rotary(x, table, positions=None, interleaved=False):
    """x (B, L, H, D); table (n, R); positions (B, L) or (L,) or None."""
    R = table.shape[1]
    rows = table[:x.shape[1]] if positions is None else table[positions.long()]
    if rows.dim() == 2:
        rows = rows[None]
    c, s = rows[:, :, None, :R // 2], rows[:, :, None, R // 2:]
    j = torch.arange(R // 2)
    one, two = (2 * j, 2 * j + 1) if interleaved else (j, j + R // 2)
    a, b = x[..., one], x[..., two]
    y = x.clone()
    y[..., one] = a * c - b * s
    y[..., two] = a * s + b * c
    return y


def norm_rotary(x, weight, table, positions=None, eps=1e-6, interleaved=False):
    return rotary(x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight, table, positions, interleaved)
