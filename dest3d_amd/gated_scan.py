"""Gated linear recurrence on MI355X: a state of one number for each channel, beside the scan whose state is a matrix for each head.

``gated_scan`` runs it over whole sequences (forward and backward), ``gated_scan_step`` one token of each sequence at a time.  Checks,
argument blocks, allocation and the autograd node are compiled (csrc/host_ops.cpp); all arithmetic runs in libissm_hip.so."""
from __future__ import annotations

from . import _lib as L


def gated_scan(x, gate, A, in_gate=None, initial_states=None, seq_idx=None, normalize=True, reverse=False, return_final_states=False):
    """
    r = sigmoid(gate), a = exp(A r), u = sigmoid(in_gate) x (x without in_gate), h_t = a_t h_{t-1} + sqrt(1 - a_t^2) u_t

    Argument:
        x: (batch, seqlen, channels), float32 or bfloat16 (other types are computed in float32 and returned in their
            own; so is all of a call whose x, gate and in_gate are not all bfloat16)
        gate: (batch, seqlen, channels), before the sigmoid
        A: (channels,) logarithm of the decay at a full gate, <= 0 (see normalize)
        in_gate: (batch, seqlen, channels), before the sigmoid, or None
        initial_states: (batch, channels) or None
        seq_idx: (batch, seqlen) integer ids (compared as int32) of the sequences packed into a row, or None.  Every change of id is a cut that nothing
            passes; initial_states count as id 0, as in ISSM_chunk_scan_combined.
        normalize: without it u_t enters as it is, and A may be positive: states that grow are right as long as they, every decay, and what four
            neighbouring decays multiply a state other than 0 by, stay within float32
        reverse: from the last token to the first; initial_states and the final states are then behind and before the row
    Return:
        h: (batch, seqlen, channels)  [, final_states (batch, channels) fp32]

    Rows of at most 2^30 tokens; batch * ceil(channels / 64) below 2^22, and that times ceil(seqlen / 28) below 2^24.
    First derivatives for x, gate, A, in_gate and initial_states.  Where nothing decays (a = 1) the root of
    ``normalize`` has no derivative: its part of the gradients of gate and A is taken as 0 there.
    """
    res = L.host().gated_scan(x, gate, A, in_gate, initial_states, seq_idx, bool(normalize), bool(reverse), bool(return_final_states))
    return (res[0], res[1]) if return_final_states else res[0]


def gated_scan_step(x, gate, A, state, in_gate=None, state_indices=None, normalize=True):
    """One token of gated_scan for each row; no gradients.  rows * ceil(channels / 1024) below 2^23.

    Argument:
        x, gate, in_gate: (rows, channels), A: (channels,)
        state: (slots, channels) float32, updated in place; it shares no memory with the others
        state_indices: (rows,) int32 or int64, the slot of each row, or None: row r has slot r.  A row whose index is outside the
            slots (-1, say) gives zeros and touches no state; rows of one slot are taken in their order, as its tokens one
            behind the other.
    Return:
        h: (rows, channels)
    """
    return L.host().gated_scan_step(x, gate, A, state, in_gate, state_indices, bool(normalize))
