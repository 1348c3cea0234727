"""Gated linear recurrence on B200: a scan over a sequence (with gradients) and its one-token step.

Per channel, with a decay and an input gate at every step (the mamba-cpu reference has no such
operator; it stands beside ``selective_scan_fn``, whose (batch, dim, seqlen) layout it shares):

    a_t = exp(A * sigmoid(decay_gate_t))
    h_t = a_t h_{t-1} + sqrt(1 - a_t^2) * sigmoid(input_gate_t) * u_t,     y_t = h_t

The gates, the root and the recurrence run in one kernel (``mb200_gated_scan_fwd`` /
``mb200_gated_scan_bwd`` in libmamba_b200.so), in float32 for every input dtype. Gradients are reverse
mode: a forward-mode tangent on any argument raises ``NotImplementedError``. Argument checks and the
autograd node are those of ``mamba_b200::gated_scan`` / ``::gated_step`` (csrc/torch_ops.cpp).
"""

import torch

from .. import _lib

_gated_scan = torch.ops.mamba_b200.gated_scan.default
_gated_step = torch.ops.mamba_b200.gated_step.default


@torch.library.register_fake("mamba_b200::gated_scan_fwd")
def _(u, decay_gate, input_gate, A, initial_state, seq_idx, save_states):
    batch, dim, seqlen = u.shape
    f32 = torch.float32
    # MB200_GATED_SCAN_STATES
    states = 4 + batch * dim * ((seqlen + 7 + _lib.GATED_SCAN_CHUNK - 1) // _lib.GATED_SCAN_CHUNK)
    return (u.new_empty((batch, dim, seqlen)), u.new_empty((batch, dim), dtype=f32),
            u.new_empty((states if save_states else 0,), dtype=f32))


@torch.library.register_fake("mamba_b200::gated_scan_bwd")
def _(u, decay_gate, input_gate, A, initial_state, seq_idx, chunk_states, dout, dlast_state):
    return (u.new_empty(u.shape), u.new_empty(u.shape), u.new_empty(u.shape), torch.empty_like(A),
            u.new_empty(u.shape[:2] if initial_state is not None else (0,), dtype=torch.float32))


@torch.library.register_fake("mamba_b200::gated_scan_update")
def _(state, u, decay_gate, input_gate, A):
    return u.new_empty(u.shape)


@torch.library.register_fake("mamba_b200::gated_scan_update_out")
def _(state, u, decay_gate, input_gate, A, new_state):
    return u.new_empty(u.shape)


def gated_linear_scan_fn(u, decay_gate, input_gate, A, initial_state=None, seq_idx=None, return_last_state=False):
    """Gated linear recurrence over a sequence.

        a_t = exp(A * sigmoid(decay_gate_t))
        h_t = a_t h_{t-1} + sqrt(1 - a_t^2) * sigmoid(input_gate_t) * u_t

    Every step's input has the factor sqrt(1 - a^2), the first one of a sequence included (there are layers that feed
    that one without it; scaling u at those steps by the factor's inverse, where it is not 0, gives them).

    u, decay_gate, input_gate: (batch, dim, seqlen), gates before their sigmoid; an input gate below -44, whose
        sigmoid is under 1e-19, counts as shut
    A: (dim,), not positive: the log of the decay at an open gate (a positive entry gives NaN)
    initial_state: (batch, dim), the state before the first step (zeros if None)
    seq_idx: (batch, seqlen) integers of 32 bits. Packs sequences into a row: a step whose id differs from the one
        before it starts from a zero state (initial_state belongs to the sequence that begins at step 0).
        Steps with a negative id are padding: their output and gradients are 0, what the inputs hold there
        is not used, and the state passes through them.
    Returns h: (batch, dim, seqlen) in u's dtype [, last_state: (batch, dim) float32, the state after
    the last step]. Differentiable in u, the gates, A and initial_state (once); a decay of exactly 1
    (A = 0 or a gate of -inf) takes gradient 0 through the root, whose slope is infinite there.

    Tensors whose rows are contiguous along seqlen are read in place; others are copied first. Calls may be
    captured into CUDA graphs; as with any autograd op, capture a backward pass while no eager graph of the
    same leaves is alive.
    """
    out, last = _gated_scan(u, decay_gate, input_gate, A, initial_state, seq_idx)
    return (out, last) if return_last_state else out


def gated_linear_scan_update(state, u, decay_gate, input_gate, A, out_state=None):
    """Single decode step of the gated linear recurrence (inference).

    state: (batch, dim), float32 or u's dtype, updated in place; or, with out_state given (shape and dtype
        of state), left as it is while the new state is written to out_state (a step that may be undone)
    u, decay_gate, input_gate: (batch, dim)
    A: (dim,)
    Returns h: (batch, dim) in u's dtype.
    """
    return _gated_step(state, u, decay_gate, input_gate, A, out_state)
