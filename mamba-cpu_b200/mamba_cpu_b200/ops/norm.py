"""Layer norm, RMS norm (with the residual sum fused in) and gated RMS norm on B200, with gradients.

The norms around a mixer: ``layer_norm_fn`` / ``rms_norm_fn`` before it, on the residual stream;
``gated_rms_norm_fn`` behind its scan. The mamba-cpu reference leaves them to PyTorch; here each is
one kernel forward and one (plus the reduction of the weight's gradient over the rows) backward,
``mb200_norm_fwd`` / ``mb200_norm_bwd`` in libmamba_b200.so. Arithmetic is float32 for every input
dtype. Gradients are reverse mode: a forward-mode tangent on any argument raises ``NotImplementedError``.
Argument checks and the autograd nodes are those of ``mamba_b200::norm`` / ``::gated_norm``
(csrc/torch_ops.cpp).
"""

import torch

from .. import _lib  # noqa: F401  (loads the ops)

_norm = torch.ops.mamba_b200.norm.default
_gated_norm = torch.ops.mamba_b200.gated_norm.default


@torch.library.register_fake("mamba_b200::norm_fwd")
def _(x, residual, z, weight, bias, eps, group_size, rms, gate, want_sum):
    total = x.new_empty(0) if residual is None else x.new_empty(x.shape if want_sum else (0,), dtype=residual.dtype)
    return x.new_empty(x.shape), total


@torch.library.register_fake("mamba_b200::norm_bwd")
def _(dout, dsum, rows, z, weight, residual_dtype, bias_dtype, eps, group_size, rms, gate, want_dresidual,
      want_dweight=True):
    dim, io = dout.shape[-1:], dout.dtype
    own_dres = want_dresidual and residual_dtype is not None and residual_dtype != io
    own_dw = weight is not None and want_dweight
    return (dout.new_empty(dout.shape),
            dout.new_empty(dout.shape if own_dres else (0,), dtype=residual_dtype if own_dres else io),
            dout.new_empty(dout.shape if z is not None else (0,)),
            dout.new_empty(dim if own_dw else (0,), dtype=weight.dtype if own_dw else io),
            dout.new_empty(dim if bias_dtype is not None else (0,), dtype=bias_dtype or io))


def layer_norm_fn(x, weight, bias=None, residual=None, eps=1e-5, prenorm=False, residual_in_fp32=False):
    """Layer norm over the last dimension of s = x + residual:
    (s - mean(s)) / sqrt(var(s) + eps) * weight + bias.

    x: (..., dim), dim <= 16384; weight, bias: (dim,) or None; residual: x's shape or None
    The sum s is held in x's dtype where the residual has it too, else (or with residual_in_fp32) in
    float32; what is normalised is s as held.
    Returns (..., dim) in x's dtype, with prenorm=True also s, the residual of the next block (without a
    residual: x itself, in float32 with residual_in_fp32). Differentiable (once) in every tensor.

    eps is 1e-5 unless given. mamba_ssm's functions of these names take 1e-6: a call ported from there has to say so.
    """
    out, total = _norm(x, weight, bias, residual, eps, prenorm, residual_in_fp32, False)
    return (out, total) if prenorm else out


def rms_norm_fn(x, weight, bias=None, residual=None, eps=1e-5, prenorm=False, residual_in_fp32=False):
    """RMS norm over the last dimension of s = x + residual: s / sqrt(mean(s^2) + eps) * weight + bias.
    Arguments and results are those of :func:`layer_norm_fn`."""
    out, total = _norm(x, weight, bias, residual, eps, prenorm, residual_in_fp32, True)
    return (out, total) if prenorm else out


def gated_rms_norm_fn(x, z, weight, eps=1e-5, group_size=None, norm_before_gate=False):
    """RMS norm with a SiLU gate, over the last dimension or over groups of ``group_size`` of its columns.

    norm_before_gate=False: v / sqrt(mean(v^2) + eps) * weight with v = x * silu(z)
    norm_before_gate=True:  x / sqrt(mean(x^2) + eps) * weight * silu(z)

    x, z: (..., dim); weight: (dim,) or None; group_size divides dim (default dim) and is at most 16384.
    Returns (..., dim) in x's dtype. Differentiable (once) in x, z and weight.

    The gate comes first unless told otherwise, as in transformers' Mamba-2 mixer, and eps is 1e-5. ``hf.mamba_split_conv1d_scan_combined``, which has
    mamba_ssm's signature, normalises first and with eps 1e-6 unless told otherwise, and passes both on: calls ported
    from there have to say norm_before_gate=True and eps=1e-6.
    """
    return _gated_norm(x, z, weight, eps, group_size, norm_before_gate)
