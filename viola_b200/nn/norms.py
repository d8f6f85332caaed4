"""RMS norms before and after a transformer block, fused with the block's gate and the residual scale.

``rms_norm_modulate(x, weight, scale)`` is the norm in front of a block, ``rms_norm_residual(x, y, weight, gate)`` what
follows it: the block's result ``y`` is normalised, gated and added to the scaled residual stream, and, with
``next_norm=True``, the new stream is normalised for the next block in the same pass::

    h = rms_norm_modulate(x, w_in, scale_in)
    x, h = rms_norm_residual(x, block(h), w_out, gate, next_norm=True, next_weight=w_in2, next_scale=scale_in2)

Each call is one kernel forward and one (plus a small one for the gradients of the vectors) backward; nothing but two
numbers per row is kept besides the inputs.  Vectors are [width] (shared by all rows) or [batch, width] with
``x`` [batch, ..., width] (one per sample, as an adaLN projection gives them).  CPU tensors take the same path through
the PyTorch restatement.  On the GPU the gradients cannot be differentiated again, and inputs with forward-mode tangents are
refused.
"""

from __future__ import annotations

from numbers import Real

import torch

from .. import ops

_DTYPES = (torch.float32, torch.bfloat16, torch.float16)
_FP32 = torch.finfo(torch.float32)


def _vector(v, x, name, samples=True):
    """Check an optional vector: [width], or with ``samples`` [batch, width]."""
    if v is None:
        return
    if v.dtype not in _DTYPES:
        raise TypeError(f"{name} must be float32, bfloat16 or float16, got {v.dtype}")
    if v.device != x.device:
        raise ValueError(f"{name} is on {v.device}, not on {x.device}")
    width = x.shape[-1]
    if v.shape == (width,) or (samples and x.dim() >= 2 and v.shape == (x.shape[0], width)):
        return
    shapes = f"({width},) or (batch, {width})" if samples else f"({width},)"
    raise ValueError(f"{name} must have shape {shapes} for x of shape {tuple(x.shape)}, got {tuple(v.shape)}")


def _call(x, y, weight, gate, next_weight, next_scale, residual_scale, eps, h_dtype):
    if not (type(residual_scale) is type(eps) is float or isinstance(residual_scale, Real) and isinstance(eps, Real)):
        raise ValueError(f"residual_scale and eps must be numbers, got {type(residual_scale).__name__} and {type(eps).__name__}")
    if x.is_cuda and x.numel():              # checked by the operator
        return ops.block_norm(x, y, weight, gate, next_weight, next_scale, residual_scale, eps, h_dtype)
    if y is not None:
        if y.shape != x.shape:
            raise ValueError(f"y must have the shape of x, got {tuple(y.shape)} and {tuple(x.shape)}")
        if y.dtype not in _DTYPES or x.dtype not in (torch.float32, y.dtype):
            raise TypeError(f"x must be float32 or have the dtype of y, got {x.dtype} and {y.dtype}")
        if y.device != x.device:
            raise ValueError(f"y is on {y.device}, not on {x.device}")
    width = x.shape[-1] if x.dim() else 0
    if not 1 <= width <= ops.MAX_NORM_WIDTH:
        raise ValueError(f"the width must be between 1 and {ops.MAX_NORM_WIDTH}, got x of shape {tuple(x.shape)}")
    if x.dtype not in _DTYPES:
        raise TypeError(f"x must be float32, bfloat16 or float16, got {x.dtype}")
    if not _FP32.tiny <= eps <= _FP32.max:
        raise ValueError(f"eps must be a positive fp32 number, got {eps}")
    if not abs(residual_scale) <= _FP32.max:
        raise ValueError(f"residual_scale must be a finite fp32 number, got {residual_scale}")
    _vector(weight, x, "weight", samples=False)
    _vector(next_weight, x, "weight" if y is None else "next_weight", samples=False)
    _vector(gate, x, "gate")
    _vector(next_scale, x, "scale" if y is None else "next_scale")
    inputs = (x, y, weight, gate, next_weight, next_scale)
    if x.numel() == 0:
        # nothing to compute, but the graph reaches every input
        empty = sum(t.sum() * 0 for t in inputs if t is not None and t.requires_grad)
        return ([x + empty] if y is not None else []) + ([(x + empty).to(h_dtype)] if h_dtype is not None else [])
    return ops.block_norm(*inputs, residual_scale, eps, h_dtype)


def rms_norm_modulate(x, weight=None, scale=None, *, eps=1e-6, dtype=None):
    """``x * (mean(x^2) + eps)^-1/2 * weight * (1 + scale)`` over the last dimension of ``x`` (at most 16384 wide).

    ``weight`` [width]; ``scale`` [width] or [batch, width].  The result has ``dtype`` (default: the autocast dtype where
    autocast is on and ``x`` is fp32, else ``x.dtype``); a 16-bit ``x`` keeps its dtype."""
    if dtype is None:
        dtype = x.dtype
        if x.is_cuda and x.dtype == torch.float32 and torch.is_autocast_enabled("cuda"):
            dtype = torch.get_autocast_dtype("cuda")
    if dtype not in _DTYPES or (x.dtype != torch.float32 and dtype != x.dtype):
        raise TypeError(f"cannot normalise {x.dtype} into {dtype}")
    return _call(x, None, None, None, weight, scale, 1.0, eps, dtype)[0]


def rms_norm_residual(x, y, weight=None, gate=None, *, residual_scale=1.0, eps=1e-6, next_norm=False, next_weight=None,
                      next_scale=None):
    """``residual_scale * x + gate * weight * y * (mean(y^2) + eps)^-1/2``: the norm after a block with its gate and the
    scaled residual connection.  ``x`` is fp32 or has the dtype of ``y``; the result has the dtype of ``x``.

    ``weight`` [width]; ``gate`` [width] or [batch, width].  With ``next_norm`` the result is ``(out, h)`` with
    ``h = out * (mean(out^2) + eps)^-1/2 * next_weight * (1 + next_scale)`` in the dtype of ``y``, taken from ``out`` before
    it is rounded: the input of the next block."""
    if not next_norm and (next_weight is not None or next_scale is not None):
        raise ValueError("next_weight and next_scale need next_norm=True")
    results = _call(x, y, weight, gate, next_weight, next_scale, residual_scale, eps, y.dtype if next_norm else None)
    return tuple(results) if next_norm else results[0]
