"""What stands between two blocks of a model on MI355X: the norm behind the first, its gate, the residual with its scale and
the norm before the second, in one pass over the rows, with gradients (``qsrt_residual_norm`` and
``qsrt_residual_norm_backward`` in ``include/qsrt_amd.h``).  Norms are by the root of the mean square.  Forward and backward can
be captured in a graph; graphs that eager calls built of the same leaves have to be freed before that."""

from __future__ import annotations

import math

import torch

from . import _native
from .packed_linear import TYPES, aligned_rows, refuse_second_derivatives, refuse_tangents

MAX_CHANNELS = 1 << 14
MAX_ROWS = 1 << 22
_NONE, _CHANNEL, _ROW = range(3)


def _vector(v: torch.Tensor | None) -> torch.Tensor | None:
    if v is None:
        return None
    return v.clone(memory_format=torch.contiguous_format) if v.data_ptr() % 16 or not v.is_contiguous() else v


def _checked(residual, y, weight, post, gate, dtype, eps):
    if residual.dim() != 2 or not residual.is_cuda:
        raise ValueError("rows must be [T, hidden] on a CUDA device")
    t, hidden = residual.shape
    if dtype not in TYPES or residual.dtype not in (torch.float32, dtype):
        raise ValueError("rows must be bfloat16 or float16; the residual may be float32")
    if not 0 < hidden <= MAX_CHANNELS or hidden % 8 or t > MAX_ROWS:
        raise ValueError(f"hidden must be a multiple of 8 up to {MAX_CHANNELS}, and at most {MAX_ROWS} rows")
    if y is not None and (y.shape != residual.shape or y.device != residual.device):
        raise ValueError("y must be [T, hidden] on the residual's device")
    if weight.dtype not in (torch.float32, dtype):
        raise ValueError("weights and gate must be float32 or of the rows' type")
    for v in (weight, post, gate):
        if v is not None and (v.dtype != weight.dtype or v.device != residual.device):
            raise ValueError("weights and gate must be of one type and on the rows' device")
    if weight.shape != (hidden,) or (post is not None and post.shape != (hidden,)):
        raise ValueError("weights must be [hidden]")
    kind = _NONE
    if gate is not None:
        if gate.shape == (hidden,):
            kind = _CHANNEL
        elif gate.shape == (t, 1):
            kind = _ROW
        else:
            raise ValueError("gate must be [hidden] or [T, 1]")
    if not (eps >= 0 and math.isfinite(eps)):
        raise ValueError("eps must be finite and not negative")
    return kind


def _like(t: torch.Tensor, dtype: torch.dtype | None = None) -> torch.Tensor:
    return torch.empty_like(t, dtype=dtype, memory_format=torch.contiguous_format)


def _at(t):
    return (None, 0) if t is None else (t.data_ptr(), t.stride(0))


def _ptr(t):
    return None if t is None else t.data_ptr()


def _forward(residual, y, weight, post, gate, kind, scale, eps, dtype, total, stats):
    normed = _like(residual, dtype)
    t, hidden = residual.shape
    if t == 0:
        return normed
    with _native.current(residual.device):
        _native.check(
            _native.lib().qsrt_residual_norm(
                *_at(residual), int(residual.dtype == torch.float32), *_at(y), TYPES[dtype], t, hidden, weight.data_ptr(),
                _ptr(post), _ptr(gate), kind, int(weight.dtype == torch.float32), scale, eps, *_at(total), *_at(normed),
                _ptr(stats), _native.stream_handle(residual.device)),
            "qsrt_residual_norm",
        )
    return normed


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, residual, y, weight, post, gate, kind, scale, eps, dtype, with_sum):
        ctx.set_materialize_grads(False)
        residual, y, weight = aligned_rows(residual), None if y is None else aligned_rows(y), _vector(weight)
        post, gate = _vector(post), _vector(gate)
        total = _like(residual) if with_sum else None
        stats = torch.empty((2, residual.shape[0]), dtype=torch.float32, device=residual.device)
        normed = _forward(residual, y, weight, post, gate, kind, scale, eps, dtype, total, stats)
        ctx.save_for_backward(residual, y, weight, post, gate, stats)
        ctx.kind, ctx.scale, ctx.dtype = kind, scale, dtype
        return total, normed

    @staticmethod
    def backward(ctx, dsum, dn):
        refuse_second_derivatives()
        refuse_tangents(dsum, dn)
        residual, y, weight, post, gate, stats = ctx.saved_tensors
        t, hidden = residual.shape
        if dsum is None and dn is None:
            return (None,) * 10
        grads = [_like(v) if needed else None for v, needed in zip((residual, y, weight, post, gate), ctx.needs_input_grad)]
        if t == 0:
            return *(None if g is None else g.zero_() for g in grads), *(None,) * 5
        dsum, dn = (None if d is None else aligned_rows(d) for d in (dsum, dn))
        lib = _native.lib()
        with _native.current(residual.device):
            ws = torch.empty(lib.qsrt_residual_norm_backward_workspace_bytes(t, hidden), dtype=torch.uint8,
                             device=residual.device)
            _native.check(
                lib.qsrt_residual_norm_backward(
                    *_at(dsum), *_at(dn), *_at(residual), int(residual.dtype == torch.float32), *_at(y), TYPES[ctx.dtype], t,
                    hidden, weight.data_ptr(), _ptr(post), _ptr(gate), ctx.kind, int(weight.dtype == torch.float32), ctx.scale,
                    stats.data_ptr(), *_at(grads[0]), *_at(grads[1]), _ptr(grads[2]), _ptr(grads[3]), _ptr(grads[4]),
                    ws.data_ptr(), ws.numel(), _native.stream_handle(residual.device)),
                "qsrt_residual_norm_backward",
            )
        return *grads, *(None,) * 5


def _run(residual, y, weight, post, gate, scale, eps, dtype, with_sum):
    refuse_tangents(residual, y, weight, post, gate)
    kind = _checked(residual, y, weight, post, gate, dtype, eps)
    leaves = [v for v in (residual, y, weight, post, gate) if v is not None]
    if torch.is_grad_enabled() and any(v.requires_grad for v in leaves):
        return _ResidualNorm.apply(residual, y, weight, post, gate, kind, scale, eps, dtype, with_sum)
    residual, y = aligned_rows(residual), None if y is None else aligned_rows(y)
    total = _like(residual) if with_sum else None
    return total, _forward(residual, y, _vector(weight), _vector(post), _vector(gate), kind, scale, eps, dtype, total, None)


def residual_norm(residual: torch.Tensor, y: torch.Tensor, weight: torch.Tensor, *, post_weight: torch.Tensor | None = None,
                  gate: torch.Tensor | None = None, scale: float = 1.0, eps: float = 1e-6):
    """``(h, n)`` with ``z = post_weight * y / rms(y)`` (without ``post_weight``: ``y``), ``h = scale * residual + gate * z``
    and ``n = weight * h / rms(h)``, ``rms(v) = sqrt(mean(v^2) + eps)`` over a row.

    ``y [T, hidden]``, a block's result, and ``n``, the next block's input, are bf16 or f16; ``residual`` and ``h`` float32 or
    of that type.  ``weight`` and ``post_weight [hidden]`` and ``gate`` (``[hidden]``, or ``[T, 1]``: each row its own) are all
    float32 or all of ``y``'s type.  ``n`` comes from ``h`` before it is rounded.  Differentiable in all five tensors, once and
    backward.  Squares are summed in FP32: a row's rms may be up to 1e17 and, with an eps of 0, down to 1e-18."""

    return _run(residual, y, weight, post_weight, gate, float(scale), float(eps), y.dtype, True)


def rms_norm(x: torch.Tensor, weight: torch.Tensor, *, eps: float = 1e-6, dtype: torch.dtype | None = None) -> torch.Tensor:
    """``weight * x / rms(x)``, what stands before the first block.  ``x [T, hidden]`` bf16, f16, or float32 with the result's
    ``dtype`` (bf16 or f16) named.  Differentiable in both, once and backward."""

    return _run(x, None, weight, None, None, 1.0, float(eps), x.dtype if dtype is None else dtype, False)[1]


__all__ = ["residual_norm", "rms_norm"]
