"""A gated feed-forward block in dense weights on MI355X, with its gradients: the expert before it is encoded, a shared expert
beside packed ones, a layer that is trained.

``gated_ffn`` is differentiable; ``gated_ffn_gradients`` returns, beside the gradients, the rows they are products of
(``qsrt_gated_ffn`` and ``qsrt_gated_ffn_backward`` in ``include/qsrt_amd.h``).  Nothing waits for the device, workspaces come
from torch's allocator on the current stream.  Forward and backward can be captured in a graph; graphs that eager calls built of
the same leaves have to be freed before that.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _native
from .packed_linear import TYPES, aligned_rows, checked_out, checked_rows, refuse_second_derivatives, refuse_tangents

ACTIVATIONS = {"swiglu": 0, "situ": 1}
MAX_CHANNELS = 1 << 17


def _checked(x, gate, up, down, activation):
    refuse_tangents(x, gate, up, down)
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {tuple(ACTIVATIONS)}")
    shape, dtype, device = gate.shape, gate.dtype, gate.device
    if len(shape) != 2 or up.shape != shape or down.shape != shape[::-1]:
        raise ValueError("gate and up must be [inter, hidden] and down [hidden, inter]")
    if dtype not in TYPES or device.type != "cuda":
        raise ValueError("the weights must be bfloat16 or float16 on a CUDA device")
    if up.dtype != dtype or down.dtype != dtype or up.device != device or down.device != device:
        raise ValueError("the weights must be of one type and on one device")
    inter, hidden = shape
    if not 0 < hidden <= MAX_CHANNELS or not 0 < inter <= MAX_CHANNELS or hidden % 8 or inter % 8:
        raise ValueError(f"hidden and inter must be multiples of 8 up to {MAX_CHANNELS}")
    if x.dtype != dtype or x.device != device:
        raise ValueError("x must be of the weights' type and on their device")
    x, gate, up, down = checked_rows(x, hidden, device), *(aligned_rows(w) for w in (gate, up, down))
    if gate.stride(0) != up.stride(0):  # one leading dimension serves both
        gate, up = gate.contiguous(), up.contiguous()
    return x, gate, up, down


def _forward(x, gate, up, down, activation, out, pre):
    t, hidden = x.shape
    inter = gate.shape[0]
    lib = _native.lib()
    with _native.current(x.device):
        ws = torch.empty(lib.qsrt_gated_ffn_workspace_bytes(t, hidden, inter), dtype=torch.uint8, device=x.device)
        _native.check(
            lib.qsrt_gated_ffn(
                x.data_ptr(), x.stride(0), gate.data_ptr(), up.data_ptr(), gate.stride(0), down.data_ptr(), down.stride(0),
                TYPES[x.dtype], t, hidden, inter, ACTIVATIONS[activation], None if pre is None else pre.data_ptr(),
                None if out is None else out.data_ptr(), 0 if out is None else out.stride(0), ws.data_ptr(), ws.numel(),
                _native.stream_handle(x.device)),
            "qsrt_gated_ffn",
        )


def _backward(dy, x, gate, up, down, activation, pre, dx, weights, rows):
    t, hidden = x.shape
    inter = gate.shape[0]
    lib = _native.lib()
    with _native.current(x.device):
        ws = torch.empty(lib.qsrt_gated_ffn_backward_workspace_bytes(t, hidden, inter), dtype=torch.uint8, device=x.device)
        _native.check(
            lib.qsrt_gated_ffn_backward(
                dy.data_ptr(), dy.stride(0), x.data_ptr(), x.stride(0), gate.data_ptr(), up.data_ptr(), gate.stride(0),
                down.data_ptr(), down.stride(0), TYPES[x.dtype], t, hidden, inter, ACTIVATIONS[activation], pre.data_ptr(),
                None if dx is None else dx.data_ptr(), hidden, *(None if w is None else w.data_ptr() for w in weights),
                *(None if r is None else r.data_ptr() for r in rows), ws.data_ptr(), ws.numel(),
                _native.stream_handle(x.device)),
            "qsrt_gated_ffn_backward",
        )


def _like(t: torch.Tensor, needed: bool = True) -> torch.Tensor | None:
    return torch.empty_like(t, memory_format=torch.contiguous_format) if needed else None


class _GatedFFN(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, up, down, activation):
        x, gate, up, down = _checked(x, gate, up, down, activation)
        y = _like(x)
        pre = torch.empty((2, x.shape[0], gate.shape[0]), dtype=torch.float32, device=x.device)
        if x.shape[0]:
            _forward(x, gate, up, down, activation, y, pre)
        ctx.save_for_backward(x, gate, up, down, pre)
        ctx.activation = activation
        return y

    @staticmethod
    def backward(ctx, dy):
        refuse_second_derivatives()
        refuse_tangents(dy)
        x, gate, up, down, pre = ctx.saved_tensors
        grads = [_like(t, needed) for t, needed in zip((x, gate, up, down), ctx.needs_input_grad)]
        if x.shape[0]:
            _backward(checked_rows(dy, x.shape[1], x.device), x, gate, up, down, ctx.activation, pre, grads[0], grads[1:],
                      (None, None, None))
        else:
            for g in grads[1:]:
                if g is not None:
                    g.zero_()
        return *grads, None


def gated_ffn(x: torch.Tensor, gate: torch.Tensor, up: torch.Tensor, down: torch.Tensor, *, activation: str = "swiglu",
              out: torch.Tensor | None = None) -> torch.Tensor:
    """``act(x gate^T, x up^T) down^T -> [T, hidden]`` in ``x``'s type.

    ``x [T, hidden]``, ``gate``, ``up [inter, hidden]``, ``down [hidden, inter]``, all bf16 or all f16, hidden and inter
    multiples of 8.  ``activation``: ``"swiglu"`` (``silu(g) u``) or ``"situ"``.  Sums are FP32; the rows between the two
    products are held in ``x``'s type (f16: infinite over 65504, off by up to 2^-25 each under 2^-14), of 64 rows or less as two
    values each.  Differentiable in all four, once and backward; the backward pass keeps the rows before the activation in FP32
    (``8 T inter`` bytes) and scales f16 rows between its products by powers of two, so that small gradients keep their bits.
    ``out``: where the result goes, of a call without gradients."""

    if torch.is_grad_enabled() and any(t.requires_grad for t in (x, gate, up, down)):
        if out is not None:
            raise ValueError("out is for calls without gradients")
        return _GatedFFN.apply(x, gate, up, down, activation)
    x, gate, up, down = _checked(x, gate, up, down, activation)
    out = _like(x) if out is None else checked_out(out, x, x.shape[1])
    if out.data_ptr() % 16 or (out.stride(0) % 8 and out.shape[0] > 1):
        raise ValueError("out's rows must be 16-byte aligned")
    if x.shape[0]:
        _forward(x, gate, up, down, activation, out, None)
    return out


@dataclass(frozen=True)
class GatedFFNGradients:
    """``x [T, hidden]``, ``gate``, ``up [inter, hidden]``, ``down [hidden, inter]`` (None where not asked for), and the rows
    ``gate_rows`` (dG), ``up_rows`` (dU) and ``middle`` (M), ``[T, inter]``:  ``gate = gate_rows^T x``, ``up = up_rows^T x``,
    ``down = dy^T middle``, but for the rows' rounding to ``x``'s type (f16: 2^-25 each under 2^-14)."""

    x: torch.Tensor | None
    gate: torch.Tensor | None
    up: torch.Tensor | None
    down: torch.Tensor | None
    gate_rows: torch.Tensor
    up_rows: torch.Tensor
    middle: torch.Tensor


@torch.no_grad()
def gated_ffn_gradients(x: torch.Tensor, dy: torch.Tensor, gate: torch.Tensor, up: torch.Tensor, down: torch.Tensor, *,
                        activation: str = "swiglu", inputs: bool = True, weights: bool = True) -> GatedFFNGradients:
    """Gradients of ``sum(dy * gated_ffn(x, gate, up, down))`` without the graph: of ``x`` where ``inputs``, of the weights
    where ``weights``, and always the rows that a weight's gradient is the product of.  ``dy [T, hidden]`` in ``x``'s type."""

    refuse_tangents(dy)
    x, gate, up, down = _checked(x, gate, up, down, activation)
    if dy.shape != x.shape or dy.dtype != x.dtype or dy.device != x.device:
        raise ValueError("dy must have x's shape and type, on its device")
    dy = checked_rows(dy, x.shape[1], x.device)
    t, inter = x.shape[0], gate.shape[0]
    grads = [_like(x, inputs), *(_like(w, weights) for w in (gate, up, down))]
    rows = [torch.empty((t, inter), dtype=x.dtype, device=x.device) for _ in range(3)]
    if t:
        pre = torch.empty((2, t, inter), dtype=torch.float32, device=x.device)
        _forward(x, gate, up, down, activation, None, pre)
        _backward(dy, x, gate, up, down, activation, pre, grads[0], grads[1:], rows)
    elif weights:
        for g in grads[1:]:
            g.zero_()
    return GatedFFNGradients(*grads, *rows)


__all__ = ["GatedFFNGradients", "gated_ffn", "gated_ffn_gradients"]
