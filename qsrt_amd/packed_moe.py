"""A mixture-of-experts layer for a few tokens, straight from its packed payloads.

``route_tokens`` chooses each token's experts, ``PackedExperts`` multiplies by them and ``PackedMoELayer`` is both
(``qsrt_route``, ``qsrt_packed_moe`` and ``qsrt_packed_moe_layer`` in ``include/qsrt_amd.h``).  Nothing waits for the
device: which experts are chosen is known there alone.  Workspaces come from torch's allocator on the current stream, so a
call can be captured in a graph (after one outside it, which loads the kernels).

Longer batches are taken too, but an expert's rows share a decode of its weights 64 at a time at the most: from about a
thousand rows an expert on, decoding its matrices once (``decode``) and a library product are faster.
"""

from __future__ import annotations

import torch

from . import _native
from .packed_linear import TYPES, LabelTables, PackedMatrix, checked_out, checked_rows, refuse_gradients
from .qsrt_coupled import CoupledHadamardSpec, rotation_signs

SCORING = {"softmax": 0, "sigmoid": 1}
ACTIVATIONS = {"swiglu": 0, "situ": 1}
MAX_EXPERTS = 1024
MAX_CHOSEN = 64


def _checked_router(weight: torch.Tensor, k: int, bias, scoring: str) -> tuple:
    if weight.dim() != 2 or not weight.is_cuda or weight.dtype not in TYPES:
        raise ValueError("the router's weight must be bfloat16 or float16 [experts, hidden] on a CUDA device")
    e, h = weight.shape
    if not 1 <= e <= MAX_EXPERTS or h == 0 or h % 8:
        raise ValueError(f"the router takes 1 .. {MAX_EXPERTS} experts and a multiple of 8 channels")
    if isinstance(k, bool) or not isinstance(k, int) or not 1 <= k <= min(MAX_CHOSEN, e):
        raise ValueError(f"k must be 1 .. {min(MAX_CHOSEN, e)}")
    if scoring not in SCORING:
        raise ValueError(f"scoring must be one of {tuple(SCORING)}")
    if bias is not None and (bias.shape != (e,) or bias.dtype != torch.float32 or bias.device != weight.device):
        raise ValueError("bias must be float32 [experts] on the router's device")
    if weight.stride(1) != 1 or weight.data_ptr() % 16 or ((weight.stride(0) % 8 or weight.stride(0) < h) and e > 1):
        weight = weight.clone(memory_format=torch.contiguous_format)
    return weight, None if bias is None else bias.contiguous()


def _route(x, weight, k, bias, scoring, normalize, scale):
    e, h = weight.shape
    if x.dtype != weight.dtype:
        raise ValueError("x must be of the router's type")
    x = checked_rows(x, h, weight.device)
    t = x.shape[0]
    weights = torch.empty((t, k), dtype=torch.float32, device=x.device)
    ids = torch.empty((t, k), dtype=torch.int32, device=x.device)
    if t == 0:
        return weights, ids
    lib = _native.lib()
    with _native.current(x.device):
        ws = torch.empty(lib.qsrt_route_workspace_bytes(t, h, e), dtype=torch.uint8, device=x.device)
        _native.check(
            lib.qsrt_route(x.data_ptr(), x.stride(0), weight.data_ptr(), weight.stride(0), TYPES[x.dtype], t, h, e,
                           k, None if bias is None else bias.data_ptr(), SCORING[scoring], int(normalize), float(scale),
                           weights.data_ptr(), ids.data_ptr(), ws.data_ptr(), ws.numel(), _native.stream_handle(x.device)),
            "qsrt_route",
        )
    return weights, ids


def route_tokens(x: torch.Tensor, weight: torch.Tensor, k: int, *, bias: torch.Tensor | None = None,
                 scoring: str = "softmax", normalize: bool = True, scale: float = 1.0):
    """The ``k`` experts of each row of ``x [T, hidden]``: ``(weights float32 [T, k], ids int32 [T, k])``.

    Scores are the softmax or the sigmoid of ``x weight^T`` (``weight [experts, hidden]``, of ``x``'s type).  The largest
    ``score + bias`` (without a bias: the largest logits) are chosen, ties to the lowest index, NaN last, and returned in
    falling order; their weights are the scores without the bias, divided by their sum where ``normalize``, times
    ``scale``.  No backward pass."""

    refuse_gradients(x, weight, bias)
    weight, bias = _checked_router(weight, k, bias, scoring)
    return _route(x, weight, k, bias, scoring, normalize, scale)


class PackedExperts:
    """The experts of one layer: ``w1`` and ``w3 [hidden, inter]`` (gate and up) and ``w2 [inter, hidden]`` (down), each a
    dict of the stacked payloads of all experts: ``trellis`` int16 ``[experts, words]``, ``suh``/``svh`` float16 (one
    vector for the layer or ``[experts, ...]``), ``record_bits`` (one rate, one schedule, or one for each expert) and
    ``rate_axis`` (default: columns for w1 and w3, rows for w2, as stored).  ``activation``: the model's, ``"swiglu"`` or
    ``"situ"``.  ``coupled``: the payloads hold coupled coordinates (``qsrt_coupled.encode_coupled_weights``) of that spec,
    of its default block sizes; ``x`` and the result are in the source's coordinates all the same.  The activation has to
    be named then: execution and calibration in coupled coordinates take ``situ`` unless told otherwise, plain payloads here
    ``swiglu``."""

    def __init__(self, w1: dict, w3: dict, w2: dict, luts_by_bits: dict, *, activation: str | None = None,
                 coupled: CoupledHadamardSpec | None = None):
        if activation is None:
            if coupled is not None:
                raise ValueError(f"coupled experts need their activation named: one of {tuple(ACTIVATIONS)}")
            activation = "swiglu"
        if activation not in ACTIVATIONS:
            raise ValueError(f"activation must be one of {tuple(ACTIVATIONS)}")
        self.experts = int(w1["trellis"].shape[0])
        self.w1, self.w3, self.w2 = (
            PackedMatrix(w["trellis"], w["suh"], w["svh"], w["record_bits"], rate_axis=w.get("rate_axis", axis),
                         keys=self.experts)
            for w, axis in ((w1, "n"), (w3, "n"), (w2, "k")))
        self.hidden, self.inter, self.device = self.w1.k, self.w1.n, self.w1.device
        if ((self.w3.k, self.w3.n) != (self.hidden, self.inter) or (self.w2.k, self.w2.n) != (self.inter, self.hidden)
                or self.w3.device != self.device or self.w2.device != self.device):
            raise ValueError("w1, w3 [hidden, inter] and w2 [inter, hidden] do not match")
        if (self.w1.suh.dim() == 1) != (self.w3.suh.dim() == 1):
            raise ValueError("w1 and w3 must both share their suh, or neither")
        self.luts = LabelTables(luts_by_bits, self.w1.rates | self.w3.rates | self.w2.rates, self.device)
        self.activation = ACTIVATIONS[activation]
        self.signs, self.sign_pointers = (), (None, None)
        if coupled is not None:
            if (coupled.residual_block_size, coupled.preactivation_block_size, coupled.postactivation_block_size) != \
                    (512, 128, 128) or self.hidden % 512:
                raise ValueError("coupled experts need blocks of 512, 128 and 128 and a multiple of 512 hidden channels")
            self.signs = tuple(rotation_signs(n, draw=coupled.intermediate_draw, axis=axis, device=self.device)
                               for n, axis in ((2 * self.inter, 1), (self.inter, 2)))
            self.sign_pointers = tuple(s.data_ptr() for s in self.signs)

    @classmethod
    def from_experts(cls, experts: list, record_bits, luts_by_bits: dict, *, activation: str,
                     coupled: CoupledHadamardSpec | None = None, device="cuda:0") -> "PackedExperts":
        """From a list of ``{"w1", "w3", "w2"}`` dicts as a layer file's reader returns them (``read_expert``).  The file does
        not say which ``activation`` its layer was calibrated with, so the caller does."""

        def stack(name):
            def scale(part):
                all_ = torch.stack([e[name][part].reshape(-1) for e in experts])
                return (all_[0] if bool((all_ == all_[0]).all()) else all_).to(device)

            return {"trellis": torch.stack([e[name]["trellis"].reshape(-1) for e in experts]).to(device),
                    "suh": scale("suh"), "svh": scale("svh"), "record_bits": record_bits}

        if not experts:
            raise ValueError("a layer needs at least one expert")
        w1, w3, w2 = (stack(name) for name in ("w1", "w3", "w2"))
        if w1["suh"].dim() != w3["suh"].dim():  # both shared or neither
            for w in (w1, w3):
                w["suh"] = w["suh"].expand(len(experts), -1).contiguous()
        return cls(w1, w3, w2, luts_by_bits, activation=activation, coupled=coupled)

    def __call__(self, x: torch.Tensor, weights: torch.Tensor, ids: torch.Tensor, *,
                 out: torch.Tensor | None = None) -> torch.Tensor:
        """``out[t] = sum_j weights[t, j] act(x_t W1_e, x_t W3_e) W2_e`` with ``e = ids[t, j]``; an id outside
        ``[0, experts)`` (-1) contributes nothing.  ``x [T, hidden]`` bf16 or f16, ``weights`` float32 and ``ids`` int32
        ``[T, k]``.  No backward pass."""

        refuse_gradients(x, weights)
        x = checked_rows(x, self.hidden, self.device)
        out = checked_out(out, x, self.hidden)
        if (ids.dim() != 2 or ids.shape[0] != x.shape[0] or ids.shape[1] < 1 or weights.shape != ids.shape
                or ids.dtype != torch.int32 or weights.dtype != torch.float32 or ids.device != self.device
                or weights.device != self.device):
            raise ValueError("weights float32 and ids int32 must be [T, k] on the payload's device")
        t, k = ids.shape
        if t == 0:
            return out
        ids, weights = ids.contiguous(), weights.contiguous()
        lib = _native.lib()
        with _native.current(self.device):
            ws = torch.empty(lib.qsrt_packed_moe_workspace_bytes(self.w1.ref, self.w3.ref, self.w2.ref, self.experts, t, k),
                             dtype=torch.uint8, device=self.device)
            _native.check(
                lib.qsrt_packed_moe(self.w1.ref, self.w3.ref, self.w2.ref, self.luts.ref, self.experts, self.activation,
                                    *self.sign_pointers, x.data_ptr(), x.stride(0), TYPES[x.dtype], t, k, ids.data_ptr(),
                                    weights.data_ptr(), out.data_ptr(), out.stride(0), ws.data_ptr(), ws.numel(),
                                    _native.stream_handle(self.device)),
                "qsrt_packed_moe",
            )
        return out


class PackedMoELayer:
    """Router and packed experts of one layer; calling it on ``x [T, hidden]`` returns ``(y, weights, ids)``.  No backward
    pass."""

    def __init__(self, router: torch.Tensor, experts: PackedExperts, k: int, *, bias: torch.Tensor | None = None,
                 scoring: str = "softmax", normalize: bool = True, scale: float = 1.0):
        self.router, self.bias = _checked_router(router, k, bias, scoring)
        if self.router.shape != (experts.experts, experts.hidden) or self.router.device != experts.device:
            raise ValueError("the router's weight must be [experts, hidden] on the experts' device")
        self.experts, self.k, self.scoring, self.normalize, self.scale = experts, k, scoring, normalize, scale

    def __call__(self, x: torch.Tensor, *, out: torch.Tensor | None = None):
        e = self.experts
        refuse_gradients(x, self.router, self.bias)
        if x.dtype != self.router.dtype:
            raise ValueError("x must be of the router's type")
        x = checked_rows(x, e.hidden, e.device)
        out = checked_out(out, x, e.hidden)
        t, k = x.shape[0], self.k
        weights = torch.empty((t, k), dtype=torch.float32, device=e.device)
        ids = torch.empty((t, k), dtype=torch.int32, device=e.device)
        if t == 0:
            return out, weights, ids
        lib = _native.lib()
        with _native.current(e.device):
            ws = torch.empty(lib.qsrt_packed_moe_workspace_bytes(e.w1.ref, e.w3.ref, e.w2.ref, e.experts, t, k),
                             dtype=torch.uint8, device=e.device)
            _native.check(
                lib.qsrt_packed_moe_layer(
                    e.w1.ref, e.w3.ref, e.w2.ref, e.luts.ref, e.experts, e.activation, *e.sign_pointers,
                    self.router.data_ptr(),
                    self.router.stride(0), None if self.bias is None else self.bias.data_ptr(), SCORING[self.scoring],
                    int(self.normalize), float(self.scale), x.data_ptr(), x.stride(0), TYPES[x.dtype], t, k,
                    weights.data_ptr(), ids.data_ptr(), out.data_ptr(), out.stride(0), ws.data_ptr(), ws.numel(),
                    _native.stream_handle(e.device)),
                "qsrt_packed_moe_layer",
            )
        return out, weights, ids


__all__ = ["PackedExperts", "PackedMoELayer", "route_tokens"]
