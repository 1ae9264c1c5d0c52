"""Products with packed trellis matrices on MI355X, with low-rank adapters.

A payload stands for ``W = diag(suh) H_L X H_R diag(svh)``; a product of a few rows with it reads the payload's bits and
nothing wider, by rotating the rows instead of the weights (``qsrt_adapter_linear`` in ``include/qsrt_amd.h``).
"""

from __future__ import annotations

import ctypes

import torch
from torch.autograd import forward_ad

from . import _native
from .decode import _check_lut

TYPES = {torch.bfloat16: 0, torch.float16: 1}
MAX_RANK = 128
RATES = (2, 3, 4)


def _records(record_bits, lead: tuple, rate_axis: str, k: int, n: int, words: int) -> tuple[list, int]:
    """Per key the table ``first word << 3 | rate`` of its records, and the rates that occur as bits."""

    axis, other = (k, n) if rate_axis == "k" else (n, k)
    rates = 0
    tables = []
    for bits in record_bits:
        bits = tuple(int(b) for b in bits)
        if len(bits) != axis // 128 or any(b not in RATES for b in bits):
            raise ValueError(f"record_bits must hold K2, K3 or K4 for each of the {axis // 128} records of the rate axis")
        cursor, table = 0, []
        for b in bits:
            table.append(cursor << 3 | b)
            rates |= 1 << b
            cursor += 8 * (other // 16) * 16 * b
        if cursor != words:
            raise ValueError(f"payload holds {words} words where its records need {cursor}")
        tables.append(table)
    if len(tables) not in (1, lead[0] if lead else 1):
        raise ValueError("record_bits must be one schedule, or one for each payload")
    return tables, rates


def refuse_tangents(*tensors) -> None:
    """For calls without forward-mode derivatives: a tensor with a tangent does not require a gradient, and the tangent would be
    dropped."""

    if getattr(forward_ad, "_current_level", 0) < 0:  # no tensor has one: 0.1 us, where asking each takes 0.6
        return
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise ValueError("there are no forward-mode derivatives here: an argument has a tangent")


def refuse_gradients(*tensors) -> None:
    """Packed products have no backward pass: better no result than one that a gradient silently stops at."""

    refuse_tangents(*tensors)
    for t in tensors:
        if t is not None and t.requires_grad and torch.is_grad_enabled():
            raise ValueError("packed products have no backward pass: call them under torch.no_grad() or detach their inputs")


def refuse_second_derivatives() -> None:
    """For a backward pass that is not differentiable itself: better no gradient than one that a graph silently stops at."""

    if torch.is_grad_enabled():  # create_graph=True
        raise RuntimeError("there are no second derivatives here: call the backward pass without create_graph")


def _aligned(t: torch.Tensor, size: int) -> torch.Tensor:
    """``t`` in one piece at a multiple of ``size`` bytes, copied where it is not."""

    t = t.contiguous()
    return t.clone() if t.data_ptr() % size else t


class PackedMatrix:
    """One payload, or those of several keys (a layer's experts), ready for products.

    ``trellis`` int16: record-major words ``[words]`` or ``[keys, words]``, or the uniform ``[K/16, N/16, 16 bits]``
    tensor of ``quantize_qsrt`` (then ``record_bits`` is its rate).  ``suh``/``svh`` float16 ``[K]``/``[N]``, shared by
    all keys, or with a leading axis of keys.  ``record_bits``: one rate, one schedule for all keys, or one for each."""

    def __init__(self, trellis: torch.Tensor, suh: torch.Tensor, svh: torch.Tensor, record_bits, *, rate_axis: str = "k",
                 keys: int | None = None):
        if not trellis.is_cuda:
            raise ValueError("packed products run on the GPU; move the payload to a CUDA device")
        if rate_axis not in ("k", "n"):
            raise ValueError("rate_axis must be 'k' or 'n'")
        if trellis.dtype != torch.int16 or suh.dtype != torch.float16 or svh.dtype != torch.float16:
            raise ValueError("a payload holds int16 words and float16 scales")
        if suh.device != trellis.device or svh.device != trellis.device:
            raise ValueError("words and scales must be on one device")
        lead = () if keys is None else (keys,)
        if keys is not None and (keys < 1 or trellis.dim() < 2 or trellis.shape[0] != keys):
            raise ValueError("the payloads' leading axis must be the keys")
        for s in (suh, svh):
            if s.dim() not in (1, len(lead) + 1) or (s.dim() == 2 and s.shape[0] != keys):
                raise ValueError("scales must be one vector, or one for each key")
        refuse_gradients(suh, svh)
        k, n = suh.shape[-1], svh.shape[-1]
        if k == 0 or n == 0 or k % 128 or n % 128:
            raise ValueError("packed products need K and N multiples of 128")
        if isinstance(record_bits, int):
            rest = trellis.shape[len(lead):]
            if len(rest) == 3 and rest != (k // 16, n // 16, 16 * record_bits):
                raise ValueError("words must be int16 [K/16, N/16, 16 * bits]")
            if len(rest) == 3 and rate_axis != "k":
                raise ValueError("tiles in row-major order are records along k")
            record_bits = (record_bits,) * ((k if rate_axis == "k" else n) // 128)
        elif trellis.dim() != len(lead) + 1:
            raise ValueError("record-major words must be [words] or [keys, words]")
        nested = len(record_bits) > 0 and not isinstance(record_bits[0], int)
        trellis = _aligned(trellis.reshape(*lead, -1), 4)
        tables, rates = _records(record_bits if nested else [record_bits], lead, rate_axis, k, n, trellis.shape[-1])
        self.device, self.keys, self.k, self.n, self.rates = trellis.device, keys, k, n, rates
        self.words, self.suh, self.svh = trellis, _aligned(suh, 8), _aligned(svh, 8)
        self.records = torch.tensor(tables, dtype=torch.int64).to(self.device)
        self.struct = _native.PackedMatrixStruct(
            self.words.data_ptr(), trellis.shape[-1] if lead else 0, self.records.data_ptr(),
            len(tables[0]) if len(tables) > 1 else 0, self.suh.data_ptr(), k if suh.dim() == 2 else 0,
            self.svh.data_ptr(), n if svh.dim() == 2 else 0, k, n, 0 if rate_axis == "k" else 1, rates)
        self.ref = ctypes.addressof(self.struct)


class LabelTables:
    """The label tables of the rates in ``rates`` (bits), on ``device``."""

    def __init__(self, luts_by_bits: dict, rates: int, device):
        missing = [b for b in RATES if rates >> b & 1 and b not in luts_by_bits]
        if missing:
            raise ValueError(f"no label table for K{missing[0]}")
        self.tensors = {b: _check_lut(luts_by_bits[b], device) for b in RATES if rates >> b & 1}
        self.array = (ctypes.c_void_p * 3)(*[self.tensors[b].data_ptr() if b in self.tensors else None for b in RATES])
        self.ref = ctypes.addressof(self.array)


def aligned_rows(t: torch.Tensor) -> torch.Tensor:
    """``t [rows, cols]`` with whole rows at multiples of 16 bytes (copied where they are not)."""

    apart, step = t.stride()
    # (a lone row's stride says nothing: a view keeps whatever its base had)
    if step != 1 or t.data_ptr() % 16 or ((apart % 8 or apart < t.shape[1]) and t.shape[0] > 1):
        return t.clone(memory_format=torch.contiguous_format)
    return t


def checked_rows(x: torch.Tensor, cols: int, device) -> torch.Tensor:
    """``x`` as rows the kernels read: ``[rows, cols]``, rows 16-byte aligned (copied where they are not)."""

    if x.dim() != 2 or x.shape[1] != cols:
        raise ValueError(f"x must be [rows, {cols}]")
    if x.dtype not in TYPES:
        raise ValueError("x must be bfloat16 or float16")
    if x.device != device:
        raise ValueError("x must be on the payload's device")
    return aligned_rows(x)


def checked_out(out: torch.Tensor | None, x: torch.Tensor, cols: int) -> torch.Tensor:
    """``out``, or a new tensor.  A kernel writes it behind autograd's back: one that is part of a graph is refused, and a graph
    that has kept its values is told that they change, as it would be of torch's own calls."""

    if out is None:
        return torch.empty((x.shape[0], cols), dtype=x.dtype, device=x.device)
    if out.requires_grad and torch.is_grad_enabled():
        raise ValueError("out requires a gradient, and the call has no backward pass: detach it, or call under torch.no_grad()")
    refuse_tangents(out)
    if (out.shape != (x.shape[0], cols) or out.dtype != x.dtype or out.device != x.device or out.stride(1) != 1
            or out.data_ptr() % 8 or ((out.stride(0) % 4 or out.stride(0) < cols) and out.shape[0] > 1)):
        raise ValueError("out must be a row-major [rows, N] tensor of x's type, its rows 8-byte aligned")
    torch.autograd.graph.increment_version(out)
    return out


class PackedLinear:
    """A packed projection ``[K, N]`` with its label tables (``luts_by_bits[K]``: uint8[65536])."""

    def __init__(self, trellis: torch.Tensor, suh: torch.Tensor, svh: torch.Tensor, record_bits, luts_by_bits: dict, *,
                 rate_axis: str = "k"):
        self.matrix = PackedMatrix(trellis, suh, svh, record_bits, rate_axis=rate_axis)
        self.luts = LabelTables(luts_by_bits, self.matrix.rates, self.matrix.device)

    @classmethod
    def from_packed(cls, packed, suh: torch.Tensor, svh: torch.Tensor, luts_by_bits: dict) -> "PackedLinear":
        """From a mixed-rate ``PackedQSRTTrellis``."""

        from .qsrt import record_bits

        packed.validate()
        d = packed.descriptor
        return cls(packed.payload.reshape(-1), suh, svh, record_bits(d.mode), luts_by_bits, rate_axis=d.rate_axis)


class LowRankAdapters:
    """Adapters of one projection: ``a [adapters, r, K]``, ``b [adapters, N, r]`` (bf16 or f16), ``scale`` float32
    ``[adapters]`` (default 1).  Ranks that are no multiple of 16 are kept zero-padded: a later change of ``a`` or ``b``
    needs a new object."""

    def __init__(self, a: torch.Tensor, b: torch.Tensor, scale: torch.Tensor | None = None):
        if a.dim() != 3 or b.dim() != 3 or a.shape[0] != b.shape[0] or a.shape[1] != b.shape[2]:
            raise ValueError("adapters are a [adapters, r, K] and b [adapters, N, r]")
        if a.dtype not in TYPES or b.dtype != a.dtype or not a.is_cuda or b.device != a.device:
            raise ValueError("adapters must be bfloat16 or float16, both of one type, on a CUDA device")
        self.adapters, self.rank = a.shape[0], a.shape[1]
        if self.adapters < 1 or not 1 <= self.rank <= MAX_RANK:
            raise ValueError(f"at least one adapter, of a rank 1 .. {MAX_RANK}")
        if scale is None:
            scale = torch.ones(self.adapters, device=a.device)
        if scale.shape != (self.adapters,) or scale.dtype != torch.float32 or scale.device != a.device:
            raise ValueError("scale must be float32 [adapters] on the adapters' device")
        pad = -self.rank % 16
        self.a = _aligned(torch.nn.functional.pad(a, (0, 0, 0, pad)) if pad else a, 16)
        self.b = _aligned(torch.nn.functional.pad(b, (0, pad)) if pad else b, 16)
        self.scale = scale.contiguous()


def _run(x, linear, bank, ids, out):
    m = linear.matrix
    x = checked_rows(x, m.k, m.device)
    out = checked_out(out, x, m.n)
    rows = x.shape[0]
    if rows == 0:
        return out
    lib = _native.lib()
    adapters, rank = (bank.adapters, bank.a.shape[1]) if bank is not None else (0, 0)
    with _native.current(m.device):
        ws = torch.empty(lib.qsrt_adapter_linear_workspace_bytes(m.ref, rows, adapters, rank), dtype=torch.uint8,
                         device=m.device)
        _native.check(
            lib.qsrt_adapter_linear(
                m.ref, linear.luts.ref, None if bank is None else bank.a.data_ptr(),
                None if bank is None else bank.b.data_ptr(), None if bank is None else bank.scale.data_ptr(), adapters, rank,
                x.data_ptr(), x.stride(0), TYPES[x.dtype], rows, None if bank is None else ids.data_ptr(), out.data_ptr(),
                out.stride(0), ws.data_ptr(), ws.numel(), _native.stream_handle(m.device)),
            "qsrt_adapter_linear",
        )
    return out


def packed_linear(x: torch.Tensor, linear: PackedLinear, *, out: torch.Tensor | None = None) -> torch.Tensor:
    """``x [T, K] @ W -> [T, N]`` in ``x``'s type (bf16 or f16), FP32 sums.  No backward pass."""

    refuse_gradients(x)
    return _run(x, linear, None, None, out)


def adapter_linear(x: torch.Tensor, linear: PackedLinear, adapters: LowRankAdapters, ids: torch.Tensor, *,
                   out: torch.Tensor | None = None) -> torch.Tensor:
    """``x W + scale[a] (x A_a^T) B_a^T`` with ``a = ids[t]`` for row ``t``; an id outside ``[0, adapters)`` (-1) means
    none.  ``ids`` int32 ``[T]``, any order; one launch sequence serves all adapters.  No backward pass."""

    m = linear.matrix
    refuse_gradients(x, adapters.a, adapters.b, adapters.scale)
    if adapters.a.shape[2] != m.k or adapters.b.shape[1] != m.n:
        raise ValueError("the adapters do not match the projection")
    if adapters.a.dtype != x.dtype or adapters.a.device != m.device:
        raise ValueError("the adapters must be of x's type and on the payload's device")
    if ids.shape != x.shape[:1] or ids.dtype != torch.int32 or ids.device != m.device:
        raise ValueError("ids must be int32 [T] on the payload's device")
    return _run(x, linear, adapters, ids.contiguous(), out)


__all__ = ["LabelTables", "LowRankAdapters", "PackedLinear", "PackedMatrix", "adapter_linear", "packed_linear"]
