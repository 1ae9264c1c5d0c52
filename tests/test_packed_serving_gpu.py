"""Router, packed experts and adapter projections against their definitions in float64 (the oracle's decode).

Tolerances.  A product's rotated rows are two bf16 pieces (error at most 2^-17 of each value), its sums FP32 over at most a
few hundred steps (2^-24 each); the activation between two products has a relative slope under 4.  Together they stay
under 2^-14 of the result's 2-norm, beside the one rounding to the output's type (at most 2^-8 of each value in bf16, 2^-11 plus the
subnormal step in f16, and half of that in 2-norm).  Single values may lie off by that rounding and 2^-11 of the root mean
square of their row's result.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import fmt
from qsrt_amd import qsrt as Q
from qsrt_amd.decode import decode_packed
from qsrt_amd.exl3_reference import reconstruct_trellis_states
from qsrt_amd.packed_linear import LowRankAdapters, PackedLinear, adapter_linear, packed_linear
from qsrt_amd.packed_moe import PackedExperts, PackedMoELayer, route_tokens
from qsrt_amd.qsrt_coupled import CoupledHadamardSpec, decode_coupled_weights, rotation_signs
from qsrt_amd.sqg_e4m3 import sqg_xor_cheb_t12_bytes

pytestmark = pytest.mark.gpu

LUTS = {b: sqg_xor_cheb_t12_bytes(b) for b in (2, 3, 4)}
ROUND = {  # in 2-norm; a single value's rounding is up to twice that
    torch.bfloat16: 2.0**-9, torch.float16: 2.0**-12}


def payload(rng, k, n, record_bits, axis, svh=0.02):
    """Random words (every stream is a closed path) and scales of one matrix, and the matrix in float64."""

    other = (n if axis == "k" else k) // 16
    words = rng.integers(-32768, 32768, size=sum(8 * other * 16 * b for b in record_bits)).astype(np.int16)
    suh = (rng.uniform(0.5, 1.5, k) * rng.choice([-1, 1], k)).astype(np.float16)
    svh = (svh * rng.uniform(0.5, 1.5, n) * rng.choice([-1, 1], n)).astype(np.float16)
    return words, suh, svh


def dense(words, suh, svh, record_bits, axis):
    k, n = suh.size, svh.size
    states, bits = fmt.unpack_records(words, record_bits, axis, k // 16, n // 16)
    values = np.zeros(states.shape)
    for b, lut in LUTS.items():
        values = np.where((bits == b)[..., None], lut.view(torch.float8_e4m3fn).double().numpy()[states], values)
    return torch.from_numpy(fmt.decode_tile_values(values, suh.astype(np.float64), svh.astype(np.float64)))


def close(got, want, dtype):
    got, want = got.cpu().double(), want.double()
    assert got.shape == want.shape
    assert torch.equal(torch.isfinite(got), torch.isfinite(want))
    if want.numel() == 0 or not bool(want.abs().max() > 0):
        assert torch.equal(got, want)
        return
    step = 2.0**-25 if dtype == torch.float16 else 0.0
    rms = want.square().mean().sqrt()
    assert (got - want).norm() <= (ROUND[dtype] + 2.0**-14) * want.norm() + step * want.numel() ** 0.5
    row = want.square().mean(-1, keepdim=True).sqrt().clamp_min(rms * 2.0**-6)
    assert bool(((got - want).abs() <= 2 * ROUND[dtype] * want.abs() + 2.0**-11 * row + step).all())


def rows(rng, t, h, dtype):
    return torch.from_numpy(rng.standard_normal((t, h))).to(dtype)


# ---------------------------------------------------------------------------
# router
# ---------------------------------------------------------------------------


def choose64(x, w, k, bias, scoring, normalize, scale):
    logits = x.double() @ w.double().T
    score = torch.softmax(logits, -1) if scoring == "softmax" else torch.sigmoid(logits)
    key = logits if bias is None else score + bias.double()
    ids = torch.sort(key, dim=-1, descending=True, stable=True).indices[:, :k]
    weights = score.gather(1, ids)
    return (weights / weights.sum(-1, keepdim=True) if normalize else weights) * scale, ids


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("t,h,e,k,bias,dtype", [
    (1, 7168, 384, 8, True, torch.bfloat16), (17, 256, 8, 2, False, torch.float16), (3, 40, 1, 1, True, torch.bfloat16),
    (33, 1032, 129, 7, False, torch.bfloat16), (2, 8, 1024, 64, True, torch.float16), (16, 520, 16, 16, False, torch.float16),
])
def test_router(t, h, e, k, bias, dtype, scoring):
    rng = np.random.default_rng(t * h + e)
    x, w = rows(rng, t, h, dtype), rows(rng, e, h, dtype) / (2 if h < 64 else h**0.5)
    b = torch.from_numpy(rng.standard_normal(e) * 0.1).float() if bias else None
    got_w, got = route_tokens(x.cuda(), w.cuda(), k, bias=None if b is None else b.cuda(), scoring=scoring,
                              normalize=k != 7, scale=1.5)
    want_w, want = choose64(x, w, k, b, scoring, k != 7, 1.5)
    assert got.dtype == torch.int32 and torch.equal(got.cpu().long(), want)
    # exact products; FP32 sums of `h` terms of about one, then exp, sum and quotient in FP32
    assert torch.allclose(got_w.cpu().double(), want_w, rtol=2e-5, atol=0)


def test_router_ties_masks_and_nan():
    x = torch.ones((3, 64), dtype=torch.bfloat16)
    w = torch.zeros((70, 64), dtype=torch.bfloat16)
    w[5], w[66] = 1.0, 1.0
    _, ids = route_tokens(x.cuda(), w.cuda(), 4)
    assert ids.cpu().tolist() == [[5, 66, 0, 1]] * 3  # ties to the lowest index
    bias = torch.full((70,), -float("inf"))
    weights, ids = route_tokens(x.cuda(), w.cuda(), 3, bias=bias.cuda(), scoring="sigmoid", normalize=False)
    assert ids.cpu().tolist() == [[0, 1, 2]] * 3 and torch.equal(weights.cpu(), torch.full((3, 3), 0.5))
    bias[7] = 0.0
    _, ids = route_tokens(x.cuda(), w.cuda(), 2, bias=bias.cuda(), scoring="softmax")
    assert ids.cpu().tolist() == [[7, 0]] * 3
    w[5] = float("nan")
    _, ids = route_tokens(x.cuda(), w.cuda(), 3)
    assert ids.cpu().tolist() == [[66, 0, 1]] * 3
    x[1] = float("nan")
    _, ids = route_tokens(x.cuda(), w.cuda(), 3)
    assert ids.cpu().tolist()[1] == [0, 1, 2]
    assert route_tokens(x[:0].cuda(), w.cuda(), 3)[1].shape == (0, 3)


def test_router_takes_strided_rows():
    rng = np.random.default_rng(5)
    x, w = rows(rng, 9, 300, torch.bfloat16).cuda(), rows(rng, 12, 272, torch.bfloat16).cuda()
    want = route_tokens(x[:, 3:267].contiguous(), w[:, 8:].contiguous(), 3)
    got = route_tokens(x[:, 3:267], w[:, 8:], 3)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


# ---------------------------------------------------------------------------
# experts
# ---------------------------------------------------------------------------


class Experts:
    """Payloads of a small layer, and its experts in float64."""

    def __init__(self, seed, hidden, inter, experts, bits, shared=True, act="swiglu", axes=("n", "n", "k")):
        rng = np.random.default_rng(seed)
        self.mats, self.hidden, self.act = [], hidden, act
        stacked = []
        for (k, n), axis, local in zip(((hidden, inter), (hidden, inter), (inter, hidden)), axes, (2, 2, 1)):
            each = [payload(rng, k, n, bits[e] if isinstance(bits[0], tuple) else bits, axis) for e in range(experts)]
            if shared:  # the hidden side's scales
                each = [tuple(each[0][j] if j == 3 - local else v for j, v in enumerate(p)) for p in each]
            self.mats.append([dense(*p, bits[e] if isinstance(bits[0], tuple) else bits, axis) for e, p in enumerate(each)])

            def cat(j):
                return torch.from_numpy(each[0][j] if shared and j == 3 - local else np.stack([p[j] for p in each])).cuda()

            stacked.append({"trellis": cat(0), "suh": cat(1), "svh": cat(2), "record_bits": bits, "rate_axis": axis})
        self.packed = PackedExperts(*stacked, LUTS, activation=act)

    def __call__(self, x, weights, ids):
        x, y = x.double(), torch.zeros((x.shape[0], self.hidden), dtype=torch.float64)
        for t in range(ids.shape[0]):
            for j, e in enumerate(ids[t].tolist()):
                if not 0 <= e < len(self.mats[0]):
                    continue
                g, u = x[t] @ self.mats[0][e], x[t] @ self.mats[1][e]
                mid = (g * torch.sigmoid(g) * u if self.act == "swiglu" else
                       4 * torch.tanh(g / 4) * torch.sigmoid(g) * 25 * torch.tanh(u / 25))
                y[t] += float(weights[t, j]) * (mid @ self.mats[2][e])
        return y


@pytest.mark.parametrize("hidden,inter,experts,bits,shared,act,t,k,dtype", [
    (256, 512, 8, (2,) * 4, False, "swiglu", 1, 2, torch.bfloat16),
    (384, 256, 5, (3, 4), True, "situ", 7, 3, torch.float16),
    (128, 384, 3, (2, 3, 4), True, "swiglu", 40, 1, torch.bfloat16),   # three rates; chunks of two groups, ragged
    (128, 128, 2, (4,), False, "situ", 70, 2, torch.float16),          # chunks of four groups
    (640, 128, 16, (3,), True, "swiglu", 64, 4, torch.bfloat16),
    (128, 256, 1, (2, 4), True, "swiglu", 3, 5, torch.bfloat16),       # one expert, chosen again and again
])
def test_experts(hidden, inter, experts, bits, shared, act, t, k, dtype):
    layer = Experts(hidden + inter, hidden, inter, experts, bits, shared, act)
    rng = np.random.default_rng(t)
    x = rows(rng, t, hidden, dtype)
    ids = torch.from_numpy(rng.integers(-1, experts, (t, k))).int()
    weights = torch.from_numpy(rng.uniform(0.1, 1, (t, k))).float()
    close(layer.packed(x.cuda(), weights.cuda(), ids.cuda()), layer(x, weights, ids), dtype)


@pytest.mark.parametrize("axes", [("k", "k", "n"), ("k", "k", "k"), ("n", "n", "n")])
def test_experts_rates_along_the_other_axis(axes):
    bits = ((2, 3, 3, 4),) * 2 + ((4, 2, 3, 3),) + ((3, 3, 3, 3),)  # a schedule for each expert, equal lengths
    layer = Experts(11, 512, 512, 4, bits, False, axes=axes)
    rng = np.random.default_rng(12)
    x, ids = rows(rng, 6, 512, torch.bfloat16), torch.from_numpy(rng.integers(0, 4, (6, 2))).int()
    weights = torch.from_numpy(rng.uniform(0.1, 1, (6, 2))).float()
    close(layer.packed(x.cuda(), weights.cuda(), ids.cuda()), layer(x, weights, ids), torch.bfloat16)


def test_experts_no_expert_no_token_and_bad_ids():
    layer = Experts(3, 128, 256, 4, (3, 3))
    rng = np.random.default_rng(4)
    x = rows(rng, 5, 128, torch.bfloat16)
    weights = torch.from_numpy(rng.uniform(0.1, 1, (5, 2))).float()
    ids = torch.tensor([[-1, -1], [0, -1], [4, 2], [1 << 30, -(1 << 31)], [3, 3]], dtype=torch.int32)
    got = layer.packed(x.cuda(), weights.cuda(), ids.cuda())
    close(got, layer(x, weights, ids), torch.bfloat16)
    assert not bool(got[0].any()) and not bool(got[3].any())
    none = layer.packed(x.cuda(), weights.cuda(), torch.full_like(ids, -1).cuda())
    assert not bool(none.any())
    assert layer.packed(x[:0].cuda(), weights[:0].cuda(), ids[:0].cuda()).shape == (0, 128)


def test_experts_strides_streams_and_repeats():
    layer = Experts(5, 256, 384, 6, (3, 3, 4))
    rng = np.random.default_rng(6)
    t, k = 11, 3
    wide = rows(rng, t, 300, torch.bfloat16).cuda()
    ids = torch.from_numpy(rng.integers(0, 6, (t, 2 * k))).int().cuda()[:, ::2]
    weights = torch.from_numpy(rng.uniform(0.1, 1, (k, t))).float().cuda().T
    x = wide[:, 1:257]
    want = layer(x.cpu(), weights.cpu(), ids.cpu())
    out = torch.full((t, 264), 7.0, dtype=torch.bfloat16, device="cuda")
    got = layer.packed(x, weights, ids, out=out[:, :256])
    assert got.data_ptr() == out.data_ptr() and bool((out[:, 256:] == 7).all())
    close(got, want, torch.bfloat16)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = layer.packed(x, weights, ids)
    stream.synchronize()
    assert torch.equal(other, got)  # the same bits whenever and wherever it runs
    # a token's result is its own: the same bits without its neighbours' tokens up to the cut of the sums
    close(layer.packed(x[4:5], weights[4:5], ids[4:5]), want[4:5], torch.bfloat16)


def test_experts_offsets_past_32_bits():
    hidden, inter, experts = 2048, 1024, 6000
    words = hidden * inter * 3 // 16
    assert words * experts > 1 << 31  # words; the bytes pass 32 bits too
    rng = np.random.default_rng(8)
    one = [payload(rng, *shape, (3,) * 8, axis) for shape, axis in
           (((hidden, inter), "n"), ((hidden, inter), "n"), ((inter, hidden), "k"))]
    stacked = []
    for p, axis in zip(one, ("n", "n", "k")):
        trellis = torch.zeros((experts, words), dtype=torch.int16, device="cuda")
        trellis[-1] = torch.from_numpy(p[0]).cuda()
        stacked.append({"trellis": trellis, "suh": torch.from_numpy(p[1]).cuda(), "svh": torch.from_numpy(p[2]).cuda(),
                        "record_bits": 3, "rate_axis": axis})
    packed = PackedExperts(*stacked, LUTS)
    mats = [dense(*p, (3,) * 8, axis) for p, axis in zip(one, ("n", "n", "k"))]
    x = rows(rng, 2, hidden, torch.bfloat16)
    ids = torch.tensor([[experts - 1], [-1]], dtype=torch.int32)
    got = packed(x.cuda(), torch.ones((2, 1)).cuda(), ids.cuda())
    g, u = x[:1].double() @ mats[0], x[:1].double() @ mats[1]
    close(got[:1], (g * torch.sigmoid(g) * u) @ mats[2], torch.bfloat16)
    assert not bool(got[1].any())


def test_layer_is_router_then_experts():
    experts = Experts(9, 256, 256, 12, (3, 4))
    rng = np.random.default_rng(10)
    x = rows(rng, 5, 256, torch.bfloat16)
    router = rows(rng, 12, 256, torch.bfloat16) / 16
    bias = torch.from_numpy(rng.standard_normal(12) * 0.1).float()
    layer = PackedMoELayer(router.cuda(), experts.packed, 4, bias=bias.cuda(), scoring="sigmoid", scale=2.5)
    y, weights, ids = layer(x.cuda())
    want_w, want = choose64(x, router, 4, bias, "sigmoid", True, 2.5)
    assert torch.equal(ids.cpu().long(), want)
    close(y, experts(x, want_w, want), torch.bfloat16)


def test_layer_in_a_graph():
    """Captured once, replayed on new rows with eager work in between."""

    experts = Experts(13, 256, 384, 6, (2, 3, 4))
    rng = np.random.default_rng(14)
    layer = PackedMoELayer((rows(rng, 6, 256, torch.bfloat16) / 16).cuda(), experts.packed, 2)
    x = rows(rng, 4, 256, torch.bfloat16).cuda()
    layer(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, weights, ids = layer(x)
    for _ in range(4):
        x.copy_(rows(rng, 4, 256, torch.bfloat16))
        want = layer(x)
        layer(x[:1].contiguous())
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want[0]) and torch.equal(weights, want[1]) and torch.equal(ids, want[2])


# ---------------------------------------------------------------------------
# adapters
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("t,k,n,bits,axis,adapters,rank,dtype", [
    (1, 256, 128, (2,) * 2, "k", 1, 1, torch.bfloat16),
    (1, 1024, 256, (3,) * 8, "k", 5, 16, torch.float16),
    (7, 384, 256, (2, 3, 4), "k", 3, 27, torch.bfloat16),
    (16, 128, 384, (4, 3, 3), "n", 2, 128, torch.float16),
    (31, 256, 256, (3, 4), "n", 40, 8, torch.bfloat16),
    (65, 128, 128, (4,), "k", 3, 33, torch.bfloat16),
    (200, 640, 128, (2,) * 5, "k", 1, 64, torch.float16),
    (129, 384, 256, (2, 4, 3), "k", 9, 16, torch.bfloat16),            # three rates, many rows
    (700, 512, 256, (3, 4), "n", 4, 40, torch.float16),
    (1030, 256, 128, (4, 4), "k", 2, 5, torch.bfloat16),
])
def test_adapters(t, k, n, bits, axis, adapters, rank, dtype):
    rng = np.random.default_rng(t + k + rank)
    p = payload(rng, k, n, bits, axis)
    linear = PackedLinear(*(torch.from_numpy(v).cuda() for v in p), bits, LUTS, rate_axis=axis)
    w = dense(*p, bits, axis)
    x = rows(rng, t, k, dtype)
    a = (rows(rng, adapters * rank, k, dtype) / k**0.5).view(adapters, rank, k)
    b = (rows(rng, adapters * n, rank, dtype) / rank**0.5).view(adapters, n, rank)
    scale = torch.from_numpy(rng.uniform(0.5, 2, adapters)).float()
    ids = torch.from_numpy(rng.integers(-1, adapters + 1, t)).int()
    base = x.double() @ w
    want = base.clone()
    for row, i in enumerate(ids.tolist()):
        if 0 <= i < adapters:
            want[row] += float(scale[i]) * ((x[row].double() @ a[i].double().T) @ b[i].double().T)
    bank = LowRankAdapters(a.cuda(), b.cuda(), scale.cuda())
    close(adapter_linear(x.cuda(), linear, bank, ids.cuda()), want, dtype)
    close(packed_linear(x.cuda(), linear), base, dtype)
    close(adapter_linear(x.cuda(), linear, bank, torch.full_like(ids, -1).cuda()), base, dtype)


def test_adapters_uniform_payload_strides_and_no_rows():
    rng = np.random.default_rng(21)
    k, n = 256, 384
    p = payload(rng, k, n, (3,) * 2, "k")
    words = torch.from_numpy(p[0]).view(k // 16, n // 16, 48).cuda()  # as quantize_qsrt leaves it
    linear = PackedLinear(words, *(torch.from_numpy(v).cuda() for v in p[1:]), 3, LUTS)
    wide = rows(rng, 19, 262, torch.bfloat16).cuda()
    out = torch.full((19, 400), 3.0, dtype=torch.bfloat16, device="cuda")
    got = packed_linear(wide[:, 5:261], linear, out=out[:, 8:392])
    close(got, wide[:, 5:261].cpu().double() @ dense(*p, (3,) * 2, "k"), torch.bfloat16)
    assert bool((out[:, :8] == 3).all()) and bool((out[:, 392:] == 3).all())
    bank = LowRankAdapters(torch.zeros((2, 3, k), dtype=torch.bfloat16).cuda(),
                           torch.zeros((2, n, 3), dtype=torch.bfloat16).cuda())
    empty = adapter_linear(wide[:0, :256].contiguous(), linear, bank, torch.empty(0, dtype=torch.int32, device="cuda"))
    assert empty.shape == (0, n)


def test_infinities_stay_in_their_row():
    rng = np.random.default_rng(23)
    p = payload(rng, 256, 128, (3, 3), "k")
    linear = PackedLinear(*(torch.from_numpy(v).cuda() for v in p), (3, 3), LUTS)
    x = rows(rng, 18, 256, torch.bfloat16)
    want = x.double() @ dense(*p, (3, 3), "k")
    x[3, 7], x[17, 200] = float("inf"), float("nan")
    got = packed_linear(x.cuda(), linear).cpu()
    keep = [r for r in range(18) if r not in (3, 17)]
    close(got[keep], want[keep], torch.bfloat16)
    assert not bool(torch.isfinite(got[[3, 17]]).any())


# ---------------------------------------------------------------------------
# refusals
# ---------------------------------------------------------------------------


def test_refusals():
    rng = np.random.default_rng(31)
    words, suh, svh = (torch.from_numpy(v).cuda() for v in payload(rng, 256, 128, (3, 4), "k"))
    linear = PackedLinear(words, suh, svh, (3, 4), LUTS)
    x = torch.zeros((2, 256), dtype=torch.bfloat16, device="cuda")
    ids = torch.zeros(2, dtype=torch.int32, device="cuda")
    for bad in (lambda: PackedLinear(words.cpu(), suh.cpu(), svh.cpu(), (3, 4), LUTS),
                lambda: PackedLinear(words, suh, svh, (3, 3), LUTS),          # another length
                lambda: PackedLinear(words, suh, svh, (3, 5), LUTS),
                lambda: PackedLinear(words, suh, svh, (3,), LUTS),
                lambda: PackedLinear(words, suh.float(), svh, (3, 4), LUTS),
                lambda: PackedLinear(words, suh[:100], svh, (3, 4), LUTS),
                lambda: PackedLinear(words, suh, svh, (3, 4), {3: LUTS[3]}),
                lambda: PackedLinear(words, suh, svh, (3, 4), LUTS, rate_axis="m"),
                lambda: packed_linear(x.float(), linear),
                lambda: packed_linear(x[:, :128], linear),
                lambda: packed_linear(x.cpu(), linear),
                lambda: packed_linear(x, linear, out=torch.empty((2, 127), dtype=x.dtype, device="cuda")),
                lambda: packed_linear(x, linear, out=torch.empty((2, 128), device="cuda")),
                lambda: LowRankAdapters(torch.zeros((1, 129, 256), dtype=x.dtype).cuda(),
                                        torch.zeros((1, 128, 129), dtype=x.dtype).cuda()),
                lambda: LowRankAdapters(torch.zeros((1, 4, 256), dtype=x.dtype).cuda(),
                                        torch.zeros((1, 128, 5), dtype=x.dtype).cuda()),
                lambda: LowRankAdapters(torch.zeros((1, 4, 256)).cuda(), torch.zeros((1, 128, 4)).cuda())):
        with pytest.raises(ValueError):
            bad()
    bank = LowRankAdapters(torch.zeros((1, 4, 256), dtype=x.dtype).cuda(), torch.zeros((1, 128, 4), dtype=x.dtype).cuda())
    for bad in (lambda: adapter_linear(x, linear, bank, ids.long()), lambda: adapter_linear(x, linear, bank, ids[:1]),
                lambda: adapter_linear(x.half(), linear, bank, ids),
                lambda: adapter_linear(x, PackedLinear(words, suh, svh, (3, 4), LUTS), LowRankAdapters(
                    torch.zeros((1, 4, 128), dtype=x.dtype).cuda(), torch.zeros((1, 128, 4), dtype=x.dtype).cuda()), ids)):
        with pytest.raises(ValueError):
            bad()

    router = torch.zeros((8, 256), dtype=x.dtype, device="cuda")
    for bad in (lambda: route_tokens(x, router, 0), lambda: route_tokens(x, router, 9), lambda: route_tokens(x, router, True),
                lambda: route_tokens(x.half(), router, 2), lambda: route_tokens(x[:, :248], router, 2),
                lambda: route_tokens(x, router, 2, scoring="tanh"),
                lambda: route_tokens(x, router, 2, bias=torch.zeros(7, device="cuda")),
                lambda: route_tokens(x, router[:, :252], 2),
                lambda: route_tokens(x, torch.zeros((1025, 256), dtype=x.dtype, device="cuda"), 2)):
        with pytest.raises(ValueError):
            bad()

    layer = Experts(33, 128, 256, 4, (3, 3))
    x = torch.zeros((2, 128), dtype=torch.bfloat16, device="cuda")
    weights, ids = torch.ones((2, 1), device="cuda"), torch.zeros((2, 1), dtype=torch.int32, device="cuda")
    for bad in (lambda: layer.packed(x, weights.half(), ids), lambda: layer.packed(x, weights, ids.long()),
                lambda: layer.packed(x, weights[:1], ids[:1]), lambda: layer.packed(x, weights.cpu(), ids),
                lambda: layer.packed(x[:, :64], weights, ids), lambda: layer.packed(x.float(), weights, ids),
                lambda: PackedMoELayer(router, layer.packed, 2),
                lambda: PackedMoELayer(torch.zeros((4, 128), dtype=x.dtype).cuda(), layer.packed, 5)):
        with pytest.raises(ValueError):
            bad()


# ---------------------------------------------------------------------------
# runs, sharing and files
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("t,k,n,adapters,rank,run,dtype", [
    (2, 256, 128, 2, 16, 1, torch.bfloat16),       # under four rows
    (15, 256, 128, 2, 48, 8, torch.float16),       # two adapters in a block of 16 rows
    (50, 128, 256, 3, 40, 16, torch.bfloat16),     # one and none
    (64, 384, 128, 9, 128, 5, torch.float16),      # four: some blocks take the other way
    (2100, 2048, 128, 5, 128, 300, torch.bfloat16),  # first products of 32 rows at once
])
def test_adapters_in_runs(t, k, n, adapters, rank, run, dtype):
    rng = np.random.default_rng(t + rank)
    bits = (3,) * (k // 128)
    p = payload(rng, k, n, bits, "k")
    linear = PackedLinear(*(torch.from_numpy(v).cuda() for v in p), bits, LUTS)
    x = rows(rng, t, k, dtype)
    a = (rows(rng, adapters * rank, k, dtype) / k**0.5).view(adapters, rank, k)
    b = (rows(rng, adapters * n, rank, dtype) / rank**0.5).view(adapters, n, rank)
    scale = torch.from_numpy(rng.uniform(0.5, 2, adapters)).float()
    ids = ((torch.arange(t) // run) % (adapters + 1)).int() - 1
    want = x.double() @ dense(*p, bits, "k")
    for i in range(adapters):
        want[ids == i] += float(scale[i]) * ((x[ids == i].double() @ a[i].double().T) @ b[i].double().T)
    bank = LowRankAdapters(a.cuda(), b.cuda(), scale.cuda())
    close(adapter_linear(x.cuda(), linear, bank, ids.cuda()), want, dtype)
    if adapters > 1:  # an adapter's infinities stay in its rows
        bank.b[0, 3, 1] = float("inf")
        got = adapter_linear(x.cuda(), linear, bank, ids.cuda()).cpu()
        keep = ids != 0
        close(got[keep], want[keep], dtype)
        assert not bool(torch.isfinite(got[~keep][:, 3]).any())


def test_router_of_many_experts_in_a_layer():
    """More experts than one workgroup chooses from: choice and grouping are launches of their own."""

    experts = Experts(41, 128, 128, 600, (3,))
    rng = np.random.default_rng(42)
    x, router = rows(rng, 3, 128, torch.bfloat16), rows(rng, 600, 128, torch.bfloat16) / 8
    y, weights, ids = PackedMoELayer(router.cuda(), experts.packed, 5)(x.cuda())
    want_w, want = choose64(x, router, 5, None, "softmax", True, 1.0)
    assert torch.equal(ids.cpu().long(), want)
    close(y, experts(x, want_w, want), torch.bfloat16)


@pytest.mark.parametrize("shared", [True, False])
def test_layer_rotates_beside_its_router(shared):
    experts = Experts(43, 256, 128, 7, (3, ), shared)
    rng = np.random.default_rng(44)
    router = rows(rng, 7, 256, torch.float16) / 16
    layer = PackedMoELayer(router.cuda(), experts.packed, 3, scoring="sigmoid")
    for t in (1, 2, 70, 90):  # with scales of their own: rotated before the choice is known, 90 after it
        x = rows(rng, t, 256, torch.float16)
        y, weights, ids = layer(x.cuda())
        want_w, want = choose64(x, router, 3, None, "sigmoid", True, 1.0)
        keep = (ids.cpu().long() == want).all(-1)  # scores nearer than FP32 sums tell apart are no fault of the experts
        assert int(keep.sum()) >= t - 1
        close(y.cpu()[keep], experts(x, want_w, want)[keep], torch.float16)


def block_hadamard64(v, size):
    h = torch.tensor([[1.0]], dtype=torch.float64)
    while h.shape[0] < size:
        h = torch.cat((torch.cat((h, h), 1), torch.cat((h, -h), 1)))
    return (v.reshape(*v.shape[:-1], -1, size) @ h / size**0.5).reshape(v.shape)


@pytest.mark.parametrize("hidden,inter,experts,bits,shared,act,t,k,draw,dtype", [
    (512, 128, 3, (3,), True, "swiglu", 1, 1, 0, torch.bfloat16),      # one block of channels, half from each product
    (1024, 384, 4, (2, 4, 3), False, "situ", 5, 2, 3, torch.float16),  # three blocks: one from both products
    (512, 256, 5, (3, 4), True, "swiglu", 90, 5, 7, torch.bfloat16),   # rows laid out by 16
    (512, 256, 5, (2, 2), False, "swiglu", 3, 9, 1, torch.bfloat16),   # more experts than shares
])
def test_coupled_experts(hidden, inter, experts, bits, shared, act, t, k, draw, dtype):
    spec = CoupledHadamardSpec(intermediate_draw=draw)
    layer = Experts(hidden + t, hidden, inter, experts, bits, shared, act)
    mats = [[m[e].clone() for m in layer.mats] for e in range(experts)]
    signs = [rotation_signs(n, draw=draw, axis=a, device="cpu").double() for n, a in ((2 * inter, 1), (inter, 2))]
    stacked = [{"trellis": m.words.view(experts, -1), "suh": m.suh, "svh": m.svh, "record_bits": bits}
               for m in (layer.packed.w1, layer.packed.w3, layer.packed.w2)]
    packed = PackedExperts(*stacked, LUTS, activation=act, coupled=spec)
    rng = np.random.default_rng(t)
    x = rows(rng, t, hidden, dtype)
    ids = torch.from_numpy(rng.integers(-1, experts, (t, k))).int()
    weights = torch.from_numpy(rng.uniform(0.1, 1, (t, k))).float()
    want, turned = torch.zeros((t, hidden), dtype=torch.float64), block_hadamard64(x.double(), 512)
    for i in range(t):
        for j, e in enumerate(ids[i].tolist()):
            if e < 0:
                continue
            z = torch.cat((turned[i] @ mats[e][0], turned[i] @ mats[e][1]))
            both = block_hadamard64(z, 128) * signs[0]
            g, u = both[0::2], both[1::2]
            mid = (g * torch.sigmoid(g) * u if act == "swiglu" else
                   4 * torch.tanh(g / 4) * torch.sigmoid(g) * 25 * torch.tanh(u / 25))
            want[i] += float(weights[i, j]) * (block_hadamard64(mid * signs[1], 128) @ mats[e][2])
    want = block_hadamard64(want, 512)
    close(packed(x.cuda(), weights.cuda(), ids.cuda()), want, dtype)
    # the source's weights, from the framework's own inverse (FP32), mean the same
    w1, w3, w2 = decode_coupled_weights(tuple(m.T.float().contiguous() for m in mats[0]), spec)
    got = packed(x.cuda(), torch.ones((t, 1)).cuda(), torch.zeros((t, 1), dtype=torch.int32).cuda())
    g, u = x.double() @ w1.double().T, x.double() @ w3.double().T
    mid = g * torch.sigmoid(g) * u if act == "swiglu" else \
        4 * torch.tanh(g / 4) * torch.sigmoid(g) * 25 * torch.tanh(u / 25)
    close(got, mid @ w2.double().T, dtype)


def test_coupled_refusals():
    layer = Experts(61, 384, 128, 2, (3,))
    stacked = [{"trellis": m.words.view(2, -1), "suh": m.suh, "svh": m.svh, "record_bits": (3,)}
               for m in (layer.packed.w1, layer.packed.w3, layer.packed.w2)]
    for spec in (CoupledHadamardSpec(), CoupledHadamardSpec(residual_block_size=128)):
        with pytest.raises(ValueError):
            PackedExperts(*stacked, LUTS, coupled=spec)


@pytest.mark.parametrize("rate_axis", ["k", "n"])
def test_projection_of_a_packed_trellis(rate_axis):
    """A mixed-rate ``PackedQSRTTrellis``, against the framework's own decode of it (FP32)."""

    geometry = Q.Geometry(512, 256)
    mode = Q.resolve_mode("R1", geometry)
    rates = Q.record_bits(mode)
    shape = (32, 16) if rate_axis == "k" else (16, 32)
    states, gen = torch.empty((*shape, 256), dtype=torch.int16), torch.Generator().manual_seed(71)
    for r, bits in enumerate(rates):
        at = (slice(8 * r, 8 * r + 8), slice(None)) if rate_axis == "k" else (slice(None), slice(8 * r, 8 * r + 8))
        states[at] = reconstruct_trellis_states(torch.randint(0, 1 << bits, (*states[at].shape[:2], 256), generator=gen), bits)
    packed = Q.pack_qsrt_trellis(states.cuda(), mode, rate_axis=rate_axis)
    k, n = 16 * shape[0], 16 * shape[1]
    suh = (torch.rand(k, generator=gen) + 0.5).half().cuda()
    svh = (torch.rand(n, generator=gen) - 0.5).half().cuda()
    luts = {b: LUTS[b] for b in set(rates)}
    x = rows(np.random.default_rng(72), 5, k, torch.bfloat16)
    want = x.double() @ decode_packed(packed, suh, svh, luts, out_dtype=torch.float32).cpu().double()
    close(packed_linear(x.cuda(), PackedLinear.from_packed(packed, suh, svh, luts)), want, torch.bfloat16)


@pytest.mark.parametrize("experts,t", [(96, 16), (96, 17), (200, 8), (200, 9)])
def test_layer_chooses_and_groups_at_once_or_apart(experts, t):
    layer = Experts(81, 128, 128, experts, (3,))
    rng = np.random.default_rng(82)
    x, router = rows(rng, t, 128, torch.bfloat16), rows(rng, experts, 128, torch.bfloat16) / 8
    y, weights, ids = PackedMoELayer(router.cuda(), layer.packed, 5)(x.cuda())
    alone = route_tokens(x.cuda(), router.cuda(), 5)
    assert torch.equal(weights, alone[0]) and torch.equal(ids, alone[1])
    close(y, layer(x, weights.cpu(), ids.cpu()), torch.bfloat16)
