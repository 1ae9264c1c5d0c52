"""Packed products hold what they multiply in 24 bits.

Outputs of 16 bits hide smaller faults, so the inputs here cancel: a payload's blocks of 128 channels come in pairs of equal
words whose rows are x and -x (1 + 2^-10), and what is left is 2^-10 of either.  A relative error of a held value comes out
2^10 times larger.  FP32 forms stay under 2^-20 of either half in 2-norm (about ten roundings of 2^-24 in a rotation, sums of a
few dozen steps), so under 2^-10 of the result, beside its rounding to the output's type; values held in 17 bits are off by
2^-18.5 at the root mean square, 2^-8 of the result.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from qsrt_amd.packed_linear import LowRankAdapters, PackedLinear, adapter_linear, packed_linear
from qsrt_amd.packed_moe import PackedExperts
from qsrt_amd.qsrt_coupled import CoupledHadamardSpec, rotation_signs
from test_packed_serving_gpu import LUTS, ROUND, dense, rows

pytestmark = pytest.mark.gpu
NEAR = 1.0 + 2.0**-10  # exact in f16


def near(got, want, dtype):
    got, want = got.cpu().double(), want.double()
    assert bool(torch.isfinite(got).all())
    error = float((got - want).norm() / want.norm())
    assert error <= ROUND[dtype] + 2.0**-10, error


def paired(rng, k, n, bits, svh):
    """A matrix of records along k in pairs of equal words, the second of each at scales ``NEAR`` times the first's."""

    words = []
    for b in bits[::2]:
        words += 2 * [rng.integers(-32768, 32768, size=8 * (n // 16) * 16 * b).astype(np.int16)]
    suh = np.concatenate([np.concatenate((s, s * NEAR)) for s in rng.choice([-1.0, 1.0], (k // 256, 128))]).astype(np.float16)
    svh = (svh * rng.uniform(0.5, 1.5, n) * rng.choice([-1, 1], n)).astype(np.float16)
    return np.concatenate(words), suh, svh


def opposite(rng, t, k, dtype):
    x = rows(rng, t * (k // 256), 128, dtype)
    return torch.cat((x, -x), -1).reshape(t, k)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bits", [(3, 3), (2, 2), (3, 3, 4, 4)])
@pytest.mark.parametrize("t,n", [(1, 256), (8, 128), (16, 128), (40, 128), (100, 128), (130, 256), (1025, 128)])
def test_projection(t, n, bits, dtype):
    rng = np.random.default_rng(t + len(bits))
    p = paired(rng, 128 * len(bits), n, bits, 8.0)
    linear = PackedLinear(*(torch.from_numpy(v).cuda() for v in p), bits, LUTS)
    x = opposite(rng, t, 128 * len(bits), dtype)
    near(packed_linear(x.cuda(), linear), x.double() @ dense(*p, bits, "k"), dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("size", [2.0**-100, 2.0**100])
def test_rows_of_any_size(size, dtype):
    """Rows of one call as far apart as their type goes, none of them scaled by another's; with one of zeros among them."""

    rng = np.random.default_rng(7)
    bits = (3, 3)
    p = paired(rng, 256, 128, bits, 8.0)
    linear = PackedLinear(*(torch.from_numpy(v).cuda() for v in p), bits, LUTS)
    if dtype == torch.float16:  # results 2^-10 of the rows come to the type's normal values
        size = 2.0**12 if size > 1 else 2.0**-3
    for t in (5, 200):
        x = opposite(rng, t, 256, dtype)
        x[1::2] *= size
        x[0] = 0
        want = x.double() @ dense(*p, bits, "k") * torch.where(torch.arange(t) % 2 == 1, 1 / size, 1.0)[:, None]
        got = packed_linear(x.cuda(), linear).cpu().double()
        assert not bool(got[0].any())
        got[1::2] /= size
        near(got[1::2], want[1::2], dtype)
        near(got[2::2], want[2::2], dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_infinities_leave_the_scales_of_other_rows_alone(dtype):
    rng = np.random.default_rng(8)
    p = paired(rng, 256, 128, (3, 3), 8.0)
    linear = PackedLinear(*(torch.from_numpy(v).cuda() for v in p), (3, 3), LUTS)
    x = opposite(rng, 200, 256, dtype)
    want = x.double() @ dense(*p, (3, 3), "k")
    bad = [3, 64, 127, 199]
    for row, value in zip(bad, (float("inf"), float("nan"), -float("inf"), float("nan"))):
        x[row, (50 * row) % 256] = value
    got = packed_linear(x.cuda(), linear).cpu()
    keep = [i for i in range(200) if i not in bad]
    near(got[keep], want[keep], dtype)
    assert not bool(torch.isfinite(got[bad]).any())


def test_scaled_rows_in_a_graph():
    """Captured once, replayed on rows of other sizes with eager work in between."""

    rng = np.random.default_rng(9)
    p = paired(rng, 256, 128, (3, 3), 8.0)
    linear = PackedLinear(*(torch.from_numpy(v).cuda() for v in p), (3, 3), LUTS)
    bank = LowRankAdapters(rows(rng, 2 * 16, 256, torch.bfloat16).view(2, 16, 256).cuda(),
                           rows(rng, 2 * 128, 16, torch.bfloat16).view(2, 128, 16).cuda())
    x, ids = rows(rng, 150, 256, torch.bfloat16).cuda(), ((torch.arange(150) // 40) % 3 - 1).int().cuda()
    adapter_linear(x, linear, bank, ids)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = adapter_linear(x, linear, bank, ids)
    for size in (1.0, 2.0**20, 2.0**-30, 1.0):
        x.copy_(rows(rng, 150, 256, torch.bfloat16) * size)
        want = adapter_linear(x, linear, bank, ids)
        packed_linear(x[:7].contiguous(), linear)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("t,run", [(2, 1), (40, 40), (200, 60)])
def test_second_product_of_an_adapter(t, run, dtype):
    """First products that cancel in the second, where the projection itself is nothing."""

    rng = np.random.default_rng(t)
    k, n, bits = 256, 128, (3, 3)
    p = paired(rng, k, n, bits, 0.0)
    linear = PackedLinear(*(torch.from_numpy(v).cuda() for v in p), bits, LUTS)
    parts = (1.0, -NEAR) if dtype == torch.float16 else (1.0, -(1 + 2.0**-7), 2.0**-7 * (1 - 2.0**-3))  # sum -2^-10
    a, b = torch.zeros((2, 16, k)), torch.zeros((2, n, 16))
    sign = torch.from_numpy(rng.choice([-1.0, 1.0], (2, k)))
    value = rows(rng, 2 * n, 1, dtype).view(2, n).double()
    for i, v in enumerate(parts):
        a[:, 3 * i + 1], b[:, :, 3 * i + 1] = (v * sign).float(), value.float()
    a, b = a.to(dtype), b.to(dtype)
    x, ids = rows(rng, t, k, dtype), ((torch.arange(t) // run) % 2).int()
    want = torch.stack([(x[i].double() @ a[j].double().T) @ b[j].double().T for i, j in enumerate(ids.tolist())])
    near(adapter_linear(x.cuda(), linear, LowRankAdapters(a.cuda(), b.cuda()), ids.cuda()), want, dtype)


def stacked(p, bits, axis):
    return {"trellis": torch.from_numpy(p[0])[None].cuda(), "suh": torch.from_numpy(p[1]).cuda(),
            "svh": torch.from_numpy(p[2]).cuda(), "record_bits": bits, "rate_axis": axis}


def turn(v, size):
    """The normalised Hadamard on blocks of ``size``, in ``v``'s type."""

    h = torch.ones((1, 1), dtype=v.dtype)
    while h.shape[0] < size:
        h = torch.cat((torch.cat((h, h), 1), torch.cat((h, -h), 1)))
    return (v.unflatten(-1, (-1, size)) @ h / size**0.5).flatten(-2)


def silu_up(g, u):
    return g * torch.sigmoid(g) * u


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bits", [(3, 3), (2, 2)])
@pytest.mark.parametrize("t", [1, 7, 20, 90])
def test_first_product_of_an_expert(t, bits, dtype):
    rng = np.random.default_rng(t)
    gate, up = paired(rng, 256, 128, bits, 32.0), paired(rng, 256, 128, bits, 32.0)
    up = (up[0], gate[1], up[2])
    down = paired(rng, 256, 256, bits, 0.05)
    down = (down[0][:down[0].size // 2], down[1][:128], down[2])
    packed = PackedExperts(stacked(gate, bits, "k"), stacked(up, bits, "k"), stacked(down, bits[:1], "k"), LUTS)
    x = opposite(rng, t, 256, dtype)
    mid = silu_up(x.double() @ dense(*gate, bits, "k"), x.double() @ dense(*up, bits, "k"))
    want = mid @ dense(*down, bits[:1], "k")
    # gate and up are off by 2^-10 at the most each; silu's slope is under 2 of its value where that is not small
    got = packed(x.cuda(), torch.ones((t, 1)).cuda(), torch.zeros((t, 1), dtype=torch.int32).cuda()).cpu().double()
    assert float((got - want).norm() / want.norm()) <= ROUND[dtype] + 3 * 2.0**-10


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bits", [(3, 3), (2, 2)])
@pytest.mark.parametrize("t", [1, 7, 20, 90])
def test_second_product_of_an_expert(t, bits, dtype):
    """Gate and up channels 128 .. 255 are those of 0 .. 127, up with the other sign: the middle's halves cancel."""

    rng = np.random.default_rng(t)
    first = []
    for sign in (1, -1):
        words = rng.integers(-32768, 32768, size=8 * 16 * 16 * bits[0]).astype(np.int16)
        svh = (0.05 * rng.uniform(0.5, 1.5, 128)).astype(np.float16)
        first.append((np.concatenate((words, words)), rng.choice([-1.0, 1.0], 256).astype(np.float16),
                      np.concatenate((svh, sign * svh))))
    gate, up = first
    up = (up[0], gate[1], up[2])
    down = paired(rng, 256, 256, bits, 8.0)
    packed = PackedExperts(stacked(gate, bits, "n"), stacked(up, bits, "n"), stacked(down, bits, "k"), LUTS)
    x = rows(rng, t, 256, dtype)
    mid = silu_up(x.double() @ dense(*gate, bits, "n"), x.double() @ dense(*up, bits, "n"))
    near(packed(x.cuda(), torch.ones((t, 1)).cuda(), torch.zeros((t, 1), dtype=torch.int32).cuda()),
         mid @ dense(*down, bits, "k"), dtype)


def test_coupled_results_are_as_near_as_in_32_bits():
    """f16 results that are not the rounding of the exact value: no more of them than with the same steps in FP32 throughout."""

    hidden, inter, t, bits = 512, 256, 90, (3, 3)
    rng = np.random.default_rng(3)
    mats = []
    for k, n, axis, svh in ((hidden, inter, "n", 0.05), (hidden, inter, "n", 0.05), (inter, hidden, "k", 0.1)):
        words = rng.integers(-32768, 32768, size=2 * 8 * (hidden // 16) * 16 * 3).astype(np.int16)
        suh = rng.uniform(0.5, 1.5, k).astype(np.float16)
        mats.append((words, suh, (svh * rng.uniform(0.5, 1.5, n)).astype(np.float16)))
    mats[1] = (mats[1][0], mats[0][1], mats[1][2])
    packed = PackedExperts(*(stacked(p, bits, a) for p, a in zip(mats, "nnk")), LUTS, activation="swiglu",
                           coupled=CoupledHadamardSpec())
    x = rows(rng, t, hidden, torch.float16)
    got = packed(x.cuda(), torch.ones((t, 1)).cuda(), torch.zeros((t, 1), dtype=torch.int32).cuda())

    def plain(dtype):
        w1, w3, w2 = (dense(*p, bits, a).to(dtype) for p, a in zip(mats, "nnk"))
        signs = [rotation_signs(n, draw=0, axis=a, device="cpu").to(dtype) for n, a in ((2 * inter, 1), (inter, 2))]
        turned = turn(x.to(dtype), 512)
        both = turn(torch.cat((turned @ w1, turned @ w3), -1), 128) * signs[0]
        return turn(turn(silu_up(both[:, 0::2], both[:, 1::2]) * signs[1], 128) @ w2, 512)

    want = plain(torch.float64).to(torch.float16)
    assert float(want.abs().median()) > 2.0**-10  # normal values
    moved = int((got.cpu() != want).sum())
    assert moved <= int((plain(torch.float32).to(torch.float16) != want).sum()), moved
