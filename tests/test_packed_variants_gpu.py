"""Every variant of the packed products and of the router's choice, at sizes that the rules send there.

The products' variants are asked for first (``qsrt_adapter_linear_plan``, ``qsrt_packed_moe_plan``), so that a rule that
changes does not leave one untested.
"""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from qsrt_amd import _native
from qsrt_amd.packed_linear import PackedLinear, packed_linear
from qsrt_amd.packed_moe import PackedMoELayer, route_tokens
from test_packed_serving_gpu import LUTS, Experts, choose64, close, dense, payload, rows

pytestmark = pytest.mark.gpu


def linear_plan(linear, t):
    plan = (ctypes.c_int64 * 3)()
    _native.check(_native.lib().qsrt_adapter_linear_plan(linear.matrix.ref, t, 0, 0, plan), "qsrt_adapter_linear_plan")
    return tuple(plan)


@pytest.mark.parametrize("t,k,n,bits,share,turns,dtype", [
    (5, 256, 256, (2, 2), 8, 1, torch.bfloat16),
    (5, 384, 128, (4, 3, 2), 8, 1, torch.float16),
    (13, 256, 256, (2, 2), 16, 1, torch.float16),
    (33, 384, 128, (2, 2, 2), 32, 1, torch.bfloat16),
    (47, 256, 256, (4, 3), 32, 1, torch.float16),
    (100, 384, 128, (2, 2, 2), 64, 1, torch.float16),
    (100, 256, 256, (3, 4), 64, 1, torch.bfloat16),
    (128, 256, 128, (3, 3), 64, 1, torch.bfloat16),
    (129, 384, 128, (2, 2, 2), 256, 1, torch.float16),
    (2100, 128, 8192, (4,), 256, 3, torch.bfloat16),      # workgroups go through three pieces of work
    (2000, 128, 8192, (3,), 512, 1, torch.bfloat16),
    (1990, 256, 8192, (2, 4), 512, 1, torch.float16),     # two tables
    (3900, 128, 8192, (2,), 512, 2, torch.float16),
    (3900, 384, 8192, (4, 2, 3), 512, 2, torch.bfloat16),  # two passes
])
def test_projections(t, k, n, bits, share, turns, dtype):
    rng = np.random.default_rng(t + n)
    p = payload(rng, k, n, bits, "k")
    linear = PackedLinear(*(torch.from_numpy(v).cuda() for v in p), bits, LUTS)
    plan = linear_plan(linear, t)
    units = torch.cuda.get_device_properties(0).multi_processor_count
    if units == 256:
        assert plan[0] == share and (turns == 1 or -(-plan[2] // units) == turns), plan
    x = rows(rng, t, k, dtype)
    keep = slice(None, None, 7 if n > 1024 else 1)  # every place of a block of 128 columns all the same
    close(packed_linear(x.cuda(), linear)[:, keep], x.double() @ dense(*p, bits, "k")[:, keep], dtype)


@pytest.mark.parametrize("experts,t,k,bits,share,dtype", [
    (9, 4, 3, (2, 2), 8, torch.bfloat16), (3, 8, 2, (2, 2), 16, torch.float16), (3, 10, 2, (2, 2), 16, torch.bfloat16),
    (3, 31, 2, (2, 2), 32, torch.float16), (2, 45, 2, (2, 2), 64, torch.bfloat16), (2, 45, 2, (3, 4), 64, torch.float16),
    (2, 150, 2, (4, 4), 64, torch.bfloat16),
])
def test_experts(experts, t, k, bits, share, dtype):
    layer = Experts(t, 256, 256, experts, bits)
    plan = (ctypes.c_int64 * 3)()
    w = layer.packed
    _native.check(_native.lib().qsrt_packed_moe_plan(w.w1.ref, w.w3.ref, w.w2.ref, experts, t, k, plan), "qsrt_packed_moe_plan")
    assert plan[0] == share
    rng = np.random.default_rng(t)
    x, ids = rows(rng, t, 256, dtype), torch.from_numpy(rng.integers(-1, experts, (t, k))).int()
    weights = torch.from_numpy(rng.uniform(0.1, 1, (t, k))).float()
    close(layer.packed(x.cuda(), weights.cuda(), ids.cuda()), layer(x, weights, ids), dtype)


@pytest.mark.parametrize("t,h,e,k", [
    (3, 4096, 450, 8),    # eight experts a lane, the sums of eight splits in two turns
    (2, 2048, 640, 5),    # sixteen, four splits in two turns
    (1, 8192, 1000, 64),
    (40, 1536, 385, 3),
])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_routers(t, h, e, k, scoring):
    rng = np.random.default_rng(e)
    x, w = rows(rng, t, h, torch.bfloat16), rows(rng, e, h, torch.bfloat16) / h**0.5
    got_w, got = route_tokens(x.cuda(), w.cuda(), k, scoring=scoring)
    want_w, want = choose64(x, w, k, None, scoring, True, 1.0)
    assert torch.equal(got.cpu().long(), want)
    # exact products; FP32 sums of `h` terms of about one, then exp, sum and quotient in FP32
    assert torch.allclose(got_w.cpu().double(), want_w, rtol=2e-5, atol=0)


@pytest.mark.parametrize("t", [1, 8, 9])
def test_layer_of_eight_experts_a_lane(t):
    """Up to eight tokens are chosen for and grouped in one launch."""

    experts = Experts(83, 128, 128, 450, (2,))
    rng = np.random.default_rng(84)
    x, router = rows(rng, t, 128, torch.bfloat16), rows(rng, 450, 128, torch.bfloat16) / 8
    y, weights, ids = PackedMoELayer(router.cuda(), experts.packed, 6)(x.cuda())
    alone = route_tokens(x.cuda(), router.cuda(), 6)
    assert torch.equal(weights, alone[0]) and torch.equal(ids, alone[1])
    close(y, experts(x, weights.cpu(), ids.cpu()), torch.bfloat16)


def test_plans_refuse():
    plan, lib = (ctypes.c_int64 * 3)(), _native.lib()
    p = payload(np.random.default_rng(85), 128, 128, (3,), "k")
    w = PackedLinear(*(torch.from_numpy(v).cuda() for v in p), 3, LUTS).matrix.ref
    for args in ((None, 1, 0, 0, plan), (w, 0, 0, 0, plan), (w, -1, 0, 0, plan), (w, 1, 0, 0, None), (w, 1, 2, 8, plan)):
        assert lib.qsrt_adapter_linear_plan(*args) == -1
    for args in ((None, w, w, 2, 1, 1, plan), (w, w, w, 2, 0, 1, plan), (w, w, w, 0, 1, 1, plan), (w, w, w, 2, 1, 1, None)):
        assert lib.qsrt_packed_moe_plan(*args) == -1
