"""Packed serving has no backward pass and says so, instead of returning results that a gradient silently stops at."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from qsrt_amd.packed_linear import LowRankAdapters, PackedLinear, adapter_linear, packed_linear
from qsrt_amd.packed_moe import PackedMoELayer, route_tokens
from test_packed_serving_gpu import LUTS, Experts, payload, rows

pytestmark = pytest.mark.gpu


def test_inputs_that_require_a_gradient_are_refused():
    rng = np.random.default_rng(95)
    p = payload(rng, 256, 128, (3, 3), "k")
    linear = PackedLinear(*(torch.from_numpy(v).cuda() for v in p), (3, 3), LUTS)
    x = rows(rng, 2, 256, torch.bfloat16).cuda()
    a, b = rows(rng, 8, 256, torch.bfloat16).view(1, 8, 256).cuda(), rows(rng, 128, 8, torch.bfloat16).view(1, 128, 8).cuda()
    ids = torch.zeros(2, dtype=torch.int32, device="cuda")
    experts, router = Experts(96, 256, 128, 3, (3,)).packed, rows(rng, 3, 256, torch.bfloat16).cuda()
    chosen, weights = torch.zeros((2, 1), dtype=torch.int32, device="cuda"), torch.ones((2, 1), device="cuda")
    bias, scale = torch.zeros(3, device="cuda"), torch.ones(1, device="cuda")

    def parameter(t):
        return t.clone().requires_grad_()

    calls = (lambda g: packed_linear(g(x), linear),
             lambda g: adapter_linear(g(x), linear, LowRankAdapters(a, b), ids),
             lambda g: adapter_linear(x, linear, LowRankAdapters(g(a), b), ids),  # rank 8: padded, a part of the graph
             lambda g: adapter_linear(x, linear, LowRankAdapters(a, g(b)), ids),
             lambda g: adapter_linear(x, linear, LowRankAdapters(a, b, g(scale)), ids),
             lambda g: experts(g(x), weights, chosen), lambda g: experts(x, g(weights), chosen),
             lambda g: PackedMoELayer(router, experts, 2)(g(x))[0], lambda g: PackedMoELayer(g(router), experts, 2)(x)[0],
             lambda g: PackedMoELayer(router, experts, 2, bias=g(bias))(x)[0],
             lambda g: route_tokens(g(x), router, 2)[0], lambda g: route_tokens(x, g(router), 2)[0],
             lambda g: route_tokens(x, router, 2, bias=g(bias))[0])
    for call in calls:
        with pytest.raises(ValueError, match="backward"):
            call(parameter)
        with torch.no_grad():
            got = call(parameter)
        assert torch.equal(got, call(lambda t: t)) and not got.requires_grad
