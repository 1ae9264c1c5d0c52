"""Packed serving takes views as they come: whatever they are cut from, results are those of a tensor of its own."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from qsrt_amd.packed_linear import LowRankAdapters, PackedLinear, adapter_linear, packed_linear
from qsrt_amd.packed_moe import PackedMoELayer, route_tokens
from test_packed_serving_gpu import LUTS, Experts, payload, rows

pytestmark = pytest.mark.gpu


def lone_rows(x):
    """``x`` of one row as views whose strides, and addresses, are those of what they are cut from."""

    wide = torch.zeros((3, x.shape[1] + 6), dtype=x.dtype, device=x.device)
    wide[1, 2:-4] = x[0]
    odd = torch.zeros((8 + x.shape[1], 3), dtype=x.dtype, device=x.device)
    odd[8:, 1] = x[0]
    return wide[1:2, 2:-4], x[0].expand(1, -1), x.as_strided(x.shape, (12, 1)), odd[8:, 1:2].T


def test_lone_rows_of_any_stride():
    rng = np.random.default_rng(91)
    p = payload(rng, 256, 256, (3, 4), "k")
    linear = PackedLinear(*(torch.from_numpy(v).cuda() for v in p), (3, 4), LUTS)
    bank = LowRankAdapters(rows(rng, 2 * 16, 256, torch.bfloat16).view(2, 16, 256).cuda(),
                           rows(rng, 2 * 256, 16, torch.bfloat16).view(2, 256, 16).cuda())
    experts = Experts(92, 256, 128, 3, (3,)).packed
    router = rows(rng, 3, 256, torch.bfloat16).cuda()
    layer = PackedMoELayer(router, experts, 2)
    x = rows(rng, 1, 256, torch.bfloat16).cuda()
    ids, chosen = torch.ones(1, dtype=torch.int32, device="cuda"), torch.tensor([[2, 0]], dtype=torch.int32, device="cuda")
    weights = torch.ones((1, 2), device="cuda")
    for call in (lambda v, out=None: packed_linear(v, linear, out=out),
                 lambda v, out=None: adapter_linear(v, linear, bank, ids, out=out),
                 lambda v, out=None: experts(v, weights, chosen, out=out),
                 lambda v, out=None: layer(v, out=out)[0],
                 lambda v, out=None: route_tokens(v, router, 2)[0]):
        want = call(x)
        for view in lone_rows(x):
            assert torch.equal(call(view), want)
        if want.shape[1] == 256:
            wide = torch.full((3, 262), 7.0, dtype=x.dtype, device="cuda")
            call(x, out=wide[1:2, 2:258])  # 8-byte aligned, its stride is not
            assert torch.equal(wide[1:2, 2:258], want) and int((wide == 7).sum()) >= 3 * 262 - 256


def test_a_lone_expert_of_any_stride():
    rng = np.random.default_rng(93)
    router, x = rows(rng, 1, 256, torch.bfloat16).cuda(), rows(rng, 4, 256, torch.bfloat16).cuda()
    want = route_tokens(x, router, 1, scoring="sigmoid", normalize=False)
    for view in lone_rows(router):
        got = route_tokens(x, view, 1, scoring="sigmoid", normalize=False)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_payloads_at_any_address():
    """Words and scales cut from larger buffers, at addresses that the kernels' loads do not take."""

    rng = np.random.default_rng(94)
    words, suh, svh = (torch.from_numpy(v).cuda() for v in payload(rng, 256, 128, (3, 4), "k"))

    def moved(v):
        wide = torch.zeros(v.numel() + 1, dtype=v.dtype, device="cuda")
        wide[1:] = v
        return wide[1:]

    x = rows(rng, 3, 256, torch.bfloat16).cuda()
    want = packed_linear(x, PackedLinear(words, suh, svh, (3, 4), LUTS))
    for cut in ((moved(words), suh, svh), (words, moved(suh), svh), (words, suh, moved(svh))):
        assert torch.equal(packed_linear(x, PackedLinear(*cut, (3, 4), LUTS)), want)
