"""Tensors with a forward-mode tangent are refused: they do not require a gradient, and the tangent would be dropped.  The refusal
comes before any other, so it needs no GPU."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from qsrt_amd.block_norm import residual_norm, rms_norm
from qsrt_amd.gated_ffn import _GatedFFN, gated_ffn, gated_ffn_gradients
from qsrt_amd.gradient_guided_viterbi import expert_guidance
from qsrt_amd.packed_linear import packed_linear, refuse_gradients, refuse_tangents
from qsrt_amd.packed_moe import route_tokens

X, W, D = torch.ones(2, 16, dtype=torch.bfloat16), torch.ones(8, 16, dtype=torch.bfloat16), torch.ones(16, 8, dtype=torch.bfloat16)
V = torch.ones(16, dtype=torch.bfloat16)
CALLS = [
    (lambda *a: gated_ffn(*a), (X, W, W, D)),
    (lambda *a: gated_ffn_gradients(*a), (X, X, W, W, D)),
    (lambda *a: expert_guidance(*a, anchor_id="a", objective_id="o"), (X, X, W, W, D)),
    (lambda r, y, w, p, g: residual_norm(r, y, w, post_weight=p, gate=g), (X, X, V, V, V)),
    (lambda *a: rms_norm(*a), (X, V)),
    (lambda x, w, b: route_tokens(x, w, 1, bias=b), (X, W, torch.ones(8))),
    (lambda x: packed_linear(x, None), (X,)),
]


@pytest.mark.parametrize("no_grad", [False, True])
@pytest.mark.parametrize("number", range(len(CALLS)))
def test_calls_refuse_tangents(number, no_grad):
    call, tensors = CALLS[number]
    with forward_ad.dual_level():
        for i, t in enumerate(tensors):
            given = [forward_ad.make_dual(v, torch.ones_like(v)) if i == j else v for j, v in enumerate(tensors)]
            with torch.set_grad_enabled(not no_grad), pytest.raises(ValueError, match="tangent"):
                call(*given)


def test_jvp_is_refused():
    with pytest.raises(ValueError, match="tangent"):
        torch.func.jvp(lambda x: gated_ffn(x, W, W, D), (X,), (X,))


def test_a_tangent_of_the_results_gradient_is_refused():
    with forward_ad.dual_level(), torch.no_grad(), pytest.raises(ValueError, match="tangent"):
        _GatedFFN.backward(None, forward_ad.make_dual(X, X))


def test_tensors_without_a_tangent_pass():
    refuse_tangents(X, None)
    with forward_ad.dual_level():
        refuse_tangents(X, None)
        refuse_gradients(X, None)
        with pytest.raises(ValueError, match="CUDA"):
            gated_ffn(X, W, W, D)
