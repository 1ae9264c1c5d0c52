"""``out`` of the serving calls is written by a kernel: autograd hears of it."""

from __future__ import annotations

import pytest
import torch

from qsrt_amd.gated_ffn import gated_ffn
from qsrt_amd.packed_linear import checked_out

X = torch.zeros(3, 16, dtype=torch.bfloat16)


def test_graphs_that_kept_out_are_told():
    out = torch.ones(3, 8, dtype=torch.bfloat16)
    w = torch.ones(3, 8, dtype=torch.bfloat16, requires_grad=True)
    loss = (out * w).sum()
    assert checked_out(out, X, 8) is out
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_out_of_a_graph_is_refused():
    leaf = torch.ones(3, 8, dtype=torch.bfloat16, requires_grad=True)
    for out in (leaf, leaf * 2):
        with pytest.raises(ValueError, match="out requires a gradient"):
            checked_out(out, X, 8)
        with torch.no_grad():
            assert checked_out(out, X, 8) is out


def test_out_with_a_tangent_is_refused():
    with torch.autograd.forward_ad.dual_level():
        out = torch.autograd.forward_ad.make_dual(X, X.clone())
        with pytest.raises(ValueError, match="tangent"):
            checked_out(out, X, 16)


def test_inference_tensors_pass():
    with torch.inference_mode():
        out = torch.ones(3, 8, dtype=torch.bfloat16)
        assert checked_out(out, X, 8) is out
    assert checked_out(out, X, 8) is out
    assert checked_out(None, X, 8).shape == (3, 8)


@pytest.mark.gpu
def test_the_block_tells_too():
    g = torch.Generator(device="cuda").manual_seed(1)
    x, gate, up, down = (torch.randn(shape, generator=g, device="cuda").to(torch.bfloat16) for shape in ((3, 16), (8, 16), (8, 16), (16, 8)))
    out = torch.ones_like(x)
    loss = (out * x.detach().requires_grad_()).sum()
    gated_ffn(x, gate, up, down, out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
