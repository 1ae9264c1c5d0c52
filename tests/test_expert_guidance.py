"""``expert_guidance`` by itself: the gradients of the block are stood in for, so it needs no GPU."""

from __future__ import annotations

import pytest
import torch

from qsrt_amd import gradient_guided_viterbi as guided
from qsrt_amd.gated_ffn import GatedFFNGradients


@pytest.fixture
def stand_in(monkeypatch):
    """The block's rows in 64 bits, rounded to x's type once as its own are."""

    @torch.no_grad()
    def gradients(x, dy, gate, up, down, *, activation, inputs, weights):
        assert activation == "swiglu" and not inputs and not weights
        g, u, dm = x.double() @ gate.double().T, x.double() @ up.double().T, dy.double() @ down.double()
        s = torch.sigmoid(g)
        rows = dm * u * s * (1 + g * (1 - s)), dm * g * s, g * s * u
        return GatedFFNGradients(None, None, None, None, *(r.to(x.dtype) for r in rows))

    monkeypatch.setattr(guided, "gated_ffn_gradients", gradients)


def draw(dtype, scale=1.0):
    g = torch.Generator().manual_seed(1)

    def normal(*shape, by=1.0):
        return (by * torch.randn(shape, generator=g)).to(dtype)

    return normal(24, 64), (scale * normal(24, 64).float()).to(dtype), *(normal(*shape, by=0.125) for shape in ((40, 64), (40, 64), (64, 40)))


def call(x, dy, gate, up, down):
    return guided.expert_guidance(x, dy, gate, up, down, anchor_id="a", objective_id="o", activation="swiglu")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_no_graph_is_kept(dtype, stand_in):
    """x in the middle of a graph, the weights parameters of a module: what a trained model gives."""

    x, dy, gate, up, down = draw(dtype)
    x = x.requires_grad_() * 1
    assert x.grad_fn is not None
    guidance = call(x, dy, *(torch.nn.Parameter(w) for w in (gate, up, down)))
    for g, shape in zip(guidance.values(), ((64, 40), (64, 40), (40, 64))):
        assert not any(t.requires_grad for t in (g.left, g.right, g.anchor))
        g.validate(shape)
        out = torch.zeros(16, shape[1])
        out.copy_(g.rows(slice(0, 16), device="cpu", dtype=torch.float32))
        out.numpy()


@pytest.mark.parametrize("size", [1.0, 1e-4, 1e-6, 2.0**-24])
def test_small_f16_gradients_keep_their_bits(size, stand_in):
    """dG and dU are f16, off by 2^-11 of themselves or 2^-25, half the type's last step.  dy's largest value is brought to 2^-4 or
    more for them: 2^-25 there is 2^-21 of it here."""

    x, dy, gate, up, down = draw(torch.float16, size)
    guidance = call(x, dy, gate, up, down)
    X, Y, G, U, D = (t.double() for t in (x, dy, gate, up, down))
    g, u = X @ G.T, X @ U.T
    s = torch.sigmoid(g)
    most = float(Y.abs().max())
    for name, by in (("w1", u * s * (1 + g * (1 - s))), ("w3", g * s)):
        rows = (Y @ D) * by
        off = (guidance[name].right.double() - rows).abs()
        assert bool((off <= 2.0**-11 * rows.abs() + 2.0**-21 * most).all()), name
    assert torch.equal(guidance["w2"].right, dy.float())


@pytest.mark.parametrize("value", [float("inf"), float("nan")])
def test_gradients_that_are_not_finite_are_found(value, stand_in):
    x, dy, gate, up, down = draw(torch.float16)
    dy[3, 5] = value
    for g, shape in zip(call(x, dy, gate, up, down).values(), ((64, 40), (64, 40), (40, 64))):
        with pytest.raises(ValueError, match="finite"):
            g.validate(shape)


def test_a_gradient_of_zeros(stand_in):
    x, dy, gate, up, down = draw(torch.float16, 0.0)
    for name, g in call(x, dy, gate, up, down).items():
        assert bool((g.left @ g.right == 0).all())
