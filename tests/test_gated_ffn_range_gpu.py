"""Gradients of the gated feed-forward block where f16 ends, against 64 bits, element by element, with the bounds of
``test_gated_ffn_gpu``.

The rows between the products of the backward pass (M, dG, dU) are f16 too, whose steps stop shrinking at 2^-24.  They are scaled
there by a power of two, so that a bound on all of them lies from 2^14 to 2^15: max |M| for M, and for dG and dU the largest norm
of a row of dy, times sqrt(hidden) max |down| (of a column of down no norm is larger), times the largest slope.  A rounding
is then off by ``u`` of the value or 2^-25, half of the smallest step, over the scale: 2^-39 of the bound."""

from __future__ import annotations

import pytest
import torch

from qsrt_amd.gated_ffn import gated_ffn, gated_ffn_gradients
from qsrt_amd.gradient_guided_viterbi import expert_guidance
from test_gated_ffn_gpu import V, check, draw, slopes

pytestmark = pytest.mark.gpu
F16 = torch.float16


def want(x, gate, up, down, dy, activation):
    """``{name: (value, bound)}`` of the gradients in 64 bits."""

    pieces = 1 if x.shape[0] > 64 else 2
    u = torch.finfo(x.dtype).eps / 2
    tiny = float(torch.finfo(x.dtype).smallest_normal) * u  # of a result: the type's own
    row = u if pieces == 1 else u * u
    x, gate, up, down, dy = (t.double() for t in (x, gate, up, down, dy))
    t, hidden = x.shape
    inter = gate.shape[0]
    g, p = x @ gate.T, x @ up.T
    dg, dp = ((hidden + 1) * V * (x.abs() @ w.abs().T) for w in (gate, up))
    m, by_g, by_u = slopes(g, p, activation)
    flow = 32 * V
    mag_g, mag_u = 1.1 * p.abs(), 1.1 * g.abs()
    m_off = mag_g * dg + mag_u * dp + dg * dp + flow * g.abs() * p.abs()
    slope_g, slope_u = 1.1 * p.abs() * dg + 1.1 * dp + flow * mag_g, 1.1 * (dg + dp) + flow * mag_u
    most = float(dy.norm(dim=1).max()) * hidden**0.5 * float(down.abs().max()) * max(float(by_g.abs().max()), float(by_u.abs().max()))

    def rounded(value, off, by, floor):
        return off + by * (value.abs() + off) + floor

    def product(a, a_off, b, k):
        return a_off @ b.abs() + (k + 1) * V * ((a.abs() + a_off) @ b.abs())

    m_off = rounded(m, m_off, row, 2.0**-39 * float(m.abs().max()))
    rows = dy @ down
    rows_off = (hidden + 1) * V * (dy.abs() @ down.abs())
    (vg, og), (vu, ou) = [
        (rows * by, rounded(rows * by, rows_off * by.abs() + (rows.abs() + rows_off) * off + 4 * V * (rows * by).abs(), row,
                            2.0**-39 * most)) for by, off in ((by_g, slope_g), (by_u, slope_u))]
    out = {"x": (vg @ gate + vu @ up, product(torch.cat((vg, vu), 1), torch.cat((og, ou), 1), torch.cat((gate, up)), 2 * pieces * inter))}
    for name, v, off in (("gate", vg, og), ("up", vu, ou)):
        out[name] = (v.T @ x, product(v.T.contiguous(), off.T.contiguous(), x, pieces * t))
    out["down"] = (dy.T @ m, product(m.T.contiguous(), m_off.T.contiguous(), dy, pieces * t).T)
    return {name: (value, rounded(value, off, u, tiny)) for name, (value, off) in out.items()}


def spread(seed, t, hidden, inter, size, by):
    """Rows of dy of about ``size``; x times ``by`` and gate and up over it: G and U, and so the rows between, stay as they are."""

    x, gate, up, down, dy = draw(seed, t, hidden, inter, F16)
    x, gate, up = (x.float() * by).half(), (gate.float() / by).half(), (up.float() / by).half()
    return x, gate, up, down, (dy.float() * (4 * size)).half()


SIZES = [(1, 72, 200), (12, 264, 136), (33, 520, 72), (64, 136, 264), (65, 264, 520), (129, 1032, 392), (500, 264, 1032), (3, 8, 8)]


@pytest.mark.parametrize("size", [1.0, 1e-4, 1e-5, 1e-6])
@pytest.mark.parametrize("t,hidden,inter", SIZES)
def test_small_gradients(t, hidden, inter, size):
    activation = ("swiglu", "situ")[t % 2]
    for by in (2.0**6, 2.0**-6):  # x large shows dG and dU in the gradients of gate and up, the matrices large in those of x
        x, gate, up, down, dy = spread(t + hidden, t, hidden, inter, size, by)
        got = gated_ffn_gradients(x, dy, gate, up, down, activation=activation)
        check(vars(got), want(x, gate, up, down, dy, activation), ["x", "gate", "up", "down"])
        leaves = [v.detach().requires_grad_() for v in (x, gate, up, down)]
        for a, b in zip(torch.autograd.grad(gated_ffn(*leaves, activation=activation), leaves, dy), vars(got).values()):
            assert torch.equal(a, b)


@pytest.mark.parametrize("t,hidden,inter", SIZES)
def test_small_rows_between_the_products(t, hidden, inter):
    """G and U of 2^-8, M of about 2^-17, a dy that makes its gradient large."""

    x, gate, up, down, dy = draw(t, t, hidden, inter, F16)
    x, dy = (x.float() * 2.0**-8).half(), (dy.float() * 2.0**8).half()
    got = gated_ffn_gradients(x, dy, gate, up, down)
    check(vars(got), want(x, gate, up, down, dy, "swiglu"), ["x", "gate", "up", "down"])


@pytest.mark.parametrize("t", [5, 90])
def test_rows_asked_for_are_not_scaled(t):
    x, gate, up, down, dy = draw(t, t, 136, 72, F16)
    dy = (dy.float() * 2.0**-10).half()
    alone = gated_ffn_gradients(x, dy, gate, up, down, inputs=False, weights=False)
    for part in ({}, {"inputs": False}, {"weights": False}):
        got = gated_ffn_gradients(x, dy, gate, up, down, **part)
        for name in ("gate_rows", "up_rows", "middle"):
            assert torch.equal(getattr(got, name), getattr(alone, name))


@pytest.mark.parametrize("t", [4, 70])
def test_gradients_of_nothing(t):
    x, gate, up, down, dy = draw(t, t, 72, 136, F16)
    for zeros in ((dy,), (x,), (down,)):
        a, b, c = (torch.zeros_like(v) if any(v is z for z in zeros) else v for v in (x, dy, down))
        got = gated_ffn_gradients(a, b, gate, up, c)
        for name, (value, bound) in want(a, gate, up, c, b, "swiglu").items():
            assert bool(((getattr(got, name).double() - value).abs() <= bound).all()), name


@pytest.mark.parametrize("t", [6, 50, 300])
def test_rows_that_are_not_finite_stay_alone(t):
    """They do not count for the scale."""

    x, gate, up, down, dy = draw(t, t, 264, 200, F16)
    dy = (dy.float() * 2.0**-14).half()
    bad_x, bad_dy = x.clone(), dy.clone()
    bad_x[1], bad_x[3, 5], bad_dy[4, 7], bad_dy[2] = float("nan"), float("inf"), float("-inf"), float("nan")
    fine = [0, *range(5, t)]
    got, expected = gated_ffn_gradients(bad_x, bad_dy, gate, up, down), want(x, gate, up, down, dy, "swiglu")["x"]
    assert bool(((got.x.double() - expected[0]).abs() <= expected[1])[fine].all())
    assert not torch.isfinite(got.x[1:5]).all(1).any()


def test_captured_gradients_are_scaled_by_the_replays_rows():
    x, gate, up, down, dy = draw(3, 40, 264, 136, F16)
    static_x, static_dy = x.clone(), dy.clone()
    gated_ffn_gradients(static_x, static_dy, gate, up, down)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = gated_ffn_gradients(static_x, static_dy, gate, up, down)
    for i, size in enumerate((1e-6, 1.0, 1e-4, 1e-5)):
        a, _, _, _, b = draw(10 + i, 40, 264, 136, F16)
        static_x.copy_(a)
        static_dy.copy_(b.float() * size)
        graph.replay()
        torch.cuda.synchronize()
        for v, w in zip(vars(gated_ffn_gradients(static_x, static_dy, gate, up, down)).values(), vars(got).values()):
            assert torch.equal(v, w)


def test_two_replays_in_turn_keep_their_scales():
    """Two captured graphs of calls of one size: each has its own workspace."""

    graphs = []
    for i, size in enumerate((1e-6, 1.0)):
        x, gate, up, down, dy = draw(20 + i, 70, 264, 136, F16)
        args = x, (dy.float() * size).half(), gate, up, down
        gated_ffn_gradients(*args)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = gated_ffn_gradients(*args)
        graphs.append((graph, args, got))
    for i in (0, 1, 1, 0):
        graph, args, got = graphs[i]
        graph.replay()
        torch.cuda.synchronize()
        for v, w in zip(vars(gated_ffn_gradients(*args)).values(), vars(got).values()):
            assert torch.equal(v, w)


@pytest.mark.parametrize("t", [8, 100])
def test_views_and_a_lone_row(t):
    x, gate, up, down, dy = draw(t, t, 264, 136, F16)
    dy = (dy.float() * 2.0**-16).half()
    wide = torch.full((t, 300), float("nan"), dtype=F16, device="cuda")
    apart, other = wide[:, :264], torch.full((264, 160), float("nan"), dtype=F16, device="cuda")[:, :136]
    apart.copy_(dy)
    other.copy_(down)
    for a, b in zip(vars(gated_ffn_gradients(x, apart, gate, up, other)).values(), vars(gated_ffn_gradients(x, dy, gate, up, down)).values()):
        assert torch.equal(a, b)
    one = gated_ffn_gradients(x[:1], dy[:1].as_strided((1, 264), (3, 1)), gate, up, down)
    check(vars(one), want(x[:1], gate, up, down, dy[:1], "swiglu"), ["x", "gate", "up", "down"])


@pytest.mark.parametrize("size", [1.0, 1e-4, 1e-6])
@pytest.mark.parametrize("t", [5, 100])
def test_guidance_of_small_gradients(t, size):
    """The factors dG and dU: FP32 sums of ``hidden`` products, times a slope, rounded to f16 once, or off by 2^-25 of dy's largest
    over 2^-4."""

    x, gate, up, down, dy = draw(t, t, 264, 136, F16)
    dy = (dy.float() * size).half()
    guidance = expert_guidance(x, dy, gate, up, down, anchor_id="a", objective_id="o", activation="swiglu")
    X, G, U, D, Y = (v.double() for v in (x, gate, up, down, dy))
    g, u = X @ G.T, X @ U.T
    _, by_g, by_u = slopes(g, u, "swiglu")
    dg, du = (265 * V * (X.abs() @ w.abs().T) for w in (G, U))
    slope_g, slope_u = 1.1 * u.abs() * dg + 1.1 * du + 32 * V * 1.1 * u.abs(), 1.1 * (dg + du) + 32 * V * 1.1 * g.abs()
    rows, rows_off = Y @ D, 265 * V * (Y.abs() @ D.abs())
    for name, by, slope in (("w1", by_g, slope_g), ("w3", by_u, slope_u)):
        value = rows * by
        off = rows_off * by.abs() + (rows.abs() + rows_off) * slope + 4 * V * value.abs()
        bound = off + 2.0**-11 * (value.abs() + off) + 2.0**-21 * float(Y.abs().max())
        assert float(((guidance[name].right.double() - value).abs() / bound).max()) <= 1, name
        assert torch.equal(guidance[name].left, x.T.float())


@pytest.mark.parametrize("t", [12, 90])
def test_large_gradients_are_not_scaled(t):
    """The bound is over 2^15, the rows are not: they go as they are."""

    x, gate, up, down, dy = spread(t, t, 264, 136, 128.0, 1.0)
    check(vars(gated_ffn_gradients(x, dy, gate, up, down)), want(x, gate, up, down, dy, "swiglu"), ["x", "gate", "up", "down"])
