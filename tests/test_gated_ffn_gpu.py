"""The gated feed-forward block and its gradients against 64-bit products, element by element.

Bounds, with ``u = finfo(type).eps / 2`` for a rounding to the type and ``v = 2^-24`` for FP32: a sum of K products in any
order is off by at most ``(K + 1) v sum|a||b|`` (products of 16-bit values are exact in FP32), a rounded result by ``u`` of
itself, a row between two products by ``u`` of itself (as two values by ``u^2``); what that does to the result goes through
absolute values.  Activations and slopes are a dozen FP32 operations and library functions of 2 ulp or better: 32 v of their
factors.  The slopes change by at most 1.1 (by the other row) and 1.1 |u| (by their own) for each unit of G and U."""

from __future__ import annotations

import pytest
import torch

from qsrt_amd.gated_ffn import gated_ffn, gated_ffn_gradients

pytestmark = pytest.mark.gpu
V = 2.0**-24


def draw(seed, t, hidden, inter, dtype):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, scale):
        return (scale * torch.randn(shape, generator=g, device="cuda")).to(dtype)

    x = normal(t, hidden, scale=1.5)
    gate, up = (normal(inter, hidden, scale=hidden**-0.5) for _ in range(2))
    return x, gate, up, normal(hidden, inter, scale=inter**-0.5), normal(t, hidden, scale=0.25)


def slopes(g, u, activation):
    s = torch.sigmoid(g)
    if activation == "swiglu":
        return g * s * u, u * s * (1 + g * (1 - s)), g * s
    a, b = torch.tanh(g / 4), torch.tanh(u / 25)
    f = 4 * a * s
    return f * 25 * b, 25 * b * ((1 - a * a) * s + f * (1 - s)), f * (1 - b * b)


def want(x, gate, up, down, dy, activation, pieces):
    """``{name: (value, bound)}`` in 64 bits."""

    u = torch.finfo(x.dtype).eps / 2
    tiny = float(torch.finfo(x.dtype).smallest_normal) * u  # below the smallest normal value a rounding is absolute
    row = u if pieces == 1 else u * u
    x, gate, up, down, dy = (t.double() for t in (x, gate, up, down, dy))
    t, hidden = x.shape
    inter = gate.shape[0]
    g, p = x @ gate.T, x @ up.T
    dg, dp = ((hidden + 1) * V * (x.abs() @ w.abs().T) for w in (gate, up))
    m, by_g, by_u = slopes(g, p, activation)
    flow = 32 * V
    mag_m, mag_g, mag_u = g.abs() * p.abs(), 1.1 * p.abs(), 1.1 * g.abs()
    dm = mag_g * dg + mag_u * dp + dg * dp + flow * mag_m
    slope_g, slope_u = 1.1 * p.abs() * dg + 1.1 * dp + flow * mag_g, 1.1 * (dg + dp) + flow * mag_u

    def rounded(value, off, by=u):
        return off + by * (value.abs() + off) + tiny

    m_off = rounded(m, dm, row)

    def product(a, a_off, b, b_off, k):  # a [.., k] by b [k, ..]
        off = a_off @ b.abs() + a.abs() @ b_off if b_off is not None else a_off @ b.abs()
        return off + (k + 1) * V * ((a.abs() + a_off) @ (b.abs() if b_off is None else b.abs() + b_off))

    out = {"middle": (m, rounded(m, dm))}
    y = m @ down.T
    out["y"] = (y, rounded(y, product(m, m_off, down.T, None, pieces * inter)))
    rows = dy @ down
    rows_off = (hidden + 1) * V * (dy.abs() @ down.abs())
    grads = []
    for name, by, off in (("gate_rows", by_g, slope_g), ("up_rows", by_u, slope_u)):
        value = rows * by
        value_off = rows_off * by.abs() + (rows.abs() + rows_off) * off + 4 * V * value.abs()
        out[name] = (value, rounded(value, value_off))
        grads.append((value, rounded(value, value_off, row)))
    (vg, og), (vu, ou) = grads
    dx = vg @ gate + vu @ up
    out["x"] = (dx, rounded(dx, product(torch.cat((vg, vu), 1), torch.cat((og, ou), 1), torch.cat((gate, up)), None,
                                        2 * pieces * inter)))
    for name, v, off in (("gate", vg, og), ("up", vu, ou)):
        dw = v.T @ x
        out[name] = (dw, rounded(dw, product(v.T.contiguous(), off.T.contiguous(), x, None, pieces * t)))
    dw = dy.T @ m
    out["down"] = (dw, rounded(dw, product(m.T.contiguous(), m_off.T.contiguous(), dy, None, pieces * t).T))
    return out


def check(got, expected, names):
    for name in names:
        value, bound = expected[name]
        off = (got[name].double() - value).abs()
        assert torch.isfinite(off).all(), name
        worst = float((off / bound).max())
        assert worst <= 1, f"{name}: {worst:.3g} times the bound"


SIZES = [(1, 8, 8), (1, 256, 512), (2, 200, 24), (5, 1032, 136), (16, 72, 1000), (31, 264, 128), (32, 512, 256), (33, 64, 72),
         (63, 328, 520), (64, 1000, 64), (65, 128, 200), (129, 520, 392), (333, 2056, 1400), (700, 384, 1032)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,hidden,inter", SIZES)
def test_against_64_bits(t, hidden, inter, dtype):
    activation = ("swiglu", "situ")[(t + hidden // 8) % 2]
    x, gate, up, down, dy = draw(t + hidden, t, hidden, inter, dtype)
    expected = want(x, gate, up, down, dy, activation, 1 if t > 64 else 2)
    check({"y": gated_ffn(x, gate, up, down, activation=activation)}, expected, ["y"])
    got = gated_ffn_gradients(x, dy, gate, up, down, activation=activation)
    check(vars(got), expected, ["middle", "gate_rows", "up_rows", "x", "gate", "up", "down"])


@pytest.mark.parametrize("activation", ["swiglu", "situ"])
def test_many_rows(activation):
    x, gate, up, down, dy = draw(3, 4100, 4104, 2080, torch.bfloat16)
    expected = want(x, gate, up, down, dy, activation, 1)
    leaves = [v.requires_grad_() for v in (x, gate, up, down)]
    y = gated_ffn(*leaves, activation=activation)
    grads = torch.autograd.grad(y, leaves, dy)
    check({"y": y.detach()} | dict(zip(("x", "gate", "up", "down"), grads)), expected, ["y", "x", "gate", "up", "down"])
