"""The norms, gate and residual between two blocks, and their gradients, against 64-bit formulas.

Bounds: statistics and products are a few FP32 operations on the unrounded inputs, sums over a row or over all rows are off by
``(K + 1) 2^-24`` of the absolute sum; a 16-bit result is rounded once, ``finfo(type).eps / 2`` of itself."""

from __future__ import annotations

import pytest
import torch

from qsrt_amd.block_norm import residual_norm, rms_norm

pytestmark = pytest.mark.gpu
V = 2.0**-24
EPS = 1e-6


def draw(seed, t, hidden, dtype, residual, post, gate, params):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, scale=1.0):
        return scale * torch.randn(shape, generator=g, device="cuda")

    v = {"residual": (3 * normal(t, hidden)).to(residual), "y": normal(t, hidden).to(dtype),
         "weight": (1 + normal(hidden, scale=0.2)).to(params)}
    v["post"] = (1 + normal(hidden, scale=0.2)).to(params) if post else None
    v["gate"] = {"none": None, "channel": (0.5 + normal(hidden, scale=0.2)).to(params),
                 "row": torch.sigmoid(normal(t, 1)).to(params)}[gate]
    return v, normal(t, hidden, scale=0.2).to(residual), normal(t, hidden, scale=0.2).to(dtype)


def want(v, dsum, dn, scale):
    """Values in 64 bits by differentiating, and what each is a sum of, in absolute values."""

    leaf = {k: t.double().requires_grad_() for k, t in v.items() if t is not None}
    z = leaf["y"]
    if "post" in leaf:
        sy = (z.square().mean(1, keepdim=True) + EPS).rsqrt()
        yhat = z * sy
        z = yhat * leaf["post"]
    gate = leaf.get("gate", torch.ones(1, dtype=torch.float64, device="cuda"))
    h = scale * leaf["residual"] + gate * z
    sh = (h.square().mean(1, keepdim=True) + EPS).rsqrt()
    n = leaf["weight"] * h * sh
    grads = dict(zip(leaf, torch.autograd.grad((h, n), list(leaf.values()), (dsum.double(), dn.double()))))
    out = {"h": h.detach(), "n": n.detach()} | {"d" + k: g for k, g in grads.items()}
    with torch.no_grad():
        hidden = h.shape[1]
        size_h = abs(scale) * leaf["residual"].abs() + (gate * z).abs()
        e = (dn.double() * leaf["weight"]).abs()
        dh = dsum.double().abs() + sh * (e + size_h * sh * sh * (e * size_h).mean(1, keepdim=True))
        size = {"h": size_h, "n": leaf["weight"].abs() * size_h * sh, "dresidual": abs(scale) * dh}
        size["dweight"] = (dn.double().abs() * size_h * sh).sum(0)
        size["dy"] = gate.abs() * dh
        if "post" in leaf:
            d = gate.abs() * dh * leaf["post"].abs()
            size["dpost"] = (gate.abs() * dh * yhat.abs()).sum(0)
            size["dy"] = sy * (d + yhat.abs() * (d * yhat.abs()).mean(1, keepdim=True))
        if "gate" in leaf:
            size["dgate"] = (dh * z.abs()).sum(0) if leaf["gate"].dim() == 1 else (dh * z.abs()).sum(1, keepdim=True)
    return out, size, hidden


def check(got, expected, size, hidden, t):
    for name, value in expected.items():
        if name not in got:
            continue
        u = torch.finfo(got[name].dtype).eps / 2
        # a statistic is off by half a row's sum (the root), twice at most in a chain; 64 for the operations themselves
        bound = (2 * hidden + (t if name in ("dweight", "dpost", "dgate") else 0) + 64) * V * size[name]
        bound = bound + u * (value.abs() + bound) + float(torch.finfo(got[name].dtype).smallest_normal) * u
        off = (got[name].double() - value).abs()
        assert torch.isfinite(off).all(), name
        worst = float((off / bound).max())
        assert worst <= 1, f"{name}: {worst:.3g} times the bound"


def call(v, dsum, dn, scale):
    leaf = {k: t.detach().requires_grad_() for k, t in v.items() if t is not None}
    h, n = residual_norm(leaf["residual"], leaf["y"], leaf["weight"], post_weight=leaf.get("post"), gate=leaf.get("gate"),
                         scale=scale, eps=EPS)
    grads = torch.autograd.grad((h, n), list(leaf.values()), (dsum, dn))
    return {"h": h.detach(), "n": n.detach()} | {"d" + k: g for k, g in zip(leaf, grads)}


SIZES = [(1, 8), (1, 7168), (3, 2048), (7, 2056), (300, 520), (513, 4104), (33, 8200), (5, 16384), (1100, 5120),
         (8200, 264)]


@pytest.mark.parametrize("gate", ["none", "channel", "row"])
@pytest.mark.parametrize("t,hidden", SIZES)
def test_against_64_bits(t, hidden, gate):
    at = SIZES.index((t, hidden)) + ("none", "channel", "row").index(gate)
    dtype = (torch.bfloat16, torch.float16)[at % 2]
    residual, params = (torch.float32, dtype)[at // 2 % 2], (torch.float32, dtype)[at // 3 % 2]
    for post in (True, False):
        v, dsum, dn = draw(at, t, hidden, dtype, residual, post, gate, params)
        scale = (1.0, 0.5)[at % 2]
        expected, size, width = want(v, dsum, dn, scale)
        got = call(v, dsum, dn, scale)
        for name, g in got.items():
            source = {"h": v["residual"], "n": v["y"]}.get(name, v.get(name[1:]))
            assert g.dtype == source.dtype and g.shape == source.shape
        check(got, expected, size, width, t)


@pytest.mark.parametrize("t,hidden", [(1, 64), (130, 1000)])
@pytest.mark.parametrize("source", [torch.float32, torch.bfloat16])
def test_first_norm(t, hidden, source):
    g = torch.Generator(device="cuda").manual_seed(t)
    x = torch.randn((t, hidden), generator=g, device="cuda").to(source).requires_grad_()
    weight = (1 + 0.2 * torch.randn(hidden, generator=g, device="cuda")).requires_grad_()
    n = rms_norm(x, weight, eps=EPS, dtype=torch.bfloat16)
    dn = torch.randn((t, hidden), generator=g, device="cuda").to(torch.bfloat16)
    dx, dw = torch.autograd.grad(n, (x, weight), dn)
    v = {"residual": x.detach(), "y": torch.zeros((t, hidden), device="cuda"), "weight": weight.detach(), "post": None, "gate": None}
    expected, size, width = want(v, torch.zeros((t, hidden), device="cuda"), dn, 1.0)
    got = {"n": n.detach(), "dresidual": dx, "dweight": dw}
    assert dx.dtype == source and dw.dtype == torch.float32
    check(got, expected, size, width, t)
