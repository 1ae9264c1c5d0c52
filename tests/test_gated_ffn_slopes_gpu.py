"""SiTU's slopes where its tanh and sigmoid are next to 1, against 64 bits."""

from __future__ import annotations

import pytest
import torch

from qsrt_amd.gated_ffn import gated_ffn_gradients

pytestmark = pytest.mark.gpu
V = 2.0**-24


def exact(g, u):
    """Slopes by g and u in 64 bits, and the sizes of the terms that they are sums of: 1 - tanh^2 as 1 / cosh^2, 1 - sigmoid(g) as
    sigmoid(-g)."""

    s, rest = torch.sigmoid(g), torch.sigmoid(-g)
    f = 4 * torch.tanh(g / 4) * s
    parts = s / torch.cosh(g / 4) ** 2, f * rest
    b = 25 * torch.tanh(u / 25)
    return b * (parts[0] + parts[1]), b.abs() * (parts[0] + parts[1].abs()), f / torch.cosh(u / 25) ** 2


@pytest.mark.parametrize("dtype,least,most,size", [(torch.bfloat16, -40.0, 40.0, 1.0), (torch.float16, 14.0, 40.0, 2.0**12)])
@pytest.mark.parametrize("t", [40, 126])
def test_saturated_slopes(t, dtype, least, most, size):
    """G of a column and U of a row as given (a product with 1 and zeros), dM = ``size`` everywhere.

    A slope is a dozen FP32 operations and functions of 2 ulp or better, 32 V of its terms; the arguments of the exponentials behind
    them are up to 40 and rounded once or twice (64 V); dM is exact, the result is rounded once."""

    g = torch.linspace(least, most, 168, device="cuda").to(dtype)
    u = torch.linspace(-250, 250, t, device="cuda").to(dtype)
    x, gate, up, down, dy = (torch.zeros(shape, dtype=dtype, device="cuda") for shape in ((t, 8), (168, 8), (168, 8), (8, 168), (t, 8)))
    x[:, 0], x[:, 1], gate[:, 0], up[:, 1], down[0], dy[:, 0] = 1, u, g, 1, 1, size
    got = gated_ffn_gradients(x, dy, gate, up, down, activation="situ", inputs=False, weights=False)
    by_g, terms, by_u = exact(g.double()[None], u.double()[:, None])
    eps, tiny = torch.finfo(dtype).eps / 2, float(torch.finfo(dtype).smallest_normal) * torch.finfo(dtype).eps / 2
    for name, value, of in (("gate_rows", by_g, terms), ("up_rows", by_u, by_u.abs())):
        bound = size * (eps * value.abs() + 96 * V * of) + tiny
        off = (getattr(got, name).double() - size * value).abs()
        assert float((off / bound).max()) <= 1, name
