"""Gradients of the norms for rows far from 1, against the 64-bit formulas and bounds of ``test_block_norm_gpu``: the inverse root
of a row's mean square, and its second and third power, may leave FP32's range by themselves, what they multiply does not."""

from __future__ import annotations

import pytest
import torch

import test_block_norm_gpu as plain
from qsrt_amd.block_norm import rms_norm

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def scaled(v, by):
    """Rows of residual and y times ``by`` (a power of two, [T, 1])."""

    return v | {k: (v[k].float() * by).to(v[k].dtype) for k in ("residual", "y")}


@pytest.mark.parametrize("residual", [torch.float32, BF16])
@pytest.mark.parametrize("post,gate", [(True, "channel"), (False, "row"), (False, "none"), (True, "row")])
@pytest.mark.parametrize("t,hidden,power", [(3, 264, -50), (5, 1032, -43), (5, 1032, 40), (40, 264, 47), (4, 8200, 54), (300, 64, None)])
def test_rows_of_any_size(t, hidden, power, post, gate, residual, monkeypatch):
    monkeypatch.setattr(plain, "EPS", 0.0 if power is None or power < 0 else 1e-6)
    v, dsum, dn = plain.draw(t + hidden, t, hidden, BF16, residual, post, gate, torch.float32)
    powers = torch.full((t, 1), 0.0 if power is None else power, device="cuda")
    if power is None:  # every row its own
        powers = torch.randint(-50, 50, (t, 1), generator=torch.Generator(device="cuda").manual_seed(t), device="cuda").float()
    v = scaled(v, torch.exp2(powers))
    # of the sum's own gradient nothing, or as much as the norm's: else it hides what the norm passes on
    for d in (torch.zeros_like(dsum), (dsum.float() * torch.exp2(-powers)).to(residual)):
        expected, size, width = plain.want(v, d, dn, 0.5)
        plain.check(plain.call(v, d, dn, 0.5), expected, size, width, t)


@pytest.mark.parametrize("eps", [1e-30, 1e-12])
@pytest.mark.parametrize("post,gate", [(True, "channel"), (False, "row"), (False, "none")])
def test_rows_of_zeros_leave_the_others_gradients_alone(post, gate, eps, monkeypatch):
    monkeypatch.setattr(plain, "EPS", eps)
    v, dsum, dn = plain.draw(7, 6, 264, BF16, torch.float32, post, gate, torch.float32)
    for k in ("residual", "y"):
        v[k][2] = v[k][5] = 0
    expected, size, width = plain.want(v, dsum, dn, 1.0)
    plain.check(plain.call(v, dsum, dn, 1.0), expected, size, width, 6)


@pytest.mark.parametrize("power", [-45, 45])
def test_first_norm_of_rows_of_any_size(power, monkeypatch):
    monkeypatch.setattr(plain, "EPS", 0.0)
    g = torch.Generator(device="cuda").manual_seed(3)
    x = (torch.randn((33, 520), generator=g, device="cuda") * 2.0**power).requires_grad_()
    weight = (1 + 0.2 * torch.randn(520, generator=g, device="cuda")).requires_grad_()
    dn = torch.randn((33, 520), generator=g, device="cuda").to(BF16)
    dx, dw = torch.autograd.grad(rms_norm(x, weight, eps=0.0, dtype=BF16), (x, weight), dn)
    zero = torch.zeros((33, 520), device="cuda")
    v = {"residual": x.detach(), "y": zero, "weight": weight.detach(), "post": None, "gate": None}
    expected, size, width = plain.want(v, zero, dn, 1.0)
    plain.check({"dresidual": dx, "dweight": dw}, expected, size, width, 33)
