"""Further arguments that the entries of the dense block refuse on the host: no GPU is needed here."""

from __future__ import annotations

import pytest
import torch

from qsrt_amd.gated_ffn import gated_ffn_gradients
from test_gated_ffn_entries import ffn, ffn_backward, native, norm, norm_backward, refused


@native
@pytest.mark.parametrize("hidden", [8 - (1 << 32), 64 - (1 << 33), -8, (1 << 32) + 64, 1 << 62])
def test_channels_that_would_fit_in_32_bits(hidden):
    for rows in (1, 3):
        refused(norm(rows=rows, hidden=hidden), "channels")
        refused(norm_backward(rows=rows, hidden=hidden), "channels")
    refused(ffn(hidden=hidden), "channels")
    refused(ffn_backward(inter=hidden), "channels")


@pytest.mark.gpu
def test_a_gradient_on_another_device_is_named():
    x, w, d = (torch.zeros(shape, dtype=torch.bfloat16, device="cuda") for shape in ((2, 16), (8, 16), (16, 8)))
    with pytest.raises(ValueError, match="dy must"):
        gated_ffn_gradients(x, x.cpu(), w, w, d)
