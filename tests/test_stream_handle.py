"""Tensors in host memory are stopped before a launch: kernels would read their addresses."""

from __future__ import annotations

import pytest
import torch

from qsrt_amd import _native


@pytest.mark.parametrize("device", ["cpu", "meta"])
def test_no_stream_of_a_device_without_one(device):
    with pytest.raises(ValueError, match="CUDA device"):
        _native.stream_handle(torch.device(device))


@pytest.mark.gpu
def test_the_stream_is_the_current_one():
    device = torch.device("cuda:0")
    assert _native.stream_handle(device) == torch.cuda.current_stream(device).cuda_stream
    assert _native.stream_handle(torch.device("cuda")) == torch.cuda.current_stream().cuda_stream
    with torch.cuda.stream(torch.cuda.Stream()):
        assert _native.stream_handle(device) == torch.cuda.current_stream(device).cuda_stream
