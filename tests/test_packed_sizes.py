"""Workspace functions of packed serving take any numbers, and nothing is allocated for a call that is refused."""

from __future__ import annotations

import ctypes
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from qsrt_amd import _native

ROOT = Path(__file__).resolve().parents[1]
needs_library = pytest.mark.skipif(not _native.LIB_PATH.exists(), reason="the native library is not built")
BIG = (1 << 62, 1 << 60, -(1 << 63), (1 << 63) - 1, -1)


@needs_library
def test_route_workspace_of_any_sizes():
    """In a process of its own: an integer division by an overflowed product would end this one."""

    code = f"""
from qsrt_amd import _native
need = _native.lib().qsrt_route_workspace_bytes
for v in {BIG}:
    for sizes in ((v, 8, 1024), (v, 8, 8), (4, v, 8), (4, 8, v), (v, v, v)):
        assert need(*sizes) == 0, sizes
assert need(0, 256, 8) == 0 and need(4, 256, 1025) == 0 and need(4, 0, 8) == 0 and need(4, 256, 8) >= 128
"""
    run = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True)
    assert run.returncode == 0, (run.returncode, run.stderr)


def struct(**changes):
    fields = {"words": 1, "key_stride": 0, "records": 1, "record_stride": 0, "suh": 1, "suh_stride": 0, "svh": 1,
              "svh_stride": 0, "rows": 256, "cols": 128, "rate_axis": 0, "rates": 8}
    fields.update(changes)
    return ctypes.byref(_native.PackedMatrixStruct(**fields))


@needs_library
@pytest.mark.parametrize("experts,words", [(1024, "too many tokens"), (8, None)])
def test_a_layer_counts_the_threads_of_router_and_rotation_together(experts, words):
    """2^20 tokens of 3968 channels: the rotation alone has 0.97 of the threads a launch can have."""

    at = 1 << 12  # an aligned address; nothing reads it
    tables = (ctypes.c_void_p * 3)(at, at, at)
    up = struct(words=at, records=at, suh=at, svh=at, rows=3968, cols=128)
    down = struct(words=at, records=at, suh=at, svh=at, rows=128, cols=3968)
    rc = _native.lib().qsrt_packed_moe_layer(up, up, down, ctypes.addressof(tables), experts, 0, None, None, at, 3968, None, 0, 1,
                                             1.0, at, 3968, 0, 1 << 20, 1, at, at, at, 3968, None, 0, None)
    message = _native.lib().qsrt_last_error().decode()
    if words:
        assert rc == -1 and words in message, (rc, message)
    else:  # goes on to its workspace, or without a GPU to the device
        assert rc in (-2, -3), (rc, message)


@needs_library
@pytest.mark.parametrize("x_ld,out_ld", [(3, 128), (256, 1), (0, 0)])
def test_leading_dimensions_of_a_lone_row(x_ld, out_ld):
    """Taken as they are; of two rows they are refused."""

    at, lib = 1 << 12, _native.lib()
    tables = (ctypes.c_void_p * 3)(at, at, at)
    w = struct(words=at, records=at, suh=at, svh=at)
    down = struct(words=at, records=at, suh=at, svh=at, rows=128, cols=256)
    for n, codes in ((1, (-2, -3)), (2, (-1,))):
        assert lib.qsrt_adapter_linear(w, ctypes.addressof(tables), None, None, None, 0, 0, at, x_ld, 0, n, None, at, out_ld, None, 0,
                                       None) in codes
        assert lib.qsrt_packed_moe(w, w, down, ctypes.addressof(tables), 4, 0, None, None, at, x_ld, 0, n, 1, at, at, at, out_ld,
                                   None, 0, None) in codes
        if x_ld != 256:
            assert lib.qsrt_route(at, x_ld, at, 256, 0, n, 256, 8, 1, None, 0, 1, 1.0, at, at, None, 0, None) in codes
            assert lib.qsrt_route(at, 256, at, x_ld, 0, 3, 256, n, 1, None, 0, 1, 1.0, at, at, None, 0, None) in codes


@pytest.mark.gpu
def test_product_workspaces_of_any_sizes():
    up, down, lib = struct(), struct(rows=128, cols=256), _native.lib()
    assert lib.qsrt_packed_moe_workspace_bytes(up, up, down, 4, 2, 2) > 0
    assert lib.qsrt_adapter_linear_workspace_bytes(up, 3, 2, 16) > 0
    for tokens, k in ((1 << 20, 2), (1 << 21, 1), (-1, 2), (2, -1), (2, 0), (1 << 62, 4), (1 << 57, 1)):
        assert lib.qsrt_packed_moe_workspace_bytes(up, up, down, 4, tokens, k) == 0
    for experts in (0, -1, 8192, 1 << 62):
        assert lib.qsrt_packed_moe_workspace_bytes(up, up, down, experts, 2, 2) == 0
    for rows, adapters, rank in (((1 << 20) + 1, 0, 0), (-1, 0, 0), (1 << 57, 0, 0), (1 << 62, 2, 16), (3, -1, 16), (3, 2, 8),
                                 (3, 2, 144), (3, 2, -16), (3, 1 << 62, 16)):
        assert lib.qsrt_adapter_linear_workspace_bytes(up, rows, adapters, rank) == 0
    for bad in (struct(rows=1 << 40, cols=1 << 40), struct(rows=0), struct(cols=-128), struct(rows=96), struct(rates=0)):
        assert lib.qsrt_packed_moe_workspace_bytes(bad, bad, bad, 4, 2, 2) == 0
        assert lib.qsrt_adapter_linear_workspace_bytes(bad, 3, 0, 0) == 0


@pytest.mark.gpu
def test_a_refused_call_allocates_no_workspace():
    import numpy as np

    from qsrt_amd.packed_linear import PackedLinear, packed_linear
    from test_packed_serving_gpu import LUTS, Experts, payload

    experts = Experts(97, 128, 128, 2, (3,)).packed
    t, k = 1 << 17, 9  # 2^20 pairs and 2^17 more; every pair would take a kilobyte or more
    ids, weights = torch.zeros((t, k), dtype=torch.int32, device="cuda"), torch.ones((t, k), device="cuda")
    x = torch.zeros((t, 128), dtype=torch.bfloat16, device="cuda")
    p = payload(np.random.default_rng(98), 4096, 128, (2,) * 32, "k")
    linear = PackedLinear(*(torch.from_numpy(v).cuda() for v in p), (2,) * 32, LUTS)
    rows = torch.zeros((1, 4096), dtype=torch.bfloat16, device="cuda").expand(1 << 20, -1)
    for call, words in ((lambda: experts(x, weights, ids), "2\\^20"), (lambda: packed_linear(rows, linear), "rows")):
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        with pytest.raises(ValueError, match=words):
            call()
        most = torch.cuda.max_memory_allocated() - before
        # the result, and for the projection a copy of the rows that overlap
        assert most <= (x.numel() * 2 if words != "rows" else (1 << 20) * (4096 + 128) * 2) + (1 << 21), most
