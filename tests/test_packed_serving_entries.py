"""The C entries of packed serving refuse bad arguments on the host, before any GPU call: no GPU is needed here."""

import ctypes

import numpy as np
import pytest

from qsrt_amd import _native

pytestmark = pytest.mark.skipif(not _native.LIB_PATH.exists(), reason="the native library is not built")

BUF = np.zeros(4096 + 64, dtype=np.uint8)
P = (BUF.ctypes.data + 63) // 64 * 64  # an aligned address; nothing reads it
LUTS = (ctypes.c_void_p * 3)(P, P, P)


def matrix(**changes):
    fields = {"words": P, "key_stride": 0, "records": P, "record_stride": 0, "suh": P, "suh_stride": 0, "svh": P,
              "svh_stride": 0, "rows": 256, "cols": 128, "rate_axis": 0, "rates": 8}
    fields.update(changes)
    return _native.PackedMatrixStruct(**fields)


def refused(rc, words):
    message = _native.lib().qsrt_last_error().decode()
    assert rc == -1 and words in message, (rc, message)


def route(**changes):
    a = {"x": P, "x_ld": 256, "weight": P, "weight_ld": 256, "dtype": 0, "tokens": 2, "hidden": 256, "experts": 8, "k": 2,
         "bias": None, "scoring": 0, "normalize": 1, "scale": 1.0, "weights": P, "ids": P, "ws": P, "ws_bytes": 1 << 20,
         "stream": None}
    a.update(changes)
    return _native.lib().qsrt_route(*a.values())


@pytest.mark.parametrize("changes,words", [
    ({"tokens": -1}, "sizes"), ({"tokens": (1 << 20) + 1}, "sizes"), ({"experts": 1025}, "sizes"), ({"experts": 0}, "sizes"),
    ({"hidden": 0}, "sizes"), ({"hidden": 252}, "8 channels"), ({"x_ld": 255}, "8 channels"), ({"x": P + 2}, "16-byte"),
    ({"x_ld": 128}, "rows"), ({"k": 0}, "k must"), ({"k": 9}, "k must"), ({"k": 65, "experts": 100}, "k must"),
    ({"dtype": 2}, "dtype"), ({"scoring": 2}, "scoring"), ({"x": None}, "null"), ({"ids": None}, "null"),
])
def test_route_refuses(changes, words):
    refused(route(**changes), words)


def test_route_names_the_workspace_it_needs():
    need = _native.lib().qsrt_route_workspace_bytes(2, 256, 8)
    assert need >= 2 * 8 * 4
    for changes in ({"ws_bytes": need - 1}, {"ws": None}):
        assert route(**changes) not in (0, -1)
        assert str(need) in _native.lib().qsrt_last_error().decode()


def linear(w, **changes):
    a = {"luts": ctypes.addressof(LUTS), "a": P, "b": P, "scale": P, "adapters": 2, "rank": 16, "x": P, "x_ld": 256, "dtype": 0,
         "rows": 3, "ids": P, "out": P, "out_ld": 128, "ws": P, "ws_bytes": 0, "stream": None}
    a.update(changes)
    return _native.lib().qsrt_adapter_linear(ctypes.byref(w) if w else None, *a.values())


@pytest.mark.parametrize("changes,words", [
    ({"words": None}, "null"), ({"records": None}, "null"), ({"suh": None}, "null"), ({"rows": 200}, "multiples of 128"),
    ({"cols": 0}, "multiples of 128"), ({"rows": 1 << 16, "cols": 1 << 16}, "too large"), ({"rows": 1 << 23}, "too large"),
    ({"rate_axis": 2}, "rate_axis"), ({"rates": 0}, "rates"), ({"rates": 2}, "rates"), ({"words": P + 2}, "4-byte"),
    ({"key_stride": -2}, "negative"), ({"key_stride": 3}, "4-byte"), ({"suh": P + 2}, "8-byte"), ({"svh_stride": 2}, "8-byte"),
])
def test_matrices_are_checked(changes, words):
    refused(linear(matrix(**changes)), words)


@pytest.mark.parametrize("changes,words", [
    ({"luts": None}, "label table"), ({"rows": -1}, "rows"), ({"rows": (1 << 20) + 1}, "rows"), ({"dtype": 3}, "dtype"),
    ({"adapters": -1}, "adapters"), ({"adapters": 8192}, "adapters"), ({"rank": 8}, "rank"), ({"rank": 144}, "rank"),
    ({"rank": 40}, "rank"), ({"a": None}, "adapters need"), ({"a": P + 8}, "16-byte"), ({"ids": None}, "adapters need"),
    ({"x": None}, "null"), ({"x_ld": 252}, "aligned"), ({"x": P + 8}, "aligned"), ({"out": P + 2}, "aligned"),
    ({"out_ld": 127}, "aligned"), ({"out_ld": 124}, "aligned"),
])
def test_adapter_projection_refuses(changes, words):
    refused(linear(matrix(), **changes), words)
    assert linear(matrix(), rows=0) == 0  # nothing to do, nothing launched


def test_too_many_rows_for_one_launch():
    big = matrix(rows=1 << 14, cols=128)
    refused(linear(big, rows=1 << 18, x_ld=1 << 14), "too many rows")


def moe(w1, w3, w2, **changes):
    a = {"luts": ctypes.addressof(LUTS), "experts": 4, "activation": 0, "pre": None, "post": None, "x": P, "x_ld": 256, "dtype": 0, "tokens": 2, "k": 2,
         "ids": P, "weights": P, "out": P, "out_ld": 256, "ws": P, "ws_bytes": 0, "stream": None}
    a.update(changes)
    return _native.lib().qsrt_packed_moe(*(ctypes.byref(w) for w in (w1, w3, w2)), *a.values())


@pytest.mark.parametrize("changes,words", [
    ({"experts": 0}, "experts"), ({"experts": 8192}, "experts"), ({"tokens": -1}, "tokens"), ({"k": 0}, "tokens"),
    ({"tokens": 1 << 20}, "tokens"), ({"dtype": 5}, "dtype"), ({"activation": 2}, "activation"), ({"x": None}, "null"),
    ({"x": P + 4}, "aligned"), ({"x_ld": 128}, "aligned"), ({"out": P + 4}, "aligned"), ({"ids": None}, "routing"),
    ({"weights": None}, "routing"), ({"pre": P}, "sign"), ({"post": P}, "sign"), ({"pre": P + 4, "post": P}, "sign"),
    ({"pre": P, "post": P}, "512"),
])
def test_experts_refuse(changes, words):
    up, down = matrix(), matrix(rows=128, cols=256)
    refused(moe(up, up, down, **changes), words)
    assert moe(up, up, down, tokens=0) == 0


def test_experts_refuse_matrices_that_do_not_match():
    up, down = matrix(), matrix(rows=128, cols=256)
    refused(moe(up, matrix(rows=128), down), "do not match")
    refused(moe(up, up, matrix()), "do not match")
    refused(moe(up, matrix(rate_axis=1), down), "do not match")
    refused(moe(up, matrix(suh_stride=256), down), "share")
    refused(moe(up, up, matrix(rows=128, cols=256, rates=0)), "rates")


def test_layer_refuses_what_its_router_cannot_read():
    up, down = matrix(), matrix(rows=128, cols=256)
    tail = [ctypes.addressof(LUTS), 4, 0, None, None]
    call = _native.lib().qsrt_packed_moe_layer
    refused(call(*(ctypes.byref(w) for w in (up, up, down)), *tail, P, 256, None, 0, 1, 1.0, P, 256, 0, -1, 2, P, P, P, 256, P,
                 0, None), "sizes")
    refused(call(None, *(ctypes.byref(w) for w in (up, down)), *tail, P, 256, None, 0, 1, 1.0, P, 256, 0, 1, 2, P, P, P, 256,
                 P, 0, None), "sizes")
