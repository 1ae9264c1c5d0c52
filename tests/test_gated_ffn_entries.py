"""The entries of the gated feed-forward block and of the norms refuse bad arguments on the host: no GPU is needed here."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from qsrt_amd import _native
from qsrt_amd.block_norm import residual_norm, rms_norm
from qsrt_amd.gated_ffn import gated_ffn, gated_ffn_gradients
from qsrt_amd.gradient_guided_viterbi import expert_guidance

native = pytest.mark.skipif(not _native.LIB_PATH.exists(), reason="the native library is not built")

BUF = np.zeros(4096 + 64, dtype=np.uint8)
P = (BUF.ctypes.data + 63) // 64 * 64  # an aligned address; nothing reads it


def refused(rc, words):
    message = _native.lib().qsrt_last_error().decode()
    assert rc == -1 and words in message, (rc, message)


def ffn(**changes):
    a = {"x": P, "x_ld": 64, "gate": P, "up": P, "up_ld": 64, "down": P, "down_ld": 128, "dtype": 0, "tokens": 3, "hidden": 64,
         "inter": 128, "activation": 0, "pre": None, "out": P, "out_ld": 64, "ws": P, "ws_bytes": 0, "stream": None}
    a.update(changes)
    return _native.lib().qsrt_gated_ffn(*a.values())


def ffn_backward(**changes):
    a = {"dy": P, "dy_ld": 64, "x": P, "x_ld": 64, "gate": P, "up": P, "up_ld": 64, "down": P, "down_ld": 128, "dtype": 0,
         "tokens": 3, "hidden": 64, "inter": 128, "activation": 0, "pre": P, "dx": P, "dx_ld": 64, "d_gate": P, "d_up": P,
         "d_down": P, "gate_rows": None, "up_rows": None, "middle": None, "ws": P, "ws_bytes": 0, "stream": None}
    a.update(changes)
    return _native.lib().qsrt_gated_ffn_backward(*a.values())


BLOCK = [({"tokens": -1}, "tokens"), ({"tokens": (1 << 20) + 1}, "tokens"), ({"hidden": 0}, "channels"), ({"hidden": 60}, "channels"),
         ({"inter": 4}, "channels"), ({"inter": (1 << 17) + 8}, "channels"), ({"hidden": (1 << 17) + 8}, "channels"),
         ({"dtype": 2}, "dtype"), ({"activation": 2}, "activation"), ({"x": None}, "null"), ({"gate": None}, "null"),
         ({"up": None}, "null"), ({"down": None}, "null"), ({"x": P + 8}, "aligned"), ({"gate": P + 2}, "aligned"),
         ({"down": P + 4}, "aligned"), ({"x_ld": 60}, "aligned"), ({"x_ld": 56}, "aligned"), ({"up_ld": 32}, "aligned"),
         ({"down_ld": 64}, "aligned"), ({"up_ld": 1 << 23}, "2^22")]


@native
@pytest.mark.parametrize("changes,words", BLOCK + [({"out": None}, "null"), ({"out": P + 8}, "aligned"), ({"out_ld": 56}, "aligned"),
                                                   ({"pre": P + 4}, "aligned")])
def test_block_refuses(changes, words):
    refused(ffn(**changes), words)


@native
@pytest.mark.parametrize("changes,words", BLOCK + [({"dy": None}, "null"), ({"dy": P + 8}, "aligned"), ({"dy_ld": 8}, "aligned"),
                                                   ({"pre": None}, "null"), ({"pre": P + 8}, "aligned"), ({"dx": P + 8}, "aligned"),
                                                   ({"d_gate": P + 2}, "aligned"), ({"middle": P + 2}, "aligned")])
def test_block_gradients_refuse(changes, words):
    refused(ffn_backward(**changes), words)


@native
def test_no_rows_are_nothing_to_do():
    assert ffn(tokens=0, x=None) == 0 and ffn_backward(tokens=0, dy=None) == 0
    assert norm(rows=0, y=None, post=None, gate=None, gate_kind=0) == 0 and norm_backward(rows=0) == 0


@native
def test_calls_name_the_workspace_they_need():
    lib = _native.lib()
    for need, call in ((lib.qsrt_gated_ffn_workspace_bytes(3, 64, 128), ffn),
                       (lib.qsrt_gated_ffn_backward_workspace_bytes(3, 64, 128), ffn_backward),
                       (lib.qsrt_residual_norm_backward_workspace_bytes(3, 64), norm_backward)):
        assert need > 0
        for changes in ({"ws_bytes": need - 1}, {"ws": None, "ws_bytes": need}):
            assert call(**changes) == -2 and str(need) in lib.qsrt_last_error().decode()


@native
def test_workspaces_of_refused_sizes_are_empty():
    lib = _native.lib()
    for sizes in ((0, 64, 64), (-1, 64, 64), (3, 63, 64), (3, 64, 0), (1 << 21, 64, 64), (3, 1 << 18, 64)):
        assert lib.qsrt_gated_ffn_workspace_bytes(*sizes) == 0 and lib.qsrt_gated_ffn_backward_workspace_bytes(*sizes) == 0
    for sizes in ((0, 64), (-1, 64), (3, 60), (3, (1 << 14) + 8), ((1 << 22) + 1, 64)):
        assert lib.qsrt_residual_norm_backward_workspace_bytes(*sizes) == 0


def norm(**changes):
    a = {"residual": P, "residual_ld": 64, "residual_f32": 0, "y": P, "y_ld": 64, "dtype": 0, "rows": 3, "hidden": 64, "weight": P,
         "post": P, "gate": P, "gate_kind": 1, "params_f32": 0, "scale": 1.0, "eps": 1e-6, "sum": P, "sum_ld": 64, "normed": P,
         "normed_ld": 64, "stats": None, "stream": None}
    a.update(changes)
    return _native.lib().qsrt_residual_norm(*a.values())


def norm_backward(**changes):
    a = {"dsum": P, "dsum_ld": 64, "dn": P, "dn_ld": 64, "residual": P, "residual_ld": 64, "residual_f32": 0, "y": P, "y_ld": 64,
         "dtype": 0, "rows": 3, "hidden": 64, "weight": P, "post": P, "gate": P, "gate_kind": 1, "params_f32": 0, "scale": 1.0,
         "stats": P, "dresidual": P, "dresidual_ld": 64, "dy": P, "dy_ld": 64, "dweight": P, "dpost": P, "dgate": P, "ws": P,
         "ws_bytes": 0, "stream": None}
    a.update(changes)
    return _native.lib().qsrt_residual_norm_backward(*a.values())


NORM = [({"rows": -1}, "rows"), ({"rows": (1 << 22) + 1}, "rows"), ({"hidden": 0}, "channels"), ({"hidden": 60}, "channels"),
        ({"hidden": (1 << 14) + 8}, "channels"), ({"dtype": 2}, "dtype"), ({"gate_kind": 3}, "gate"), ({"gate": None}, "gate"),
        ({"gate_kind": 0}, "gate"), ({"y": None}, "without y"), ({"weight": None}, "null"), ({"residual": None}, "null"),
        ({"residual": P + 8}, "aligned"), ({"residual_ld": 56}, "aligned"), ({"y": P + 2}, "aligned"), ({"y_ld": 60}, "aligned"),
        ({"weight": P + 4}, "aligned"), ({"post": P + 4}, "aligned"), ({"gate": P + 4}, "aligned")]


@native
@pytest.mark.parametrize("changes,words", NORM + [({"eps": -1.0}, "eps"), ({"eps": float("nan")}, "eps"), ({"normed": None}, "null"),
                                                  ({"normed_ld": 8}, "aligned"), ({"sum": P + 8}, "aligned")])
def test_norms_refuse(changes, words):
    refused(norm(**changes), words)


@native
@pytest.mark.parametrize("changes,words", NORM + [({"stats": None}, "null"), ({"dsum": P + 8}, "aligned"), ({"dn_ld": 60}, "aligned"),
                                                  ({"dy": P + 8}, "aligned"), ({"dresidual_ld": 8}, "aligned"),
                                                  ({"post": None}, "not there"),
                                                  ({"gate": None, "gate_kind": 0}, "not there"),
                                                  ({"y": None, "post": None, "gate": None, "gate_kind": 0}, "without y")])
def test_norm_gradients_refuse(changes, words):
    refused(norm_backward(**changes), words)


def test_python_calls_refuse_tensors_in_host_memory():
    x, w, d = torch.zeros((2, 16), dtype=torch.bfloat16), torch.zeros((8, 16), dtype=torch.bfloat16), torch.zeros((16, 8), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        gated_ffn(x, w, w, d)
    with pytest.raises(ValueError, match="CUDA"):
        gated_ffn_gradients(x, x, w, w, d)
    with pytest.raises(ValueError, match="CUDA"):
        expert_guidance(x, x, w, w, d, anchor_id="a", objective_id="o")
    with pytest.raises(ValueError, match="identities"):
        expert_guidance(x, x, w, w, d, anchor_id="", objective_id="o")
    with pytest.raises(ValueError, match="nonnegative"):
        expert_guidance(x, x, w, w, d, anchor_id="a", objective_id="o", strength=-1.0)
    with pytest.raises(ValueError, match="CUDA"):
        residual_norm(x, x, torch.ones(16))
    with pytest.raises(ValueError, match="CUDA"):
        rms_norm(x, torch.ones(16))


def test_python_calls_refuse_shapes_before_anything_else():
    x, w, d = torch.zeros((2, 16), dtype=torch.bfloat16), torch.zeros((8, 16), dtype=torch.bfloat16), torch.zeros((16, 8), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="activation"):
        gated_ffn(x, w, w, d, activation="relu")
    for bad in ((w, w[:4], d), (w, w, d.T), (w[0], w[0], d)):
        with pytest.raises(ValueError, match="inter, hidden"):
            gated_ffn(x, *bad)


@native
@pytest.mark.parametrize("t,hidden,inter", [(0, 64, 64), (-1, 64, 64), (1, 60, 64), (1, 64, 1 << 18)])
def test_plan_refuses(t, hidden, inter):
    refused(_native.lib().qsrt_gated_ffn_plan(t, hidden, inter, (ctypes.c_int64 * 11)()), "sizes")
    refused(_native.lib().qsrt_gated_ffn_plan(1, 64, 64, None), "plan")
