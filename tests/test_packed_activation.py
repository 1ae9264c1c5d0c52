"""Which activation a layer was calibrated with stands in no payload: where the framework's own default differs, it is asked for."""

from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest

from qsrt_amd.packed_moe import PackedExperts
from qsrt_amd.qsrt_coupled import CoupledHadamardSpec

EXAMPLE = Path(__file__).resolve().parents[1] / "examples" / "serve_layer.py"


def test_coupled_experts_name_their_activation():
    with pytest.raises(ValueError, match="activation"):
        PackedExperts({}, {}, {}, {}, coupled=CoupledHadamardSpec())
    with pytest.raises(ValueError, match="activation must be one of"):
        PackedExperts({}, {}, {}, {}, activation="gelu", coupled=CoupledHadamardSpec())


def test_experts_of_a_layer_file_name_their_activation():
    with pytest.raises(TypeError, match="activation"):
        PackedExperts.from_experts([], (3,), {})


@pytest.mark.gpu
def test_coupled_experts_refuse_other_blocks():
    from test_packed_serving_gpu import LUTS, Experts

    layer = Experts(61, 384, 128, 2, (3,))
    stacked = [{"trellis": m.words.view(2, -1), "suh": m.suh, "svh": m.svh, "record_bits": (3,)}
               for m in (layer.packed.w1, layer.packed.w3, layer.packed.w2)]
    for spec in (CoupledHadamardSpec(), CoupledHadamardSpec(residual_block_size=128)):
        with pytest.raises(ValueError, match="512"):
            PackedExperts(*stacked, LUTS, activation="situ", coupled=spec)


@pytest.mark.gpu
@pytest.mark.parametrize("more", [[], ["--coupled"]])
def test_example_serves_a_layer_of_the_other_activation(more):
    spec = importlib.util.spec_from_file_location("serve_layer", EXAMPLE)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    result = example.main(["--hidden", "512", "--inter", "256", "--experts", "6", "--k", "2", "--tokens", "3", "--steps", "3",
                           "--activation", "situ", *more])
    # outputs and the projection's scales are rounded to 16 bits (2^-9 in 2-norm each), all else is FP32
    assert all(e <= 2.0**-8 for e in result["errors"].values()), result
