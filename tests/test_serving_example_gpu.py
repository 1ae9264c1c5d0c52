"""The serving example runs from a layer file to replayed steps, and its step equals products with decoded matrices."""

from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu
PATH = Path(__file__).resolve().parents[1] / "examples" / "serve_layer.py"


@pytest.mark.parametrize("tokens,more", [(1, []), (7, ["--coupled"])])
def test_example_serves_a_layer(tokens, more):
    spec = importlib.util.spec_from_file_location("serve_layer", PATH)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    result = example.main(["--hidden", "512", "--inter", "256", "--experts", "6", "--k", "2", "--tokens", str(tokens),
                           "--steps", "3", *more])
    assert (result["experts"], result["hidden"], result["inter"]) == (6, 512, 256)
    # outputs and the projection's scales are rounded to 16 bits (2^-9 in 2-norm each), all else is FP32
    assert all(e <= 2.0**-8 for e in result["errors"].values()), result
