"""Serve tokens through a packed layer: a projection with low-rank adapters, then a router and its experts.

    python examples/serve_layer.py [--file qsrt-layer-00024.safetensors] [--tokens 4] [--steps 64]

The experts come from a rate-record layer file and stay packed on the GPU.  Without ``--file`` a small synthetic layer is
written first: random words are valid payloads.  The projection is encoded here, at K3.  The step is checked against products
with the decoded matrices, captured in a HIP graph, and replayed.
"""

from __future__ import annotations

import argparse
import sys
import tempfile
import time
from pathlib import Path

if __package__ in (None, ""):
    sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import torch

from qsrt_amd import exl3_encoder_backend as backend
from qsrt_amd.decode import DecodePlan, decode_words
from qsrt_amd.ldlq import make_shared_h
from qsrt_amd.packed_linear import LowRankAdapters, PackedLinear, adapter_linear
from qsrt_amd.packed_moe import PackedExperts, PackedMoELayer
from qsrt_amd.qsrt import Geometry
from qsrt_amd.qsrt_coupled import CoupledHadamardSpec, decode_coupled_weights, situ
from qsrt_amd.qsrt_rate_atoms import QSRTRateLayerLayout, QSRTRateLayerReader, RateSchedule, materialize_rate_layer
from qsrt_amd.sqg_e4m3 import sqg_xor_cheb_t12_bytes

MATRICES = ("w1", "w3", "w2")


def write_synthetic_layer(path: Path, *, hidden: int, inter: int, experts: int, generator) -> None:
    """A layer file of random payloads, K3 with one pair of K4 records."""

    records = inter // 128
    schedule = RateSchedule(Geometry(inter, hidden), (3,) * (records - 2) + (4, 4))

    def scale(n, size):
        sign = torch.randint(0, 2, (n,), generator=generator) * 2 - 1
        return (size * sign * (torch.rand(n, generator=generator) + 0.5)).half()

    shared = {"w1": scale(hidden, 1.0), "w3": scale(hidden, 1.0), "w2": scale(hidden, 0.5 * inter**-0.5)}

    def payloads():
        for e in range(experts):
            tensors = {}
            for m in MATRICES:
                words = torch.randint(-32768, 32768, (schedule.matrix_words,), generator=generator, dtype=torch.int32)
                local = scale(inter, 0.5 * hidden**-0.5 if m != "w2" else 1.0)
                suh, svh = (local, shared[m]) if m == "w2" else (shared[m], local)
                tensors[m] = {"trellis": words.to(torch.int16), "suh": suh, "svh": svh}
            yield e, tensors

    materialize_rate_layer(path, QSRTRateLayerLayout(24, schedule, tuple(range(experts))), payloads())


def load_layer(path: Path, coupled, activation: str, device) -> tuple:
    """The file's experts: ``(PackedExperts, their payloads for the check, the schedule)``."""

    luts = {b: sqg_xor_cheb_t12_bytes(b) for b in (2, 3, 4)}
    with QSRTRateLayerReader(path) as reader:
        schedule = reader.layout.schedule
        payloads = [reader.read_expert(e) for e in reader.layout.experts]
    packed = PackedExperts.from_experts(payloads, schedule.record_bits, luts, activation=activation, coupled=coupled,
                                        device=device)
    return packed, payloads, schedule


def decoded(payloads: list, schedule: RateSchedule, coupled, device) -> list:
    """The experts' matrices in FP32, ``[K, N]``."""

    inter, hidden = schedule.geometry.intermediate_channels, schedule.geometry.latent_channels
    jobs, outs = [], []
    for p in payloads:
        out = {m: torch.empty((inter, hidden) if m == "w2" else (hidden, inter), device=device) for m in MATRICES}
        for m in MATRICES:
            jobs.append((p[m]["trellis"].to(device), schedule.record_bits, "k" if m == "w2" else "n",
                         (p[m]["suh"].float() / 128).to(device), p[m]["svh"].float().to(device), out[m]))
        outs.append(out)
    DecodePlan.for_records(jobs, {b: sqg_xor_cheb_t12_bytes(b).to(device) for b in set(schedule.record_bits)},
                           out_dtype=torch.float32).run()
    if coupled is not None:
        for out in outs:
            w1, w3, w2 = decode_coupled_weights(tuple(out[m].T.contiguous() for m in MATRICES), coupled)
            out.update(w1=w1.T, w3=w3.T, w2=w2.T)
    return outs


def encode_projection(hidden: int, device, generator) -> tuple:
    """A K3 projection ``[hidden, hidden]`` encoded with a random layer's Hessian, and its decoded weight."""

    x = torch.randn((2 * hidden, hidden), generator=generator).to(device)
    shared = make_shared_h(hidden, device, x.T @ x)
    shared["count"] = x.shape[0]
    lut = sqg_xor_cheb_t12_bytes(3)
    weight = (torch.randn((hidden, hidden), generator=generator) * hidden**-0.5).to(device)
    _, _, tensors = backend.quantize_qsrt(weight, shared, {
        "K": 3, "seed": 11, "sv_seed": 12, "sigma_reg": 0.01, "devices": [str(device)], "apply_out_scales": False,
        "tailbite_context": 128, "sqg_e4m3_lut": lut}, False)
    linear = PackedLinear(tensors["trellis"], tensors["suh"], tensors["svh"], 3, {3: lut})
    return linear, decode_words(tensors["trellis"], tensors["suh"], tensors["svh"], 3, lut, out_dtype=torch.float32)


def main(argv=None) -> dict:
    args = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    args.add_argument("--file", type=Path, help="a rate-record layer file (default: a synthetic one)")
    args.add_argument("--coupled", action="store_true", help="its weights are in coupled coordinates (default profile)")
    args.add_argument("--activation", choices=("swiglu", "situ"), default="swiglu", help="what the layer was calibrated with")
    args.add_argument("--hidden", type=int, default=1024)
    args.add_argument("--inter", type=int, default=512)
    args.add_argument("--experts", type=int, default=16)
    args.add_argument("--k", type=int, default=4, help="experts of a token")
    args.add_argument("--tokens", type=int, default=4)
    args.add_argument("--steps", type=int, default=64)
    args = args.parse_args(argv)
    coupled = CoupledHadamardSpec() if args.coupled else None
    device, gen = torch.device("cuda:0"), torch.Generator().manual_seed(0)

    with tempfile.TemporaryDirectory() as directory:
        path = args.file
        if path is None:
            path = Path(directory) / "qsrt-layer-00024.safetensors"
            write_synthetic_layer(path, hidden=args.hidden, inter=args.inter, experts=args.experts, generator=gen)
        packed, payloads, schedule = load_layer(path, coupled, args.activation, device)
    hidden, experts = packed.hidden, packed.experts
    linear, dense = encode_projection(hidden, device, gen)

    def rand(*shape):
        return torch.randn(shape, generator=gen).to(device, torch.bfloat16)

    adapters = LowRankAdapters(rand(3, 16, hidden) * hidden**-0.5, rand(3, hidden, 16) * 0.25)
    ids = (torch.arange(args.tokens, dtype=torch.int32) % 4 - 1).to(device)  # every fourth token has no adapter
    layer = PackedMoELayer(rand(experts, hidden) * hidden**-0.5, packed, min(args.k, experts), scoring="sigmoid")
    x = rand(args.tokens, hidden)

    def step():
        h = adapter_linear(x, linear, adapters, ids)
        y, weights, chosen = layer(h)
        return h, y, weights, chosen

    h, y, weights, chosen = step()
    want = x.float() @ dense
    for i, a in enumerate(ids.tolist()):
        if a >= 0:
            want[i] += (x[i].float() @ adapters.a[a].float().T) @ adapters.b[a].float().T
    errors = {"projection": float((h.float() - want).norm() / want.norm())}
    matrices, want = decoded(payloads, schedule, coupled, device), torch.zeros((args.tokens, hidden), device=device)
    for i in range(args.tokens):
        for w, e in zip(weights[i].tolist(), chosen[i].tolist()):
            g, u = h[i].float() @ matrices[e]["w1"], h[i].float() @ matrices[e]["w3"]
            middle = situ(g, u) if args.activation == "situ" else torch.nn.functional.silu(g) * u
            want[i] += w * (middle @ matrices[e]["w2"])
    errors["layer"] = float((y.float() - want).norm() / want.norm())
    del matrices

    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        h, y, weights, chosen = step()
    graph.replay()
    torch.cuda.synchronize()
    start = time.perf_counter()
    for _ in range(args.steps):
        graph.replay()
    torch.cuda.synchronize()
    result = {"experts": experts, "hidden": hidden, "inter": packed.inter, "tokens": args.tokens, "errors": errors,
              "us_per_step": (time.perf_counter() - start) / args.steps * 1e6}
    print(result, flush=True)
    return result


if __name__ == "__main__":
    main()
