"""Serving from packed weights: the router, a mixture-of-experts layer and a projection with low-rank adapters, timed.

A payload matrix stands for ``W = diag(suh) H_L X H_R diag(svh)``: ``X [K, N]`` are E4M3 labels of the 16-bit cyclic
states of 16 x 16 tiles (a tile is ``16 * bits`` words, its values in tensor-core order), ``H`` the normalised Sylvester
Hadamard on blocks of 128.  Three kinds of case:

* ``route``    router scores and the k experts of each token
* ``layer``    router, the selected experts' gate, up and down products from their payloads, and the weighted sum
* ``adapter``  ``x W + scale_a (x A_a^T) B_a^T`` where every row names its adapter ``a``, or none
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEV = "cuda:0"
DTYPE = {"bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # One generated token's router in a layer of 384 experts: latency alone.
        {"name": "route_token", "kind": "route", "t": 1, "h": 7168, "e": 384, "k": 8, "scoring": "sigmoid", "bias": True,
         "dtype": "bf16"},
        # The router of a decode batch, softmax scores, an odd number of experts.
        {"name": "route_batch", "kind": "route", "t": 96, "h": 5120, "e": 161, "k": 6, "scoring": "softmax", "bias": False,
         "dtype": "f16"},
        # The smallest layer: one token through the tiny expert's shapes.
        {"name": "layer_tiny", "kind": "layer", "t": 1, "h": 256, "i": 512, "e": 8, "k": 2, "bits": "2", "shared": False,
         "act": "swiglu", "dtype": "bf16"},
        # One generated token through the 384-expert layer, K3 records and two K4 records a matrix.
        {"name": "layer_token", "kind": "layer", "t": 1, "h": 7168, "i": 2048, "e": 384, "k": 8, "bits": "34",
         "shared": True, "act": "swiglu", "dtype": "bf16"},
        # A few drafted tokens, an odd count, experts with scales of their own.
        {"name": "layer_draft", "kind": "layer", "t": 5, "h": 5120, "i": 1536, "e": 64, "k": 6, "bits": "3",
         "shared": False, "act": "swiglu", "dtype": "f16"},
        # A decode batch on the 384-expert layer at two bits.
        {"name": "layer_batch", "kind": "layer", "t": 16, "h": 7168, "i": 2048, "e": 384, "k": 8, "bits": "2",
         "shared": True, "act": "situ", "dtype": "bf16"},
        # Few experts and many tokens: every expert sees a ragged group of rows.
        {"name": "layer_crowd", "kind": "layer", "t": 61, "h": 5120, "i": 1536, "e": 8, "k": 2, "bits": "4",
         "shared": True, "act": "swiglu", "dtype": "bf16"},
        # The largest: most of the 384 experts are touched.
        {"name": "layer_wide", "kind": "layer", "t": 48, "h": 7168, "i": 2048, "e": 384, "k": 8, "bits": "34",
         "shared": True, "act": "swiglu", "dtype": "bf16"},
        # One token and its adapter.
        {"name": "adapter_token", "kind": "adapter", "t": 1, "k": 7168, "n": 2048, "bits": "3", "adapters": 16, "r": 16,
         "runs": False, "dtype": "bf16"},
        # A decode batch whose requests bring 32 adapters, some none.
        {"name": "adapter_batch", "kind": "adapter", "t": 48, "k": 7168, "n": 2048, "bits": "3", "adapters": 32, "r": 16,
         "runs": False, "dtype": "bf16"},
        # Short prompts side by side, an odd rank and row count.
        {"name": "adapter_ragged", "kind": "adapter", "t": 333, "k": 2048, "n": 7168, "bits": "24", "adapters": 7, "r": 27,
         "runs": True, "dtype": "f16"},
        # A long prompt: rows of few requests, in runs.
        {"name": "adapter_prompt", "kind": "adapter", "t": 2048, "k": 5120, "n": 1536, "bits": "4", "adapters": 3, "r": 64,
         "runs": True, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["route", "layer", "layer", "layer", "adapter", "adapter"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if kind == "route":
        e = _log(rng, 2, 512)
        return {"kind": kind, "t": _log(rng, 1, 128), "h": 128 * _log(rng, 2, 56), "e": e, "k": rng.randint(1, min(8, e)),
                "scoring": rng.choice(["sigmoid", "softmax"]), "bias": rng.random() < 0.5, "dtype": dtype}
    if kind == "layer":
        h, i, e = 128 * _log(rng, 2, 56), 128 * _log(rng, 1, 16), _log(rng, 2, 384)
        k = rng.randint(1, min(8, e))
        most = 48 * 8 * 7168 * 2048 // (k * h * i)  # no more pairs than the largest listed case has work for
        return {"kind": kind, "t": _log(rng, 1, max(1, min(64, most))), "h": h, "i": i, "e": e, "k": k,
                "bits": rng.choice(["2", "3", "4", "34", "24"]), "shared": rng.random() < 0.6,
                "act": rng.choice(["swiglu", "situ"]), "dtype": dtype}
    k, n = 128 * _log(rng, 1, 56), 128 * _log(rng, 1, 56)
    return {"kind": kind, "t": _log(rng, 1, max(1, min(2048, 2048 * 5120 * 1536 // (k * n)))), "k": k, "n": n,
            "bits": rng.choice(["2", "3", "4", "34", "24"]), "adapters": _log(rng, 1, 64), "r": _log(rng, 1, 128),
            "runs": rng.random() < 0.5, "dtype": dtype}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------


def _table(bits):
    """A 65,536-entry table like a trellis' own: normal quantiles of standard deviation 1.5 in E4M3, in a fixed order."""

    r = torch.randperm(65536, generator=torch.Generator().manual_seed(bits))
    v = (1.5 * torch.special.ndtri((r.double() + 0.5) / 65536)).float().to(torch.float8_e4m3fn).view(torch.uint8)
    v[v == 0x80] = 0
    return v.to(DEV)


def _record_bits(bits, records):
    """One rate a record of 128 channels: the first for all, the second (if any) for one record in eight, at the end."""

    high = max(1, records // 8) if len(bits) > 1 else 0
    return tuple([int(bits[0])] * (records - high) + [int(bits[-1])] * high)


def _matrix(lead, k, n, bits, axis, gen, shared_axis=None):
    """A payload: record-major words (uniform bits, as encoded weights have), FP16 scales with signs on both sides."""

    rates = _record_bits(bits, (k if axis == "k" else n) // 128)
    words = 128 * (n if axis == "k" else k) * sum(rates) // 16

    def scale(rows, size, base):
        s = torch.rand((*rows, size), generator=gen, device=DEV) + 0.5
        sign = torch.randint(0, 2, s.shape, generator=gen, device=DEV) * 2 - 1
        return (base * s * sign).to(torch.float16)

    return {"trellis": torch.randint(-32768, 32768, (*lead, words), generator=gen, device=DEV, dtype=torch.int16),
            "suh": scale(() if shared_axis == "k" else lead, k, 1.0),
            "svh": scale(() if shared_axis == "n" else lead, n, 0.0125),
            "record_bits": rates, "rate_axis": axis}


def prepare(case, seed):
    gen, kind = torch.Generator(device=DEV).manual_seed(int(seed) + 1), case["kind"]
    dtype = DTYPE[case["dtype"]]
    state = {"case": dict(case)}

    def rows(t, h):
        x = torch.randn((t, h), generator=gen, device=DEV)
        return (x * (1 + 2 * torch.rand(h, generator=gen, device=DEV) ** 8)).to(dtype)  # a few strong channels

    if kind == "adapter":
        t, k, n, a, r = (case[q] for q in ("t", "k", "n", "adapters", "r"))
        state["matrix"] = _matrix((), k, n, case["bits"], "k", gen)
        state["luts"] = {int(b): _table(int(b)) for b in case["bits"]}
        state["a"] = (torch.randn((a, r, k), generator=gen, device=DEV) / math.sqrt(k)).to(dtype)
        state["b"] = (torch.randn((a, n, r), generator=gen, device=DEV) / math.sqrt(r)).to(dtype)
        state["scale"] = torch.rand(a, generator=gen, device=DEV) + 0.5
        ids = torch.randint(-1, a, (t,), generator=gen, device=DEV, dtype=torch.int32)
        if case["runs"]:  # whole prompts: a request's rows follow one another
            cut = torch.rand(t, generator=gen, device=DEV) < 6.0 / t
            ids = ids[torch.cummax(torch.where(cut, torch.arange(t, device=DEV), 0), 0).values].contiguous()
        state["x"], state["ids"] = rows(t, k), ids
        if own:
            from qsrt_amd.packed_linear import LowRankAdapters, PackedLinear

            m = state["matrix"]
            state["linear"] = PackedLinear(m["trellis"], m["suh"], m["svh"], m["record_bits"], state["luts"],
                                           rate_axis=m["rate_axis"])
            state["bank"] = LowRankAdapters(state["a"], state["b"], state["scale"])
        return state

    t, h, e = case["t"], case["h"], case["e"]
    state["x"] = rows(t, h)
    state["router"] = (torch.randn((e, h), generator=gen, device=DEV) / math.sqrt(h)).to(dtype)
    state["bias"] = None
    if kind == "route":
        if case["bias"]:
            state["bias"] = 0.05 * torch.randn(e, generator=gen, device=DEV)
        return state
    i, shared = case["i"], case["shared"]
    state["luts"] = {int(b): _table(int(b)) for b in case["bits"]}
    state["w1"] = _matrix((e,), h, i, case["bits"], "n", gen, "k" if shared else None)
    state["w3"] = _matrix((e,), h, i, case["bits"], "n", gen, "k" if shared else None)
    state["w2"] = _matrix((e,), i, h, case["bits"], "k", gen, "n" if shared else None)
    if own:
        from qsrt_amd.packed_moe import PackedExperts, PackedMoELayer

        experts = PackedExperts(state["w1"], state["w3"], state["w2"], state["luts"], activation=case["act"])
        state["layer"] = PackedMoELayer(state["router"], experts, case["k"], scoring="softmax", normalize=True, scale=1.0)
    return state


# ---------------------------------------------------------------------------
# The plain forms, and the framework's
# ---------------------------------------------------------------------------


def _hadamard(dtype):
    i = np.arange(128)
    bits = (i[:, None] & i[None, :]).astype(np.uint8)
    parity = np.unpackbits(bits[..., None], axis=-1).sum(-1) & 1
    return torch.from_numpy((1.0 - 2.0 * parity) / math.sqrt(128.0)).to(DEV, dtype)


def _tile_order():
    """Row and column in its 16 x 16 tile of each of the 256 trellis positions."""

    p = torch.arange(256, device=DEV)
    lane, j = p // 8, p % 8
    return 2 * (lane % 4) + (j % 2) + 8 * (j // 2 % 2), lane // 4 + 8 * (j // 4)


def _labels(words, bits, table):
    """``[..., 16 bits]`` int16 words of tiles -> their labels ``[..., 16, 16]`` in the table's type: position ``p`` is the 16
    bits of the tile's cyclic stream that end after symbol ``p``."""

    chunk = words.contiguous().view(torch.int32).long() & 0xFFFFFFFF
    first = ((torch.arange(256, device=DEV) + 1) * bits - 16) % (256 * bits)
    at, off = first // 32, first % 32
    state = ((chunk[..., at] << 32 | chunk[..., (at + 1) % (8 * bits)]) >> (48 - off)) & 0xFFFF
    row, col = _tile_order()
    place = torch.empty(256, dtype=torch.long, device=DEV)
    place[row * 16 + col] = torch.arange(256, device=DEV)
    return table[state[..., place]].unflatten(-1, (16, 16))


def _dense(words, m, suh, svh, luts, k, n):
    """One payload as a dense float32 ``[K, N]``."""

    rates, axis, cursor, strips = m["record_bits"], m["rate_axis"], 0, []
    for bits in sorted(set(rates)):  # records of one rate follow one another here
        count = rates.count(bits)
        size = count * 8 * ((n if axis == "k" else k) // 16) * 16 * bits
        part, cursor = words[cursor:cursor + size], cursor + size
        tab = luts[bits].view(torch.float8_e4m3fn).float()
        if axis == "k":
            strips.append(_labels(part.view(8 * count, n // 16, 16 * bits), bits, tab).transpose(1, 2).reshape(-1, n))
        else:
            v = _labels(part.view(count, k // 16, 8, 16 * bits), bits, tab)  # record, tile row, tile column, row, column
            strips.append(v.permute(1, 3, 0, 2, 4).reshape(k, -1))
    x = torch.cat(strips, 0 if axis == "k" else 1)
    had = _hadamard(torch.float32)
    x = (had @ x.view(k // 128, 128, n)).view(k, n) * suh.float()[:, None]
    return (x.view(k, n // 128, 128) @ had).view(k, n) * svh.float()


def _of(s, e):
    return s if s.dim() == 1 else s[e]


def _activate(g, u, act):
    if act == "swiglu":
        return g * torch.sigmoid(g) * u
    return 4 * torch.tanh(g / 4) * torch.sigmoid(g) * 25 * torch.tanh(u / 25)


def _choose(logits, k, scoring, bias):
    score = torch.softmax(logits, -1) if scoring == "softmax" else torch.sigmoid(logits)
    key = logits if bias is None else score + bias.to(score.dtype)
    ids = torch.sort(key, dim=-1, descending=True, stable=True).indices[:, :k]
    w = score.gather(1, ids)
    return w / w.sum(-1, keepdim=True), ids


def run(state):
    case = state["case"]
    if own:
        if case["kind"] == "adapter":
            from qsrt_amd.packed_linear import adapter_linear

            return adapter_linear(state["x"], state["linear"], state["bank"], state["ids"])
        if case["kind"] == "route":
            from qsrt_amd.packed_moe import route_tokens

            return route_tokens(state["x"], state["router"], case["k"], bias=state["bias"], scoring=case["scoring"],
                                normalize=True, scale=1.0)
        return state["layer"](state["x"])
    x = state["x"].float()
    if case["kind"] == "adapter":
        m, ids = state["matrix"], state["ids"].long()
        y = x @ _dense(m["trellis"], m, m["suh"], m["svh"], state["luts"], case["k"], case["n"])
        for a in range(case["adapters"]):  # every row through every adapter, the others' rows at nothing
            s = torch.where(ids == a, state["scale"][a], 0.0)
            y = y + s[:, None] * ((x @ state["a"][a].float().T) @ state["b"][a].float().T)
        return y.to(state["x"].dtype)
    w, ids = _choose(x @ state["router"].float().T, case["k"],
                     case.get("scoring", "softmax"), state["bias"])
    if case["kind"] == "route":
        return w, ids.int()
    h, i, y = case["h"], case["i"], torch.zeros_like(x)
    for pair, e in enumerate(ids.reshape(-1)):  # one expert at a time: all of them in float32 would not fit
        t, at = pair // case["k"], e.view(1)
        dense = [_dense(m["trellis"].index_select(0, at)[0], m, _of(m["suh"], e), _of(m["svh"], e), state["luts"], a, b)
                 for m, a, b in ((state["w1"], h, i), (state["w3"], h, i), (state["w2"], i, h))]
        mid = _activate(x[t:t + 1] @ dense[0], x[t:t + 1] @ dense[1], case["act"])
        y[t] += w[t, pair % case["k"]] * (mid @ dense[2])[0]
    return y.to(state["x"].dtype), w, ids.int()


# ---------------------------------------------------------------------------
# In 64 bits, from the definition
# ---------------------------------------------------------------------------


def _rotate64(v):
    had = _hadamard(torch.float64)
    return (v.unflatten(-1, (-1, 128)) @ had).flatten(-2)


def _labels64(words, bits, lut):
    """Symbols first, bit by bit, then the states as the last symbols in a row, shifted together."""

    w = words.reshape(*words.shape[:-1], -1, 2).flip(-1).reshape(words.shape).to(torch.int32)
    stream = (w[..., None] >> torch.arange(15, -1, -1, device=DEV)) & 1
    symbol = (stream.reshape(*words.shape[:-1], 256, bits) << torch.arange(bits - 1, -1, -1, device=DEV)).sum(-1).int()
    state = torch.zeros_like(symbol)
    for back in range(-(-16 // bits)):
        state |= torch.roll(symbol, back, -1) << (bits * back)
    v = lut.view(torch.float8_e4m3fn).double()[(state & 0xFFFF).long()]
    row, col = _tile_order()
    out = torch.empty_like(v)
    out[..., row * 16 + col] = v
    return out.unflatten(-1, (16, 16))


def _product64(x, words, m, suh, svh, luts, n):
    """``x W`` with the activations rotated, and not the weights."""

    k = x.shape[-1]
    x = _rotate64(x * suh.double())
    y, cursor = torch.zeros((x.shape[0], n), dtype=torch.float64, device=DEV), 0
    for r, bits in enumerate(m["record_bits"]):
        size = 8 * ((n if m["rate_axis"] == "k" else k) // 16) * 16 * bits
        part, cursor = words[cursor:cursor + size], cursor + size
        if m["rate_axis"] == "k":
            v = _labels64(part.view(8, n // 16, 16 * bits), bits, luts[bits]).transpose(1, 2).reshape(128, n)
            y += x[:, 128 * r:128 * r + 128] @ v
        else:
            v = _labels64(part.view(k // 16, 8, 16 * bits), bits, luts[bits]).transpose(1, 2).reshape(k, 128)
            y[:, 128 * r:128 * r + 128] = x @ v
    return _rotate64(y) * svh.double()


def exact(case, seed):
    state = prepare(case, seed)
    x = state["x"].double()
    if case["kind"] == "adapter":
        m = state["matrix"]
        y = _product64(x, m["trellis"], m, m["suh"], m["svh"], state["luts"], case["n"])
        for a in range(case["adapters"]):
            rows = (state["ids"] == a).nonzero()[:, 0]
            y[rows] += state["scale"][a].double() * ((x[rows] @ state["a"][a].double().T) @ state["b"][a].double().T)
        return y
    logits = x @ state["router"].double().T
    w, ids = _choose(logits, case["k"], case.get("scoring", "softmax"), state["bias"])
    if case["kind"] == "route":
        return w, None
    y = torch.zeros_like(x)
    for e in sorted(set(ids.reshape(-1).tolist())):
        t, j = (ids == e).nonzero(as_tuple=True)
        g, u = (_product64(x[t], m["trellis"][e], m, _of(m["suh"], e), _of(m["svh"], e), state["luts"], case["i"])
                for m in (state["w1"], state["w3"]))
        m = state["w2"]
        d = _product64(_activate(g, u, case["act"]), m["trellis"][e], m, _of(m["suh"], e), _of(m["svh"], e),
                       state["luts"], case["h"])
        y.index_add_(0, t, w[t, j][:, None] * d)
    return y, w, None


def work(case):
    """Payloads, scales and adapters of what is selected (an even router's expectation), rows in and out, once each."""

    t = case["t"]
    if case["kind"] == "adapter":
        k, n, r, a = case["k"], case["n"], case["r"], case["adapters"]
        used = a * (1 - (1 - 1 / (a + 1)) ** (min(t, 7) if case["runs"] else t))
        payload = k * n * sum(_record_bits(case["bits"], k // 128)) / (k // 128) / 8
        return {"bytes": payload + 2 * (k + n) + used * 2 * r * (k + n) + 2 * t * (k + n) + 4 * t,
                "flops": 2.0 * t * k * n + 2.0 * t * r * (k + n) * a / (a + 1)}
    h, e, k = case["h"], case["e"], case["k"]
    route = {"bytes": 2.0 * (t + e) * h + 8 * t * k, "flops": 2.0 * t * e * h}
    if case["kind"] == "route":
        return route
    i, distinct = case["i"], e * (1 - (1 - k / e) ** t)
    rate = sum(sum(_record_bits(case["bits"], c // 128)) / (c // 128) for c in (i, i, i)) / 8
    scales = 2 * (3 * i * distinct + 3 * h * (1 if case["shared"] else distinct))
    return {"bytes": route["bytes"] + distinct * rate * h * i + scales + 2.0 * t * h,
            "flops": route["flops"] + 6.0 * t * k * h * i}
