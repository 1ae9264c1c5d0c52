"""The gated feed-forward block and the norms as a program uses them: views, streams, graphs, parts of the gradients, rows that
are not finite, and a whole half of a transformer block forward and backward."""

from __future__ import annotations

import threading

import pytest
import torch

from qsrt_amd import _native
from qsrt_amd.block_norm import residual_norm, rms_norm
from qsrt_amd.gated_ffn import gated_ffn, gated_ffn_gradients
from qsrt_amd.gradient_guided_viterbi import expert_guidance
from qsrt_amd.qsrt_coupled import situ, situ_derivatives
from test_block_norm_gpu import draw as draw_norm
from test_gated_ffn_gpu import check, draw, want

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


def embed(t, ld, offset=0):
    """``t`` as a view of a larger buffer whose other values are NaN."""

    rows, cols = t.shape
    buffer = torch.full((rows * ld + offset + 64,), float("nan"), dtype=t.dtype, device=t.device)
    view = buffer[offset:offset + rows * ld].view(rows, ld)[:, :cols]
    view.copy_(t)
    return view


@pytest.mark.parametrize("t", [1, 5, 40, 200])
@pytest.mark.parametrize("ld,offset", [(8, 0), (3, 0), (0, 1), (16, 5)])
def test_views(t, ld, offset):
    """Rows apart by more than their length, odd strides, bases off alignment, transposed weights, an expanded dy."""

    x, gate, up, down, dy = draw(t, t, 264, 136, BF16)
    plain = gated_ffn(x, gate, up, down)
    views = embed(x, 264 + ld, offset), embed(gate, 264 + 2 * ld, offset), embed(up, 264 + ld, offset), embed(down, 136 + ld, offset)
    assert torch.equal(gated_ffn(*views), plain)
    assert torch.equal(gated_ffn(x.T.contiguous().T, gate.T.contiguous().T, up, down.T.contiguous().T), plain)
    grads = gated_ffn_gradients(x, dy, gate, up, down)
    for got, expected in zip(vars(gated_ffn_gradients(views[0], embed(dy, 264 + ld, offset), *views[1:])).values(), vars(grads).values()):
        assert torch.equal(got, expected)
    one = torch.ones((1, 1), dtype=BF16, device="cuda").expand(t, 264)
    leaves = [v.detach().requires_grad_() for v in views]
    for got, expected in zip(torch.autograd.grad(gated_ffn(*leaves), leaves, one),
                             list(vars(gated_ffn_gradients(x, one.contiguous(), gate, up, down)).values())):
        assert torch.equal(got, expected)


@pytest.mark.parametrize("ld,offset", [(8, 0), (3, 0), (0, 1), (16, 5)])
def test_views_of_the_norms(ld, offset):
    v, dsum, dn = draw_norm(5, 37, 264, BF16, torch.float32, True, "row", torch.float32)
    views = {k: embed(t, t.shape[1] + ld, offset) if t.dim() == 2 else embed(t[:, None], 1 + ld, offset)[:, 0] for k, t in v.items()}

    def run(v, dsum, dn):
        leaves = [t.detach().requires_grad_() for t in v.values()]
        h, n = residual_norm(*leaves[:3], post_weight=leaves[3], gate=leaves[4], scale=0.5)
        return [h, n, *torch.autograd.grad((h, n), leaves, (dsum, dn))]

    for got, expected in zip(run(views, embed(dsum, 264 + ld, offset), dn.T.contiguous().T), run(v, dsum, dn)):
        assert torch.equal(got, expected)
    one = torch.ones((1, 1), dtype=BF16, device="cuda").expand(37, 264)
    for got, expected in zip(run(views, one.float(), one), run(v, one.float().contiguous(), one.contiguous())):
        assert torch.equal(got, expected)


def test_lone_row_of_any_stride():
    x, gate, up, down, dy = draw(9, 1, 64, 72, BF16)
    odd = x.as_strided((1, 64), (3, 1))
    assert torch.equal(gated_ffn(odd, gate, up, down), gated_ffn(x, gate, up, down))
    for a, b in zip(vars(gated_ffn_gradients(odd, dy.as_strided((1, 64), (0, 1)), gate, up, down)).values(),
                    vars(gated_ffn_gradients(x, dy, gate, up, down)).values()):
        assert torch.equal(a, b)
    v, _, _ = draw_norm(3, 1, 64, BF16, BF16, True, "channel", BF16)
    for a, b in zip(residual_norm(v["residual"].as_strided((1, 64), (1, 1)), v["y"], v["weight"]),
                    residual_norm(v["residual"], v["y"], v["weight"])):
        assert torch.equal(a, b)


@pytest.mark.parametrize("t", [1, 30, 130])
def test_out_and_what_lies_around_it(t):
    x, gate, up, down, _ = draw(t, t, 72, 200, F16)
    buffer = torch.full((t + 3, 88), 7.0, dtype=F16, device="cuda")
    out = buffer[:t, 8:80]
    assert gated_ffn(x, gate, up, down, out=out) is out
    assert torch.equal(out, gated_ffn(x, gate, up, down))
    assert bool((buffer[t:] == 7).all()) and bool((buffer[:, :8] == 7).all()) and bool((buffer[:, 80:] == 7).all())
    for bad in (torch.empty((t, 72), device="cuda"), buffer[:t, 9:81], torch.empty((t + 1, 72), dtype=F16, device="cuda")):
        with pytest.raises(ValueError, match="out"):
            gated_ffn(x, gate, up, down, out=bad)
    with pytest.raises(ValueError, match="gradients"):
        gated_ffn(x, gate.requires_grad_(), up, down, out=out)


def test_refusals():
    x, gate, up, down, dy = draw(1, 4, 64, 72, BF16)
    for call, words in ((lambda: gated_ffn(x.half(), gate, up, down), "type"), (lambda: gated_ffn(x, gate, up.half(), down), "one type"),
                        (lambda: gated_ffn(x.float(), gate.float(), up.float(), down.float()), "bfloat16"),
                        (lambda: gated_ffn(x.cpu(), gate, up, down), "device"), (lambda: gated_ffn(x[:, :56], gate, up, down), "x must be"),
                        (lambda: gated_ffn(x[0], gate, up, down), "x must be"),
                        (lambda: gated_ffn(x[:, :60], gate[:, :60], up[:, :60], down[:60]), "multiples of 8"),
                        (lambda: gated_ffn_gradients(x, dy[:3], gate, up, down), "dy"),
                        (lambda: gated_ffn_gradients(x, dy.half(), gate, up, down), "dy")):
        with pytest.raises(ValueError, match=words):
            call()
    v, _, _ = draw_norm(1, 4, 64, BF16, BF16, True, "channel", BF16)
    r, y, w, p, g = v.values()
    for call, words in ((lambda: residual_norm(r, y[:3], w), "y must"), (lambda: residual_norm(r.half(), y, w), "rows must be"),
                        (lambda: residual_norm(r.float(), y.float(), w), "rows must be"), (lambda: residual_norm(r, y, w.half()), "weights and gate"),
                        (lambda: residual_norm(r, y, w, post_weight=p.float()), "one type"), (lambda: residual_norm(r, y, w[:8]), "hidden"),
                        (lambda: residual_norm(r, y, w, gate=g[:4]), "gate must"), (lambda: residual_norm(r, y, w, gate=g[:4].view(1, 4)), "gate must"),
                        (lambda: residual_norm(r, y, w, eps=-1.0), "eps"), (lambda: residual_norm(r[:, :60], y[:, :60], w[:60]), "multiple of 8"),
                        (lambda: rms_norm(r.float(), w), "rows must be"), (lambda: residual_norm(r[0], y[0], w), "rows must be")):
        with pytest.raises(ValueError, match=words):
            call()


def test_no_rows():
    x, gate, up, down, _ = draw(1, 0, 64, 72, BF16)
    leaves = [v.requires_grad_() for v in (x, gate, up, down)]
    y = gated_ffn(*leaves)
    assert y.shape == (0, 64)
    grads = torch.autograd.grad(y, leaves, torch.empty_like(y))
    assert grads[0].shape == (0, 64) and all(bool((g == 0).all()) for g in grads[1:])
    g = gated_ffn_gradients(x, x, gate, up, down)
    assert g.middle.shape == (0, 72) and bool((g.down == 0).all())
    w = torch.ones(64, device="cuda", requires_grad=True)
    h, n = residual_norm(x, x, w)
    assert n.shape == (0, 64) and bool((torch.autograd.grad((h, n), w, (x, x))[0] == 0).all())


@pytest.mark.parametrize("t", [3, 90])
def test_only_the_gradients_that_are_needed(t):
    tensors = draw(t, t, 136, 72, BF16)[:4]
    dy = draw(t, t, 136, 72, BF16)[4]
    expected = vars(gated_ffn_gradients(tensors[0], dy, *tensors[1:]))
    for mask in range(1, 16):
        leaves = [v.detach().requires_grad_(bool(mask >> i & 1)) for i, v in enumerate(tensors)]
        y = gated_ffn(*leaves)
        y.backward(dy)
        for i, (leaf, name) in enumerate(zip(leaves, ("x", "gate", "up", "down"))):
            assert (leaf.grad is None) != bool(mask >> i & 1)
            if leaf.grad is not None:
                assert torch.equal(leaf.grad, expected[name])
    g = gated_ffn_gradients(tensors[0], dy, *tensors[1:], inputs=False, weights=False)
    assert g.x is None and g.gate is None and torch.equal(g.gate_rows, expected["gate_rows"])


@pytest.mark.parametrize("used", ["h", "n"])
def test_one_result_of_the_norms_is_enough(used):
    v, dh, dn = draw_norm(5, 37, 136, BF16, torch.float32, True, "row", torch.float32)
    leaf = {k: t.detach().requires_grad_() for k, t in v.items()}
    call = lambda: residual_norm(leaf["residual"], leaf["y"], leaf["weight"], post_weight=leaf["post"], gate=leaf["gate"])
    one, both = call()[used == "n"], call()
    zero = torch.zeros_like
    d = (dh, zero(dn)) if used == "h" else (zero(dh), dn)
    got = torch.autograd.grad(one, list(leaf.values()), d[used == "n"], allow_unused=True)
    for a, b in zip(got, torch.autograd.grad(both, list(leaf.values()), d)):
        assert torch.equal(a, b)


def test_second_derivatives_are_refused():
    x, gate, up, down, _ = draw(1, 4, 64, 72, BF16)
    x.requires_grad_()
    for y in (gated_ffn(x, gate, up, down), residual_norm(x, x, torch.ones(64, device="cuda"))[1]):
        with pytest.raises(RuntimeError, match="second derivatives"):
            torch.autograd.grad(y.float().sum(), x, create_graph=True)


@pytest.mark.parametrize("t", [6, 50, 300])
def test_rows_that_are_not_finite_stay_alone(t):
    x, gate, up, down, dy = draw(t, t, 264, 200, BF16)
    bad = x.clone()
    bad[1], bad[3, 5], bad[4, 7] = float("nan"), float("inf"), float("-inf")
    fine = [i for i in range(t) if i not in (1, 3, 4)]
    y, g = gated_ffn(bad, gate, up, down), gated_ffn_gradients(bad, dy, gate, up, down)
    z, h = gated_ffn(x, gate, up, down), gated_ffn_gradients(x, dy, gate, up, down)
    for a, b in ((y, z), (g.x, h.x), (g.gate_rows, h.gate_rows), (g.up_rows, h.up_rows), (g.middle, h.middle)):
        assert torch.equal(a[fine], b[fine]) and not torch.isfinite(a[1]).any()
        assert not torch.isfinite(a[3]).all() and not torch.isfinite(a[4]).all()
    v, _, _ = draw_norm(t, t, 264, BF16, BF16, True, "channel", BF16)
    r = v["residual"].clone()
    r[1], r[3, 5] = float("nan"), float("inf")
    for a, b in zip(residual_norm(r, v["y"], v["weight"], post_weight=v["post"]),
                    residual_norm(v["residual"], v["y"], v["weight"], post_weight=v["post"])):
        assert torch.equal(a[fine], b[fine]) and not torch.isfinite(a[1]).any()


def test_empty_rows_and_rows_of_zeros():
    """A row of zeros has no direction: its norm is 0 and its gradient that of eps alone; the block gives zeros."""

    x, gate, up, down, dy = draw(2, 5, 64, 72, BF16)
    x[2] = 0
    assert bool((gated_ffn(x, gate, up, down)[2] == 0).all())
    assert bool((gated_ffn_gradients(x, dy, gate, up, down).middle[2] == 0).all())
    r = torch.zeros((3, 64), dtype=BF16, device="cuda").requires_grad_()
    w = torch.full((64,), 2.0, dtype=BF16, device="cuda")
    h, n = residual_norm(r, torch.zeros_like(r), w, post_weight=w, eps=0.25)
    assert bool((h == 0).all()) and bool((n == 0).all())
    (g,) = torch.autograd.grad(n, r, torch.ones_like(n))  # 2 / sqrt(0.25)
    assert bool((g == 4).all())


@pytest.mark.parametrize("t", [1, 7, 20, 300, 1100])
def test_the_same_bits_on_every_run_and_stream(t):
    x, gate, up, down, dy = draw(t, t, 520, 1032, F16)
    y, g = gated_ffn(x, gate, up, down), vars(gated_ffn_gradients(x, dy, gate, up, down))
    v, dh, dn = draw_norm(t, t, 520, F16, torch.float32, True, "channel", torch.float32)
    leaf = [v[k].detach().requires_grad_() for k in ("residual", "y", "weight", "post", "gate")]

    def norms():
        out = residual_norm(leaf[0], leaf[1], leaf[2], post_weight=leaf[3], gate=leaf[4])
        return [*out, *torch.autograd.grad(out, leaf, (dh, dn))]

    first = norms()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        again, gradients, norms_again = gated_ffn(x, gate, up, down), vars(gated_ffn_gradients(x, dy, gate, up, down)), norms()
    stream.synchronize()
    assert torch.equal(again, y) and all(torch.equal(gradients[k], g[k]) for k in g)
    assert all(torch.equal(a, b) for a, b in zip(norms_again, first))


def test_calls_of_several_threads():
    cases = [draw(t, t, 264, 136, BF16) for t in (1, 20, 40, 200)]
    expected = [(gated_ffn(*c[:4]), gated_ffn_gradients(c[0], c[4], *c[1:4])) for c in cases]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(5):
                y, g = gated_ffn(*cases[i][:4]), gated_ffn_gradients(cases[i][0], cases[i][4], *cases[i][1:4])
                torch.cuda.current_stream().synchronize()
                if not torch.equal(y, expected[i][0]) or not torch.equal(g.down, expected[i][1].down):
                    wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(cases))]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    assert not wrong


@pytest.mark.parametrize("t", [1, 24, 150])
def test_captured_forward_and_backward(t):
    """Replays see new inputs, beside eager work of other sizes between them."""

    x, gate, up, down, dy = draw(t, t, 264, 200, BF16)
    v, _, _ = draw_norm(t, t, 264, BF16, BF16, True, "channel", BF16)
    leaves = [u.requires_grad_() for u in (x, gate, up, down, v["residual"], v["weight"], v["post"], v["gate"])]

    def step():
        n = rms_norm(leaves[4], leaves[5])
        h, n = residual_norm(leaves[4], gated_ffn(n, *leaves[1:4]), leaves[5], post_weight=leaves[6], gate=leaves[7], scale=0.5)
        y = gated_ffn(x, *leaves[1:4]) + n
        return [h.detach(), y.detach(), *torch.autograd.grad((h, y), leaves, (dy, dy))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for k in range(4):
        fresh = draw(100 + k, t, 264, 200, BF16)
        with torch.no_grad():
            for old, new in zip((x, gate, up, down, dy), fresh):
                old.copy_(new)
        graph.replay()
        other = draw(k, 33 + k, 136, 72, BF16)
        gated_ffn(*other[:4])
        torch.cuda.synchronize()
        for a, b in zip(captured, step()):
            assert torch.equal(a, b)


def test_captured_backward_into_the_leaves():
    """A training step's own form, on the side stream that its eager steps ran on; those left no graph behind."""

    x, gate, up, down, dy = draw(18, 40, 136, 72, BF16)
    leaves = [v.requires_grad_() for v in (gate, up, down)]
    weight = torch.ones(136, device="cuda", requires_grad=True)

    def step():
        n = rms_norm(x, weight)
        h, n = residual_norm(x, gated_ffn(n, *leaves), weight)
        torch.autograd.backward((h, n), (dy, dy))

    params = [*leaves, weight]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        for p in params:
            p.grad = None
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()
    captured = [p.grad for p in params]
    for k in range(3):
        with torch.no_grad():
            x.copy_(draw(30 + k, 40, 136, 72, BF16)[0])
        graph.replay()
        torch.cuda.synchronize()
        got = [g.clone() for g in captured]
        for p in params:
            p.grad = None
        step()
        for a, p in zip(got, params):
            assert torch.equal(a, p.grad)
            p.grad = None


def test_gradients_against_differences():
    """Directional differences of the block in 64 bits at the kernel's own inputs: the gradients are those of its formula."""

    x, gate, up, down, dy = draw(6, 12, 64, 72, BF16)
    for activation in ("swiglu", "situ"):
        got = vars(gated_ffn_gradients(x, dy, gate, up, down, activation=activation))
        values = {"x": x.double(), "gate": gate.double(), "up": up.double(), "down": down.double()}

        def objective(v):
            g, u = v["x"] @ v["gate"].T, v["x"] @ v["up"].T
            m = g * torch.sigmoid(g) * u if activation == "swiglu" else 100 * torch.tanh(g / 4) * torch.sigmoid(g) * torch.tanh(u / 25)
            return float(((m @ v["down"].T) * dy.double()).sum())

        for name in values:
            way = torch.randn(values[name].shape, generator=torch.Generator().manual_seed(3), dtype=torch.float64).cuda()
            step = 1e-5
            there, back = ({**values, name: values[name] + s * step * way} for s in (1, -1))
            difference = (objective(there) - objective(back)) / (2 * step)
            # two roundings to bf16 and what the row's rounding does: three halves of a step of every term
            bound = 3 * torch.finfo(BF16).eps / 2 * float((got[name].double().abs() * way.abs()).sum()) + 1e-6
            assert abs(float((got[name].double() * way).sum()) - difference) <= bound, (activation, name)


def test_a_plan_of_few_tiles_of_many_parts_is_no_less_exact():
    """Sums cut into parts (narrow results of long sums), and sums of one stage."""

    for t, hidden, inter in ((20, 8192, 64), (200, 8192, 64), (200, 64, 4096), (1500, 64, 64)):
        tensors = draw(t, t, hidden, inter, BF16)
        expected = want(*tensors, "swiglu", 1 if t > 64 else 2)
        check({"y": gated_ffn(*tensors[:4])}, expected, ["y"])
        check(vars(gated_ffn_gradients(tensors[0], tensors[4], *tensors[1:4])), expected,
              ["middle", "gate_rows", "up_rows", "x", "gate", "up", "down"])


def test_half_a_block_forward_and_backward():
    """norm, block, norm with gate and residual, twice, and a loss: every parameter's gradient against 64 bits."""

    t, hidden, inter, layers = 40, 136, 264, 2
    gen = torch.Generator(device="cuda").manual_seed(11)

    def normal(*shape, scale=1.0, dtype=BF16):
        return (scale * torch.randn(shape, generator=gen, device="cuda")).to(dtype).requires_grad_()

    stream = normal(t, hidden, dtype=torch.float32)
    first = normal(hidden, dtype=torch.float32)
    blocks = [[normal(inter, hidden, scale=hidden**-0.5), normal(inter, hidden, scale=hidden**-0.5),
               normal(hidden, inter, scale=inter**-0.5), normal(hidden, dtype=torch.float32), normal(hidden, dtype=torch.float32),
               normal(hidden, dtype=torch.float32)] for _ in range(layers)]
    leaves = [stream, first, *(p for b in blocks for p in b)]
    weight = torch.randn((t, hidden), generator=gen, device="cuda")

    def run(leaves, norm, ffn, join):
        stream, first, rest = leaves[0], leaves[1], leaves[2:]
        n, h = norm(stream, first), stream
        for i in range(layers):
            gate, up, down, post, scale, weight_ = rest[6 * i:6 * i + 6]
            h, n = join(h, ffn(n, gate, up, down), weight_, post, scale)
        return (n.to(leaves[0].dtype) * weight.to(leaves[0].dtype)).sum() + h.square().sum() / 2

    ours = run(leaves, lambda x, w: rms_norm(x, w, dtype=BF16), lambda x, *w: gated_ffn(x, *w, activation="situ"),
               lambda h, y, w, p, g: residual_norm(h, y, w, post_weight=p, gate=g, scale=0.7))
    got = torch.autograd.grad(ours, leaves)
    exact = [p.detach().double().requires_grad_() for p in leaves]

    def norm64(x, w):
        return w * x * (x.square().mean(1, keepdim=True) + 1e-6).rsqrt()

    def ffn64(x, gate, up, down):
        g, u = x @ gate.T, x @ up.T
        return (100 * torch.tanh(g / 4) * torch.sigmoid(g) * torch.tanh(u / 25)) @ down.T

    def join64(h, y, w, p, g):
        h = 0.7 * h + g * norm64(y, p)
        return h, norm64(h, w)

    theirs = run(exact, norm64, ffn64, join64)
    # Of the chain of 2 x 4 rows in bf16 forward and as many backward each is off by half a step of itself; in quadrature, and
    # with the chain's slopes near 1 (norms keep the scale), the whole is off by 4 half steps: 4 * 2^-9 of the norm on average,
    # three times that allowed.
    for a, b in zip(got, torch.autograd.grad(theirs, exact)):
        assert float((a.double() - b).norm() / b.norm()) <= 12 * 2.0**-9
    assert abs(float(ours) - float(theirs)) <= 12 * 2.0**-9 * abs(float(theirs))


@pytest.mark.parametrize("activation", ["situ", "swiglu"])
def test_guidance_holds_the_gradients_of_an_expert(activation):
    x, gate, up, down, dy = draw(8, 20, 128, 256, BF16)
    guidance = expert_guidance(x, dy, gate, up, down, anchor_id="a", objective_id="o", strength=0.5, activation=activation)
    X, G, U, D, Y = (v.double() for v in (x, gate, up, down, dy))
    g, u = X @ G.T, X @ U.T
    if activation == "situ":
        middle, (by_g, by_u) = situ(g, u).double(), (d.double() for d in situ_derivatives(g, u))
    else:
        s = torch.sigmoid(g)
        middle, by_g, by_u = g * s * u, u * s * (1 + g * (1 - s)), g * s
    rows = Y @ D
    for name, left, right, weight in (("w1", X, rows * by_g, gate), ("w3", X, rows * by_u, up), ("w2", middle, Y, down)):
        one = guidance[name]
        one.validate(weight.T.shape)
        assert torch.equal(one.anchor, weight.T.float())
        # one factor is rounded to bf16 once, half a step of each of its values; FP32 elsewhere
        bound = (2.0**-8 + 2.0**-14) * (left.abs().T @ right.abs()) + 1e-12
        assert bool(((one.left.double() @ one.right.double()) - left.T @ right).abs().le(bound).all()), name
        candidate = weight.T.float() + 0.01
        assert abs(one.linear_term(candidate, dtype=torch.float64) - 0.5 * 0.01 * float((left.T @ right).sum())) <= \
            0.5 * 0.011 * float(bound.sum()) + 1e-6


def test_gradients_given_in_another_type():
    """The engine casts them to the result's type before they come here."""

    x, gate, up, down, dy = draw(12, 20, 72, 136, BF16)
    leaves = [v.requires_grad_() for v in (x, gate, up, down)]
    for got, expected in zip(torch.autograd.grad(gated_ffn(*leaves), leaves, dy.float()),
                             torch.autograd.grad(gated_ffn(*leaves), leaves, dy)):
        assert torch.equal(got, expected)
    v, dsum, dn = draw_norm(1, 6, 72, BF16, torch.float32, True, "row", BF16)
    leaves = [u.requires_grad_() for u in v.values()]

    def run(dsum, dn):
        h, n = residual_norm(*leaves[:3], post_weight=leaves[3], gate=leaves[4])
        return torch.autograd.grad((h, n), leaves, (dsum, dn))

    for got, expected in zip(run(dsum.to(BF16).double(), dn.float()), run(dsum.to(BF16).float(), dn)):
        assert torch.equal(got, expected)


def test_result_in_place_of_the_input():
    for t in (2, 30, 100):
        x, gate, up, down, _ = draw(t, t, 136, 72, BF16)
        expected = gated_ffn(x, gate, up, down)
        assert torch.equal(gated_ffn(x, gate, up, down, out=x), expected)


def test_one_matrix_as_both():
    x, gate, _, down, dy = draw(13, 33, 72, 136, F16)
    leaf = gate.requires_grad_()
    both = gated_ffn_gradients(x, dy, gate, gate, down)
    got = torch.autograd.grad(gated_ffn(x, leaf, leaf, down), leaf, dy)[0]
    assert torch.equal(got, both.gate + both.up)


@pytest.mark.parametrize("t,hidden,inter", [(3, 1 << 17, 8), (20, 8, 1 << 17), (70, 1 << 17, 16), (130, 24, 1 << 17)])
def test_the_most_channels(t, hidden, inter):
    x, gate, up, down, dy = draw(t, t, hidden, inter, BF16)
    expected = want(x, gate, up, down, dy, "swiglu", 2 if t <= 64 else 1)
    check({"y": gated_ffn(x, gate, up, down)}, expected, ["y"])
    check(vars(gated_ffn_gradients(x, dy, gate, up, down)), expected, ["middle", "gate_rows", "up_rows", "x", "gate", "up", "down"])


def test_rows_far_apart():
    """2^22 elements: offsets inside a tile nearly reach 2^31 bytes.  More is refused."""

    far, t, hidden, inter = 1 << 22, 260, 72, 264
    x, gate, up, down, dy = draw(14, t, hidden, inter, BF16)
    plain = gated_ffn_gradients(x, dy, gate, up, down)
    y = gated_ffn(x, gate, up, down)
    room = torch.full(((t + 4) * far,), float("nan"), dtype=BF16, device="cuda")

    def spread(v):
        view = room[:v.shape[0] * far].view(-1, far)[:, :v.shape[1]]
        return view.copy_(v)

    assert torch.equal(gated_ffn(spread(x), gate, up, down), y)
    for got, expected in zip(vars(gated_ffn_gradients(spread(x), dy, gate, up, down)).values(), vars(plain).values()):
        assert torch.equal(got, expected)
    for got, expected in zip(vars(gated_ffn_gradients(x, dy, gate, up, spread(down))).values(), vars(plain).values()):
        assert torch.equal(got, expected)
    wide = torch.empty((2 * (far + 8),), dtype=BF16, device="cuda").view(2, far + 8)[:, :hidden]
    with pytest.raises(ValueError, match="2\\^22"):
        gated_ffn(wide, gate, up, down)


def test_offsets_over_32_bits():
    """Rows whose elements number more than 2^31: the last ones are what they are in a small call."""

    t, hidden, inter, last = 1 << 20, 16, 2056, 128
    x, gate, up, down, _ = draw(15, t, hidden, inter, BF16)
    dy = torch.zeros_like(x)
    dy[-last:] = draw(16, last, hidden, inter, BF16)[4]
    few = gated_ffn_gradients(x[-last:], dy[-last:], gate, up, down)
    got = gated_ffn_gradients(x, dy, gate, up, down)
    assert got.middle.numel() > 1 << 31
    # sums of 16 and 2056 products, in other parts: (K + 1) 2^-24 each of values of order one, and half a step of bf16 on top
    for name in ("middle", "gate_rows", "up_rows", "x"):
        a, b = getattr(got, name)[-last:].double(), getattr(few, name).double()
        assert bool(((a - b).abs() <= 2.0**-7 * b.abs() + 2.0**-10 * b.abs().max()).all()), name
    for name in ("gate", "up", "down"):
        a, b = getattr(got, name).double(), getattr(few, name).double()
        assert bool(((a - b).abs() <= 2.0**-7 * b.abs() + 2.0**-10 * b.abs().max()).all()), name
    y = gated_ffn(x, gate, up, down)[-last:].double()
    b = gated_ffn(x[-last:], gate, up, down).double()
    assert bool(((y - b).abs() <= 2.0**-7 * b.abs() + 2.0**-10 * b.abs().max()).all())


def test_norm_offsets_over_32_bits():
    t, hidden, last = (1 << 21) + 5, 1032, 64
    residual = torch.zeros((t, hidden), dtype=BF16, device="cuda")
    y, dn = torch.zeros_like(residual), torch.zeros_like(residual)
    v, dsum, dlast = draw_norm(17, last, hidden, BF16, BF16, True, "channel", BF16)
    residual[-last:], y[-last:], dn[-last:] = v["residual"], v["y"], dlast
    assert residual.numel() > 1 << 31

    def run(r, y, dn):
        r, y = r.detach().requires_grad_(), y.detach().requires_grad_()
        h, n = residual_norm(r, y, v["weight"], post_weight=v["post"], gate=v["gate"])
        return [u[-last:] for u in (h.detach(), n.detach(), *torch.autograd.grad(n, (r, y), dn))]

    for got, expected in zip(run(residual, y, dn), run(v["residual"], v["y"], dlast)):
        assert torch.equal(got, expected)  # rows are alone
