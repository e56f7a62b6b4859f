"""GPU: the FP8 operators and the token sort as an expert layer runs them, one after the
other, in a captured graph (its backward pass too), on several streams and from several
threads, and their native calls against the general path."""

from __future__ import annotations

import threading

import pytest
import torch

import mxfp4_amd as mx
from mxfp4_amd import _lib

from _helpers import cuda, rand_act

pytestmark = pytest.mark.gpu
H, INTER, EXPERTS, TOP = 512, 256, 32, 4
BF16, F8 = torch.bfloat16, torch.float8_e4m3fn


class Layer:
    def __init__(self):
        self.gate = cuda(rand_act(1, (EXPERTS, H)) * 0.05)
        self.w13, self.s13 = mx.dynamic_fp8_block_quant(
            cuda(rand_act(2, (EXPERTS, 2 * INTER, H)).float() * 0.05), block_rows=128)
        self.w2, self.s2 = mx.dynamic_fp8_block_quant(
            cuda(rand_act(3, (EXPERTS, H, INTER)).float() * 0.05), block_rows=128)
        self.wo, self.so = mx.dynamic_fp8_block_quant(cuda(rand_act(4, (H, H)).float() * 0.05),
                                                      block_rows=128)

    def run(self, x):
        q, s = mx.dynamic_fp8_block_quant(x)
        o = mx.linear_fp8_block(q, s, self.wo, self.so)
        w, ids = mx.route_topk_grouped(o.float() @ self.gate.float().T, TOP, scoring="sigmoid")
        order = mx.sort_routes(ids, EXPERTS)
        a, sa = mx.dynamic_fp8_block_quant(o)
        gu = mx.grouped_linear_fp8_block(a, sa, self.w13, self.s13, order, gather=True)
        h, sh = mx.silu_mul_fp8_block_quant(gu)
        y = mx.grouped_linear_fp8_block(h, sh, self.w2, self.s2, order)
        return {"q": q, "s": s, "o": o, "w": w, "ids": ids, "offsets": order.offsets,
                "routes": order.routes, "position": order.position, "a": a, "sa": sa, "gu": gu,
                "h": h, "sh": sh, "y": y, "out": mx.combine_tokens(y, order, w)}


@pytest.fixture(scope="module")
def layer():
    return Layer()


def _same(a, b):
    for name in a:
        x, y = a[name], b[name]
        if x.dtype.itemsize == 1:
            x, y = x.view(torch.uint8), y.view(torch.uint8)
        assert torch.equal(x, y), name


def _rows(q, s):
    return q.double() * s.double().repeat_interleave(128, -1)[..., :q.shape[-1]]


def _weights(q, s):
    n, k = q.shape[-2:]
    s = s.double().repeat_interleave(128, -1)[..., :k].repeat_interleave(128, -2)[..., :n, :]
    return q.double() * s


@pytest.mark.parametrize("m", [1, 37, 300])
def test_layer_against_fp64_step_by_step(layer, m):
    # each step on the values the step before it gave
    r = layer.run(cuda(rand_act(10 + m, (m, H))))

    def close(got, a, w):
        want = a @ w.T
        # half a step of bf16; what the MFMA cuts off: 7 of 8 products 2^-13 of the
        # group's largest, no more than that of the product of the vectors' largest groups
        cut = 7 * 2.0 ** -13 * (a.abs().view(len(a), -1, 8).amax(-1)
                                @ w.abs().view(len(w), -1, 8).amax(-1).T)
        adds = 64 * 2.0 ** -24 * (a.abs() @ w.abs().T)
        assert ((got.double() - want).abs() <= 2.0 ** -8 * want.abs() + 1.01 * (cut + adds)).all()

    close(r["o"], _rows(r["q"], r["s"]), _weights(layer.wo, layer.so))
    off, routes = r["offsets"].tolist(), r["routes"].long()
    assert off[-1] == m * TOP
    a, h = _rows(r["a"], r["sa"]), _rows(r["h"], r["sh"])
    w13, w2 = _weights(layer.w13, layer.s13), _weights(layer.w2, layer.s2)
    for e in range(EXPERTS):
        at = slice(off[e], off[e + 1])
        if off[e + 1] > off[e]:
            assert (r["ids"].reshape(-1)[routes[at]] == e).all()
            close(r["gu"][at], a[routes[at] // TOP], w13[e])
            close(r["y"][at], h[at], w2[e])
    gate, up = r["gu"].double().split(INTER, 1)
    want = gate * torch.sigmoid(gate) * up
    unit = r["sh"].double().repeat_interleave(128, 1)
    half = torch.maximum(want.abs() * 2.0 ** -4, unit * 2.0 ** -10)
    assert ((h - want).abs() <= half * (1 + 2.0 ** -18) + want.abs() * 2.0 ** -18).all()
    terms = r["y"].double()[r["position"].long()] * r["w"].double()[..., None]
    want = terms.sum(1)
    tol = 2.0 ** -8 * want.abs() + 2 * TOP * 2.0 ** -24 * 1.01 * terms.abs().sum(1)
    assert ((r["out"].double() - want).abs() <= tol).all()


@pytest.mark.parametrize("m", [1, 64, 300])
def test_graph_replays_equal_eager(layer, m):
    buf = cuda(rand_act(7, (m, H)))
    layer.run(buf)
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            captured = layer.run(buf)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for rep in range(4):
        new = cuda(rand_act(1000 * rep + 3, (m, H)))
        buf.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        _same(captured, layer.run(new))


def test_two_graphs_in_turn(layer):
    # nothing of one call is left for another: graphs of different sizes replayed in turn
    side = torch.cuda.Stream()
    bufs, graphs, outs = [], [], []
    for m in (300, 2100):  # routes in one launch; more than one
        x = torch.zeros((m, H), dtype=BF16, device="cuda")
        ids = torch.zeros((m, 8), dtype=torch.int64, device="cuda")

        def call():
            order = mx.sort_routes(ids, EXPERTS)
            return order, mx.combine_tokens(mx.sort_tokens(x, order), order)

        call()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side), torch.cuda.graph(g, stream=side):
            outs.append(call())
        torch.cuda.current_stream().wait_stream(side)
        bufs.append((x, ids))
        graphs.append(g)
    for rep in range(3):
        for x, ids in bufs:
            x.copy_(torch.randn(x.shape, device="cuda"))
            ids.copy_(torch.randint(-1, EXPERTS, ids.shape, device="cuda"))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for (x, ids), (order, out) in zip(bufs, outs):
            want = mx.sort_routes(ids, EXPERTS)
            assert all(torch.equal(a, b) for a, b in zip(order, want))
            assert torch.equal(out, mx.combine_tokens(mx.sort_tokens(x, want), want))


def test_backward_pass_in_a_graph():
    m = 130
    ids = torch.randint(0, EXPERTS, (m, TOP), device="cuda")
    x = torch.randn((m, H), device="cuda").requires_grad_()
    w = torch.rand((m, TOP), device="cuda").requires_grad_()
    up = torch.randn((m, H), device="cuda")

    def step():
        order = mx.sort_routes(ids, EXPERTS)
        rows = mx.sort_tokens(x, order)
        out = mx.combine_tokens(rows * rows, order, w)
        return (out.detach(), *torch.autograd.grad(out, (x, w), up))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        captured = step()
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(4):
        with torch.no_grad():
            x.normal_()
            w.uniform_()
            up.normal_()
            ids.random_(-1, EXPERTS)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, step()):
            assert torch.equal(a, b)


def test_capture_beside_a_live_eager_graph_is_refused():
    # the backward pass would wait for the eager graph's stream under capture
    ids = torch.randint(0, EXPERTS, (40, TOP), device="cuda")
    x = torch.randn((40, H), device="cuda").requires_grad_()
    w = torch.rand((40, TOP), device="cuda").requires_grad_()
    order = mx.sort_routes(ids, EXPERTS)
    eager = mx.combine_tokens(mx.sort_tokens(x, order), order, w)
    side = torch.cuda.Stream()
    rows = x.detach().repeat_interleave(TOP, 0)

    def capture(f):
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
            try:
                return graph, f()
            except RuntimeError as e:
                return graph, str(e)

    wide = torch.nn.functional.pad(rows, (0, 8))[:, :H]  # not contiguous: the general path
    for f in (lambda: mx.sort_tokens(x, order), lambda: mx.combine_tokens(rows, order, w),
              lambda: mx.combine_tokens(wide, order, w)):
        assert "live eager graph" in capture(f)[1]
        with torch.no_grad():
            graph, out = capture(f)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, f())
    del eager
    graph, out = capture(lambda: mx.combine_tokens(mx.sort_tokens(x, order), order, w).detach())
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, mx.combine_tokens(mx.sort_tokens(x, order), order, w))


def test_two_streams_and_threads(layer):
    sets = [cuda(rand_act(50 + m, (m, H))) for m in (5, 200, 64, 1)]
    want = [layer.run(s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    for s, st in zip(sets, streams):
        with torch.cuda.stream(st):
            got.append(layer.run(s))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        _same(a, b)
    out = [None] * len(sets)

    def work(i):
        with torch.cuda.stream(streams[i]):
            for _ in range(3):
                out[i] = layer.run(sets[i])
            streams[i].synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(sets))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for a, b in zip(out, want):
        _same(a, b)


def _calls(layer):
    x = cuda(rand_act(5, (9, H)))
    q, s = mx.dynamic_fp8_block_quant(x)
    ids = torch.randint(-1, EXPERTS, (9, TOP), device="cuda")
    order = mx.sort_routes(ids, EXPERTS)
    y = cuda(rand_act(6, (9 * TOP, H)))
    rows, srows = mx.dynamic_fp8_block_quant(y)
    w = torch.rand((9, TOP), device="cuda")
    bias = torch.ones(H, device="cuda")
    many = torch.randint(-1, EXPERTS, (5000, 8), device="cuda", dtype=torch.int32)
    linear, grouped = mx.linear_fp8_block, mx.grouped_linear_fp8_block
    return {
        "quant": lambda: mx.dynamic_fp8_block_quant(x),
        "quant_1d": lambda: mx.dynamic_fp8_block_quant(x[0].float()),
        "quant_3d": lambda: mx.dynamic_fp8_block_quant(x.view(3, 3, H).half()),
        "silu": lambda: mx.silu_mul_fp8_block_quant(x),
        "silu_3d": lambda: mx.silu_mul_fp8_block_quant(x.view(3, 3, H)),
        "linear": lambda: linear(q, s, layer.wo, layer.so),
        "linear_rows": lambda: linear(q, s.contiguous(), layer.wo, layer.so, bias, torch.float32),
        "linear_3d": lambda: linear(q.view(3, 3, H), s.view(3, 3, -1), layer.wo, layer.so, None,
                                    torch.float16),
        "linear_1d": lambda: linear(q[2], s[2], layer.wo, layer.so),
        "grouped": lambda: grouped(rows, srows, layer.w13, layer.s13, order),
        "gathered": lambda: grouped(q, s, layer.w13, layer.s13, order, gather=True,
                                    out_dtype=torch.float32),
        "routes": lambda: mx.sort_routes(ids, EXPERTS),
        "routes_many": lambda: mx.sort_routes(many, EXPERTS),
        "sort": lambda: mx.sort_tokens(x, order),
        "combine": lambda: mx.combine_tokens(y, order, w),
        "combine_ones": lambda: mx.combine_tokens(y.float(), order),
    }


def test_native_calls_equal_the_general_path(layer, monkeypatch):
    assert _lib.host() is not None
    calls = _calls(layer)
    native = {n: f() for n, f in calls.items()}
    monkeypatch.setattr(_lib, "host", lambda: None)
    for n, f in calls.items():
        a, b = native[n], f()
        assert type(a) is type(b)
        a, b = ((list(v) if isinstance(v, tuple) else [v]) for v in (a, b))
        assert len(a) == len(b)
        for p, q in zip(a, b):
            assert p.dtype == q.dtype and p.shape == q.shape and p.stride() == q.stride(), n
            if p.dtype.itemsize == 1:
                p, q = p.view(torch.uint8), q.view(torch.uint8)
            assert torch.equal(p, q), n


def test_native_gradients_equal_the_general_path(monkeypatch):
    order = mx.sort_routes(torch.randint(-1, EXPERTS, (70, TOP), device="cuda"), EXPERTS)
    wide = torch.randn((70, H + 8), device="cuda")
    ups = [wide[:, :H].contiguous(), wide[:, 1:H + 1], torch.ones((1, 1), device="cuda").expand(70, H),
           wide[:, :H].t().contiguous().t()]
    x0, y0 = torch.randn((70, H), device="cuda"), torch.randn((70 * TOP, H), device="cuda")
    w0 = torch.rand((70, TOP), device="cuda")

    def grads():
        got = []
        for dtype in (torch.float32, BF16):
            for up in ups:
                up = up.to(dtype)
                x, y = x0.to(dtype).requires_grad_(), y0.to(dtype).requires_grad_()
                w = w0.clone().requires_grad_()
                got += torch.autograd.grad(mx.combine_tokens(y, order, w), (y, w), up)
                got += torch.autograd.grad(mx.combine_tokens(y, order, w0), y, up)
                got += torch.autograd.grad(mx.combine_tokens(y, order), y, up)
                got += torch.autograd.grad(mx.combine_tokens(y.detach(), order, w), w, up)
                many = up.repeat(TOP, 1)
                got += torch.autograd.grad(mx.sort_tokens(x, order), x, many)
                got += torch.autograd.grad(mx.combine_tokens(mx.sort_tokens(x, order), order, w),
                                           (x, w), up)
        return got

    native = grads()
    monkeypatch.setattr(_lib, "host", lambda: None)
    general = grads()
    assert len(native) == len(general)
    for a, b in zip(native, general):
        assert a.dtype == b.dtype and torch.equal(a, b)


def test_second_derivatives_are_refused(monkeypatch):
    order = mx.sort_routes(torch.randint(0, EXPERTS, (9, TOP), device="cuda"), EXPERTS)
    for native in (True, False):
        if not native:
            monkeypatch.setattr(_lib, "host", lambda: None)
        x = torch.randn((9, 64), device="cuda").requires_grad_()
        w = torch.rand((9, TOP), device="cuda").requires_grad_()
        out = mx.combine_tokens(mx.sort_tokens(x, order), order, w).square().sum()
        for d in torch.autograd.grad(out, (x, w), create_graph=True):
            with pytest.raises(RuntimeError, match="differentiable once|once_differentiable"):
                d.sum().backward(retain_graph=True)


def test_native_calls_are_taken(layer, monkeypatch):
    # plain calls do not reach the general path's library calls
    calls = _calls(layer)
    lib = _lib.load()
    for name in ("mxfp4_quant_fp8_rows", "mxfp4_linear_fp8", "mxfp4_grouped_linear_fp8",
                 "mxfp4_sort_routes", "mxfp4_sort_tokens", "mxfp4_combine_tokens",
                 "mxfp4_combine_tokens_grad"):
        monkeypatch.setattr(lib, name, None)
    for f in calls.values():
        f()
    order = mx.sort_routes(torch.zeros((4, 2), dtype=torch.int64, device="cuda"), 3)
    x = torch.randn((4, 64), device="cuda").requires_grad_()
    w = torch.rand((4, 2), device="cuda").requires_grad_()
    mx.combine_tokens(mx.sort_tokens(x, order), order, w).sum().backward()
    with pytest.raises(TypeError):
        mx.dynamic_fp8_block_quant(layer.gate.t())


def test_a_routers_weights_learn_through_frozen_experts(layer):
    # the experts' products carry no gradient; the weights' comes from their outputs
    x = cuda(rand_act(21, (60, H)))
    r = layer.run(x)
    order = mx.ExpertOrder(r["offsets"], r["routes"], r["position"])
    logits = torch.randn((60, TOP), device="cuda").requires_grad_()
    out = mx.combine_tokens(r["y"], order, torch.softmax(logits, -1))
    up = cuda(rand_act(22, (60, H)))
    got, = torch.autograd.grad(out, logits, up)
    p = torch.softmax(logits.detach().double(), -1)
    dp = (r["y"].double()[order.position.long()] * up.double()[:, None]).sum(-1)
    want = p * (dp - (p * dp).sum(-1, keepdim=True))
    size = (r["y"].double()[order.position.long()] * up.double()[:, None]).abs().sum(-1).amax(-1)
    # the sum's, softmax' and its gradient's roundings
    assert ((got.double() - want).abs() <= 64 * 2.0 ** -24 * size[:, None]).all()
