"""GPU: the 8-bit operators and the grouped router as a decoder layer runs them,
one after the other, in a captured graph, on several streams and from several
threads, and their native calls against the general path."""

from __future__ import annotations

import threading

import numpy as np
import pytest
import torch

import mxfp4_amd as mx
from mxfp4_amd import _lib
from oracle import mxfp4_oracle as O

from _helpers import cuda, rand_act, rand_mxfp4

pytestmark = pytest.mark.gpu
H, N, O_K, EXPERTS, TOP, INTER = 512, 768, 640, 32, 4, 256


class Layer:
    def __init__(self):
        rng = np.random.default_rng(11)
        self.wq, self.sq = mx.dynamic_int8_quant(cuda(rand_act(1, (N, H))))
        self.wo, self.so = mx.dynamic_int8_quant(cuda(rand_act(2, (H, O_K))))
        self.n1, self.n2 = cuda(1 + 0.1 * rand_act(3, (H,))), cuda(1 + 0.1 * rand_act(4, (H,)))
        self.gate = cuda(rand_act(5, (EXPERTS, H)) * 0.05)
        self.bias = cuda(0.05 * rand_act(6, (EXPERTS,)).float())
        w13, s13 = rand_mxfp4(rng, (EXPERTS, 2 * INTER), H, lo=116, hi=121)
        self.w13_host = (w13, s13)
        self.w13, self.s13 = cuda(w13), cuda(s13)
        self.one = torch.ones(1, device="cuda")
        self.ones = torch.ones(EXPERTS, device="cuda")

    def run(self, x, residual, attn):
        a = mx.rms_norm_quant(x, self.n1, residual)
        qkv = mx.linear_int8_w8a8(a.q, a.scales, self.wq, self.sq)
        o8, so = mx.dynamic_int8_quant(attn)
        o = mx.linear_int8_w8a8(o8, so, self.wo, self.so)
        b = mx.rms_norm_quant(o, self.n2, a.residual, fmt="mxfp8_e4m3", normed=True)
        logits = b.normed.float() @ self.gate.float().T
        w, ids = mx.route_topk_grouped(logits, TOP, num_groups=4, topk_groups=2,
                                       scoring="sigmoid", bias=self.bias, group_score="top2",
                                       scale=2.5)
        sorted_ids, expert_ids, npp = mx.make_routing(ids, 32, EXPERTS)
        c = torch.empty((x.shape[0], TOP, 2 * INTER), dtype=torch.bfloat16, device="cuda")
        mx.fused_moe_mxfp4(b.q, self.w13, c, self.one, self.ones, b.scales, self.s13, w, ids,
                           sorted_ids, expert_ids, npp, True, TOP, False, False,
                           {"BLOCK_SIZE_M": 32}, torch.bfloat16)
        return {"q": a.q, "scales": a.scales, "residual": a.residual, "qkv": qkv, "o8": o8,
                "so": so, "o": o, "q8": b.q, "mx": b.scales, "residual2": b.residual,
                "normed": b.normed, "logits": logits, "w": w, "ids": ids, "c": c}


@pytest.fixture(scope="module")
def layer():
    return Layer()


def _inputs(m, seed):
    return tuple(cuda(rand_act(seed + i, (m, k))) for i, k in enumerate((H, H, O_K)))


def _same(a, b):
    for name in a:
        x, y = a[name], b[name]
        if x.dtype.itemsize == 1:
            x, y = x.view(torch.uint8), y.view(torch.uint8)
        assert torch.equal(x, y), name


@pytest.mark.parametrize("m", [1, 37, 300])
def test_layer_against_fp64_step_by_step(layer, m):
    # each step on the values the step before it gave
    r = layer.run(*_inputs(m, 100 + m))
    half = 2.0 ** -8 + 2.0 ** -20  # bf16, and FP32 roundings
    d = lambda t: t.double()  # noqa: E731

    def close(got, want):
        assert ((d(got) - want).abs() <= half * want.abs() + 1e-30).all()

    close(r["qkv"], (d(r["q"]) @ d(layer.wq).T) * d(r["scales"])[:, None] * d(layer.sq))
    close(r["o"], (d(r["o8"]) @ d(layer.wo).T) * d(r["so"])[:, None] * d(layer.so))
    h = d((r["o"].float() + r["residual"].float()))
    assert torch.equal(r["residual2"], h.to(torch.bfloat16))
    y = h * d(layer.n2) / torch.sqrt((h * h).mean(-1, keepdim=True) + 1e-6)
    close(r["normed"], y)
    v8 = d(r["q8"]).view(m, -1, 32) * torch.exp2(d(r["mx"]) - 127)[..., None]
    # half a step of e4m3, of its subnormals, and up to 64 above the largest value
    unit = torch.exp2(d(r["mx"]) - 127).repeat_interleave(32, -1)
    z = y.abs() / unit
    tol = torch.where(z > 448, z - 448, torch.clamp(z * 2.0 ** -4, min=2.0 ** -10))
    assert ((v8.view(m, H) - y).abs() <= (tol + z * 2.0 ** -20) * unit).all()
    s = torch.sigmoid(d(r["logits"]))
    pair = (s + d(layer.bias)).view(m, 4, -1)
    kept = pair.topk(2, -1).values.sum(-1).topk(2, -1).indices
    inside = torch.zeros((m, 4), dtype=torch.bool, device="cuda").scatter_(1, kept, True)
    v = (s + d(layer.bias)).masked_fill(~inside.repeat_interleave(EXPERTS // 4, 1), -1e9)
    ids = v.topk(TOP, -1).indices
    assert torch.equal(ids, r["ids"])
    w = s.gather(1, ids)
    w = 2.5 * w / w.sum(-1, keepdim=True)
    assert torch.allclose(d(r["w"]), w, rtol=2.0 ** -23, atol=0)
    b = torch.from_numpy(O.dequant_values(*layer.w13_host, "f32")).cuda().double()
    x = v8.view(m, H)
    for t in range(0, m, max(1, m // 7)):
        want = torch.stack([b[int(e)] @ x[t] * d(r["w"])[t, i] for i, e in enumerate(r["ids"][t])])
        err = (d(r["c"][t]) - want).norm() / want.norm()
        assert float(err) <= O.NORM_TOL


@pytest.mark.parametrize("m", [1, 64, 300])
def test_graph_replays_equal_eager(layer, m):
    buf = _inputs(m, 7)
    layer.run(*buf)
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            captured = layer.run(*buf)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for rep in range(4):
        new = _inputs(m, 1000 * rep + 3)
        for t, v in zip(buf, new):
            t.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        _same(captured, layer.run(*new))


def test_two_streams_and_two_threads(layer):
    sets = [_inputs(m, 50 + m) for m in (5, 200, 64, 1)]
    want = [layer.run(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    for s, st in zip(sets, streams):
        with torch.cuda.stream(st):
            got.append(layer.run(*s))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        _same(a, b)
    out = [None] * len(sets)

    def work(i):
        with torch.cuda.stream(streams[i]):
            for _ in range(3):
                out[i] = layer.run(*sets[i])
            streams[i].synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(sets))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for a, b in zip(out, want):
        _same(a, b)


def test_native_calls_equal_the_general_path(layer, monkeypatch):
    host = _lib.host()
    assert host is not None
    x, r, attn = _inputs(9, 5)
    calls = {
        "route": lambda: mx.route_topk_grouped(x[:, :64], 3, num_groups=4, topk_groups=2),
        "route_bias": lambda: mx.route_topk_grouped(
            x[:, :EXPERTS].contiguous().float(), 3, scoring="sigmoid", bias=layer.bias,
            renormalize=False, scale=0.5, ids_dtype=torch.int32),
        "route_half": lambda: mx.route_topk_grouped(
            x[:, :64].contiguous().half(), 5, num_groups=8, topk_groups=3, group_score="top2"),
        "norm": lambda: mx.rms_norm_quant(x, layer.n1),
        "norm_res": lambda: mx.rms_norm_quant(x, layer.n1.float(), r, normed=True, eps=1e-3),
        "norm_mx": lambda: mx.rms_norm_quant(x.float(), layer.n1.float(), r.float(),
                                             fmt="mxfp8_e5m2"),
        "norm_3d": lambda: mx.rms_norm_quant(x.view(3, 3, H), layer.n1, fmt="mxfp8_e4m3"),
        "norm_1d": lambda: mx.rms_norm_quant(x[0], layer.n1),
        "int8": lambda: mx.dynamic_int8_quant(attn),
        "int8_1d": lambda: mx.dynamic_int8_quant(attn[1].half()),
        "w8a8": lambda: mx.linear_int8_w8a8(*mx.dynamic_int8_quant(x), layer.wq, layer.sq),
        "w8a8_bias": lambda: mx.linear_int8_w8a8(
            layer.wo[:5], layer.so[:5, None], layer.wo, layer.so[:, None],
            torch.ones(H, device="cuda"), torch.float32),
        "w8a8_3d": lambda: mx.linear_int8_w8a8(
            layer.wo[:6].view(2, 3, O_K), layer.so[:6].view(2, 3), layer.wo, layer.so, None,
            torch.float16),
    }
    native = {n: f() for n, f in calls.items()}
    monkeypatch.setattr(_lib, "host", lambda: None)
    for n, f in calls.items():
        a, b = native[n], f()
        a, b = ((list(v) if isinstance(v, tuple) else [v]) for v in (a, b))
        assert len(a) == len(b)
        for p, q in zip(a, b):
            assert (p is None) == (q is None), n
            if p is not None:
                assert p.dtype == q.dtype and p.shape == q.shape, n
                v = torch.uint8 if p.dtype.itemsize == 1 else p.dtype
                assert torch.equal(p.view(v), q.view(v)), n


def test_native_calls_are_taken(layer, monkeypatch):
    # plain calls do not reach the general path's library calls
    x, r, _ = _inputs(4, 5)
    a, s = mx.dynamic_int8_quant(x)
    lib = _lib.load()
    for name in ("mxfp4_moe_route_grouped", "mxfp4_rms_norm_quant", "mxfp4_quant_int8",
                 "mxfp4_linear_w8a8"):
        monkeypatch.setattr(lib, name, None)
    mx.route_topk_grouped(x[:, :64].contiguous(), 3)
    mx.rms_norm_quant(x, layer.n1, r)
    mx.dynamic_int8_quant(x)
    mx.linear_int8_w8a8(a, s, layer.wq, layer.sq)
    with pytest.raises(TypeError):
        mx.dynamic_int8_quant(x.T)


@pytest.mark.parametrize("fmt", ["mxfp8_e4m3", "mxfp8_e5m2"])
@pytest.mark.parametrize("m,k", [(5, 512), (300, 512), (300, 544), (40, 96)])
def test_tokens_that_are_not_finite_stay_so_through_both_products(fmt, m, k):
    # scale NaN / byte 255 with zeros: NaN in the token's outputs, no other changed
    rng = np.random.default_rng(3)
    n, bad = 64, [0, m // 2, m - 1]
    x, w = cuda(rand_act(60, (m, k))), cuda(1 + 0.1 * rand_act(61, (k,)))
    wq, sq = mx.dynamic_int8_quant(cuda(rand_act(62, (n, k))))
    b, bs = (cuda(t) for t in rand_mxfp4(rng, (EXPERTS, n), k, lo=116, hi=121))
    ids = (torch.arange(m * TOP, device="cuda") * 7 % EXPERTS).view(m, TOP)
    weights = torch.full((m, TOP), 0.25, device="cuda")
    one, ones = torch.ones(1, device="cuda"), torch.ones(EXPERTS, device="cuda")

    def run(x):
        q = mx.rms_norm_quant(x, w)
        y = mx.linear_int8_w8a8(q.q, q.scales, wq, sq)
        f = mx.rms_norm_quant(x, w, fmt=fmt)
        sorted_ids, expert_ids, npp = mx.make_routing(ids, 32, EXPERTS)
        c = torch.zeros((m, TOP, n), dtype=torch.bfloat16, device="cuda")
        mx.fused_moe_mxfp4(f.q, b, c, one, ones, f.scales, bs, weights, ids, sorted_ids,
                           expert_ids, npp, False, TOP, False, False, {"BLOCK_SIZE_M": 32},
                           torch.bfloat16)
        return y, c

    clean = run(x)
    x2 = x.clone()
    x2[bad[0], 3], x2[bad[1], k - 1], x2[bad[2]] = float("nan"), float("inf"), -float("inf")
    rest = torch.ones(m, dtype=torch.bool, device="cuda")
    rest[bad] = False
    for got, want in zip(run(x2), clean):
        assert got[bad].isnan().all() and want.isfinite().all()
        assert torch.equal(got[rest], want[rest])
