"""GPU: the grouped router against an FP64 oracle.  Ids are the oracle's; a
weight is FP64 rounded once to FP32: within half a step (2^-24) of it, and 1e-12
for the FP64 arithmetic of both sides."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import mxfp4_amd as mx

from _helpers import cuda

pytestmark = pytest.mark.gpu
INF = math.inf


def oracle(logits, top_k, num_groups=1, topk_groups=1, scoring="softmax", bias=None,
           group_score="max", renormalize=True, scale=1.0):
    """Row by row, from the definition."""
    x = np.asarray(logits, dtype=np.float64)
    x = np.where(np.isnan(x), -INF, x)
    rows, e = x.shape
    b = None if bias is None else np.asarray(bias, dtype=np.float64)
    if b is not None:
        b = np.where(b < INF, b, -INF)  # NaN compares false
    size = e // num_groups
    ids = np.zeros((rows, top_k), dtype=np.int64)
    w = np.zeros((rows, top_k))
    for t in range(rows):
        r = x[t]
        if scoring == "sigmoid":
            s = np.array([1 / (1 + math.exp(-v)) if v > -700 else 0.0 for v in r])
        else:
            top = r.max()
            p = np.array([0.0 if v == -INF else 1.0 if v == top else math.exp(v - top) for v in r])
            s = p / p.sum() if p.sum() > 0 else p
        v = r if b is None else s + b
        g = (s if group_score == "top2" else v) if b is None else v
        value = []
        for q in range(num_groups):
            best = sorted(g[q * size:(q + 1) * size], reverse=True)
            value.append(best[0] if group_score == "max" or num_groups == 1 else best[0] + best[1])
        kept = sorted(range(num_groups), key=lambda q: (-value[q], q))[:topk_groups]
        cand = [i for i in range(e) if i // size in kept]
        pick = sorted(cand, key=lambda i: (-v[i], i))[:top_k]
        sel = np.array([0.0 if v[i] == -INF else s[i] for i in pick])
        if renormalize:
            if scoring == "softmax":  # the quotient, also where the scores underflow
                m = max((r[i] for i in pick if v[i] != -INF), default=-INF)
                sel = np.array([0.0 if v[i] == -INF or r[i] == -INF else
                                1.0 if r[i] == m else math.exp(r[i] - m) for i in pick])
            sel = sel / sel.sum() if sel.sum() > 0 else sel
        ids[t], w[t] = pick, sel * np.float64(np.float32(scale))
    return w, ids


def check(logits, top_k, ids_dtype=torch.int64, **kw):
    w, ids = mx.route_topk_grouped(cuda(logits), top_k, ids_dtype=ids_dtype,
                                   **{**kw, "bias": None if kw.get("bias") is None
                                      else cuda(kw["bias"])})
    assert w.dtype == torch.float32 and ids.dtype == ids_dtype
    kw = {**kw, "bias": None if kw.get("bias") is None else kw["bias"].numpy()}
    ow, oids = oracle(logits.float().reshape(-1, logits.shape[-1]).numpy(), top_k, **kw)
    assert w.shape == ids.shape == (*logits.shape[:-1], top_k)
    assert np.array_equal(ids.reshape(-1, top_k).cpu().numpy(), oids)
    d = np.abs(w.reshape(-1, top_k).double().cpu().numpy() - ow)
    assert (d <= (2.0 ** -24 + 1e-12) * np.abs(ow) + 2.0 ** -150).all(), d.max()
    return w, ids


def _logits(rows, e, seed, dtype=torch.float32, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    return (spread * torch.randn((rows, e), generator=g)).to(dtype)


def _bias(e, seed):
    return 0.1 * torch.randn(e, generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("e,groups,keep,top_k", [
    (1, 1, 1, 1), (8, 1, 1, 2), (60, 1, 1, 4), (60, 5, 2, 24), (64, 64, 20, 8), (96, 3, 2, 6),
    (128, 8, 3, 8), (160, 8, 3, 6), (256, 8, 4, 8), (384, 12, 1, 32), (1000, 20, 7, 17),
    (1024, 1, 1, 64), (1024, 64, 4, 64)])
@pytest.mark.parametrize("scoring,bias,value", [
    ("softmax", False, "max"), ("softmax", True, "top2"), ("sigmoid", False, "top2"),
    ("sigmoid", True, "max"), ("sigmoid", True, "top2")])
def test_sizes(e, groups, keep, top_k, scoring, bias, value):
    if value == "top2" and groups > 1 and e == groups:
        value = "max"
    check(_logits(7, e, e + top_k), top_k, num_groups=groups, topk_groups=keep, scoring=scoring,
          bias=_bias(e, 3) if bias else None, group_score=value, scale=2.5)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_types_with_many_ties(dtype, renorm, scoring):
    # eighths: several equal logits in each row, and equal group values
    logits = (_logits(65, 64, 5) * 2).round().div(8).to(dtype)
    for kw in (dict(), dict(num_groups=8, topk_groups=3),
               dict(num_groups=8, topk_groups=3, group_score="top2", bias=torch.zeros(64)),
               dict(bias=torch.arange(64).remainder(3).div(4.0))):
        check(logits, 6, torch.int32, scoring=scoring, renormalize=renorm, **kw)


@pytest.mark.parametrize("rows", [1, 3, 4, 5, 1021])
def test_rows_strides_and_shapes(rows):
    kw = dict(num_groups=8, topk_groups=4, scoring="sigmoid", group_score="top2")
    logits, bias = _logits(rows, 128, rows), _bias(128, 1)
    w, ids = check(logits, 8, bias=bias, **kw)
    wide = torch.full((rows, 2, 140), math.nan)
    wide[:, 1, 5:133] = logits
    b2 = torch.full((128, 2), math.nan)
    b2[:, 0] = bias
    w2, ids2 = mx.route_topk_grouped(cuda(wide)[:, 1, 5:133], 8, bias=cuda(b2)[:, 0], **kw)
    assert torch.equal(w, w2) and torch.equal(ids, ids2)
    wt, idt = mx.route_topk_grouped(cuda(logits.T.contiguous()).T, 8, bias=cuda(bias), **kw)
    assert torch.equal(w, wt) and torch.equal(ids, idt)
    w3, ids3 = mx.route_topk_grouped(cuda(logits)[:, None], 8, bias=cuda(bias), **kw)
    assert w3.shape == (rows, 1, 8) and torch.equal(w3[:, 0], w) and torch.equal(ids3[:, 0], ids)
    we, ie = mx.route_topk_grouped(cuda(logits)[:0], 8, bias=cuda(bias), **kw)
    assert we.shape == ie.shape == (0, 8)


@pytest.mark.parametrize("e,groups,keep", [(256, 8, 4), (160, 2, 1), (208, 1, 1), (256, 16, 3)])
@pytest.mark.parametrize("scoring,renorm,bias", [("sigmoid", True, True), ("softmax", False, False),
                                                 ("softmax", True, True)])
def test_many_rows_and_few_choose_alike(e, groups, keep, scoring, renorm, bias):
    # the layout of a row over lanes goes by the number of rows
    logits = cuda(_logits(2500, e, 77))
    kw = dict(num_groups=groups, topk_groups=keep, scoring=scoring, renormalize=renorm,
              bias=cuda(_bias(e, 5)) if bias else None, group_score="top2" if bias else "max")
    w, ids = mx.route_topk_grouped(logits, 8, **kw)
    few = [mx.route_topk_grouped(t, 8, **kw) for t in logits.split(700)]
    assert torch.equal(ids, torch.cat([f[1] for f in few]))
    assert torch.allclose(w, torch.cat([f[0] for f in few]), rtol=2.0 ** -23, atol=0)
    check(logits[2400:2460].cpu(), 8, **{**kw, "bias": kw["bias"].cpu() if bias else None})
    assert torch.equal(ids[2400:2460], few[3][1][300:360])


def test_more_rows_than_a_grid_of_workgroups():
    logits = _logits(70001, 32, 9, torch.bfloat16)
    w, ids = mx.route_topk_grouped(cuda(logits), 3, scoring="sigmoid")
    pick = torch.arange(0, 70001, 997)
    ow, oids = oracle(logits[pick].float().numpy(), 3, scoring="sigmoid")
    assert np.array_equal(ids[cuda(pick)].cpu().numpy(), oids)
    assert np.allclose(w[cuda(pick)].cpu().numpy(), ow, rtol=2.0 ** -23, atol=0)
    assert int(ids.min()) >= 0 and int(ids.max()) < 32
    s = w.double().sum(-1)
    assert float((s - 1).abs().max()) <= 3 * 2.0 ** -24


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
def test_masked_and_extreme_logits(scoring, renorm):
    low = torch.finfo(torch.float32).min
    x = _logits(12, 64, 21)
    x[0] = -INF                       # nothing left
    x[1] = low
    x[2, 3:] = -INF                   # fewer than top_k
    x[3, ::2] = math.nan
    x[4] = math.nan
    x[5] = torch.linspace(-3e38, 3e38, 64)
    x[6, 7] = 3e38
    x[7] = 100.0 + x[7] * 1e-5        # all near one value
    x[8] = -600.0 + x[8]              # scores far below FP32
    x[9] = 0.0
    x[10, 5] = INF
    x[11] = 40.0 + x[11]              # sigmoid 1 in FP32
    for kw in (dict(), dict(num_groups=8, topk_groups=2)):
        check(x, 6, scoring=scoring, renormalize=renorm, **kw)
    # sums with a bias: rows whose scores all vanish go by the bias alone
    check(x, 6, scoring=scoring, renormalize=renorm, num_groups=8, topk_groups=2,
          group_score="top2", bias=_bias(64, 2))


@pytest.mark.parametrize("e,rows", [(64, 40), (256, 40), (256, 2060), (512, 9)])
def test_equal_and_nearly_equal_values_with_a_bias(e, rows):
    # whole rows of equal values; values that differ in the last bits of FP64,
    # which the keys do not hold
    x = torch.zeros((rows, e))
    bias = torch.zeros(e)
    for b in (bias, bias + torch.arange(e).remainder(4) * 0.25,
              (torch.arange(e).flip(0).double() * 2.0 ** -44).float(),
              torch.where(torch.arange(e) == e - 3, 2.0 ** -53, 0.0).float()):
        for scoring in ("sigmoid", "softmax"):
            kw = dict(scoring=scoring, bias=b, num_groups=8, topk_groups=3, group_score="top2")
            w, ids = check(x[:9], 8, **kw)
            all_w, all_ids = mx.route_topk_grouped(cuda(x), 8, **{**kw, "bias": cuda(b)})
            assert (all_ids == ids[0]).all() and (all_w == w[0]).all()


def test_experts_out_of_service():
    x = _logits(9, 64, 30)
    for off in ([5], list(range(0, 64, 3)), list(range(8, 64)), list(range(64))):
        bias = _bias(64, 4)
        bias[off] = -INF
        bias[off[0]] = math.nan
        bias[off[-1]] = INF
        for value in ("max", "top2"):
            w, ids = check(x, 10, num_groups=8, topk_groups=2, scoring="sigmoid", bias=bias,
                           group_score=value)
            gone = torch.isin(ids.cpu(), torch.tensor(off))
            assert (w.cpu()[gone] == 0).all()
            assert all(len(set(r)) == 10 for r in ids.tolist())


def test_choice_next_to_a_border():
    # values closer than FP32 can tell: sigmoid(12 + d) of neighbouring floats,
    # and biases that differ by one FP32 step
    base = torch.full((1, 64), 12.0)
    step = torch.nextafter(base, torch.tensor(INF)) - base
    x = base + step * torch.randperm(64, generator=torch.Generator().manual_seed(0)).float()
    assert torch.sigmoid(x).unique().numel() < 64
    check(x, 8, scoring="sigmoid", bias=torch.zeros(64))
    check(x, 8, scoring="sigmoid")
    check(x, 8, scoring="softmax", bias=torch.full((64,), 1.0))
    b = torch.full((64,), 0.5)
    b[40] = torch.nextafter(torch.tensor(0.5), torch.tensor(1.0))
    check(torch.zeros(2, 64), 3, scoring="sigmoid", bias=b)


def test_without_groups_or_bias_it_is_route_topk():
    x = cuda(_logits(33, 128, 50))
    w, ids = mx.route_topk_grouped(x, 8)
    w0, ids0 = mx.route_topk(x, 8)
    assert torch.equal(ids, ids0)
    assert torch.allclose(w, w0, rtol=2e-6, atol=0)
    # all groups kept, or one group: no choice among groups
    for kw in (dict(num_groups=16, topk_groups=16, group_score="top2"), dict(num_groups=1)):
        w1, ids1 = mx.route_topk_grouped(x, 8, **kw)
        assert torch.equal(w1, w) and torch.equal(ids1, ids)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("e,top_k", [(64, 6), (256, 8), (64, 12)])
def test_with_a_bias_only_the_bias_masks(scoring, e, top_k):
    # the documented rule: a logit of -inf or NaN has score 0 and value bias
    x = _logits(9, e, 44)
    off = [1, 2, 17, e - 1]
    x[:, off[:2]], x[:, off[2:]] = -INF, math.nan
    bias = _bias(e, 8)
    bias[off] = 2.0  # above every score + bias
    for kw in (dict(), dict(num_groups=8, topk_groups=3, group_score="top2")):
        w, ids = check(x, top_k, scoring=scoring, bias=bias, **kw)
        masked = torch.isin(ids.cpu(), torch.tensor(off))
        assert masked[:, 0].all() and (w.cpu()[masked] == 0).all()
        shut = bias.clone()
        shut[off] = -INF
        w, ids = check(x, top_k, scoring=scoring, bias=shut, **kw)
        assert not torch.isin(ids.cpu(), torch.tensor(off)).any()
        # without a bias the logit masks
        w, ids = check(x, top_k, scoring=scoring, **kw)
        assert not torch.isin(ids.cpu(), torch.tensor(off)).any()


@pytest.mark.parametrize("e,groups", [(64, 8), (256, 8), (60, 5), (32, 16)])
def test_two_best_of_a_group_with_one_expert_left(e, groups):
    # its sum is -inf, as of a group with none; the lower id is kept first
    x, size = _logits(9, e, 45), e // groups
    for alone in (0, groups // 2, groups - 1):
        bias = _bias(e, 9)
        bias[alone * size + 1:(alone + 1) * size] = -INF
        bias[alone * size] = 3.0
        for top_k in (2, min(10, 2 * size)):
            w, ids = check(x, top_k, num_groups=groups, topk_groups=2, scoring="sigmoid",
                           bias=bias, group_score="top2")
            assert (ids != alone * size).all()
            # by the largest value the group is the first choice
            w, ids = check(x, top_k, num_groups=groups, topk_groups=2, scoring="sigmoid",
                           bias=bias)
            assert (ids[:, 0] == alone * size).all()
    bias = torch.full((e,), -INF)
    bias[(groups - 1) * size] = 1.0  # the only expert left, in a group that is not kept
    w, ids = check(x, 2, num_groups=groups, topk_groups=2, scoring="sigmoid", bias=bias,
                   group_score="top2")
    assert (ids.cpu() == torch.tensor([0, 1])).all() and (w == 0).all()
