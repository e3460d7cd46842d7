"""Router gating and its gradient against the 64-bit oracle: ids exactly, weights within fp32 rounding.

Tolerance of a weight, relative: it is exp(d) / sum of exps (or built from such terms) with d = x - max in fp32.  The rounding of d
shifts the exponential by |d| 2^-24; the exponential, the division and the products add a unit of the last place or two each (2^-23);
a sum of at most 1024 terms in a tree of 16 + 6 additions adds 22 * 2^-24.  Twice (numerator and sum): 2 (dmax + 32) 2^-24.
A gradient w (g - sum g w) is bounded by that times the sum of its terms' magnitudes."""
import numpy as np
import pytest
import torch

from oracle import moe_block as O

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _logits(t, e, dtype, seed, masked=0.0):
    gen = torch.Generator().manual_seed(seed)
    x = 2.0 * torch.randn((t, e), generator=gen) + torch.randn(e, generator=gen)
    if masked:
        x = x.masked_fill(torch.rand((t, e), generator=gen) < masked, float("-inf"))
    return x.to(dtype)


def _rel(x):
    f = x[np.isfinite(x)]
    return 2 * (min(f.max() - f.min() if f.size else 0, 110.0) + 32) * 2.0 ** -24   # (exp(-104) is 0 in fp32)


def _check(es, x, topk, bias=None, scoring="softmax", renormalize=True, scale=1.0, groups=1, topk_groups=1, grad=True):
    dev = x.cuda()
    ids, w = es.es_topk_gating(dev, topk, None if bias is None else bias.cuda(), scoring, renormalize, scale, groups, topk_groups)
    xd = x.double().numpy()
    want_ids, want_w = O.topk_gating(xd, topk, None if bias is None else bias.double().numpy(), scoring, renormalize, scale, groups, topk_groups)
    assert ids.dtype == torch.int32 and w.dtype == torch.float32 and ids.shape == w.shape == (x.size(0), topk)
    assert np.array_equal(ids.cpu().numpy(), want_ids)
    got = w.double().cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(want_w))
    ok = ~np.isnan(want_w)
    tol = _rel(xd)
    assert (np.abs(got - want_w)[ok] <= tol * np.abs(want_w[ok]) + 1e-44).all(), np.nanmax(np.abs(got - want_w) / np.abs(want_w))
    if grad and ok.all():
        g = torch.randn(w.shape, generator=torch.Generator().manual_seed(7))
        d = es.es_topk_gating_backward(g.cuda(), dev, ids, scoring, renormalize, scale)
        assert d.dtype == x.dtype and d.shape == x.shape
        want = O.gating_grad(g.double().numpy(), xd, want_ids, scoring, renormalize, scale)
        # every term of a gradient is a score (or its weight) times at most the row's sum of |g|
        mag = np.abs(g.double().numpy()).sum(axis=1, keepdims=True) * abs(scale) * np.ones_like(xd)
        s = np.stack([O.scores(r, scoring) for r in xd])
        if renormalize or scoring == "sigmoid":
            full = np.zeros_like(xd)
            for i in range(x.size(0)):
                full[i, want_ids[i][want_ids[i] >= 0]] = 1.0
            s = full
        bound = 4 * tol * mag * s + HALF_STEP[x.dtype] * np.abs(want) + (2.0 ** -25 if x.dtype == torch.float16 else 1e-40)
        assert (np.abs(d.double().cpu().numpy() - want) <= bound).all()


@pytest.mark.parametrize("t,e,topk", [(1, 1, 1), (1, 256, 8), (5, 3, 3), (7, 64, 64), (33, 65, 6), (9, 130, 10), (4, 1000, 13), (3, 1024, 64),
                                      (257, 128, 8), (1003, 60, 4)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [False, True])
def test_gating(esmoe, t, e, topk, scoring, renormalize):
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        _check(esmoe, _logits(t, e, dtype, t + e), topk, None, scoring, renormalize, 2.5)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,kept", [(1, 1), (8, 2), (8, 6)])
def test_low_and_high_biases(esmoe, scoring, groups, kept):
    """Biases far below the rest decide between groups like any other, and experts that have one are chosen when nothing else is left."""
    g = torch.Generator().manual_seed(5)
    x = torch.randn((33, 128), generator=g)
    x[5, 16:] = float("-inf")
    for high in (0.0, 1000.0):
        for low in (float("-inf"), torch.finfo(torch.float32).min, -1e4, -65.0):
            b = high + torch.rand(128, generator=g) * 0.2
            b[32:64], b[3], b[127] = low, low, low
            b[64:68] -= torch.rand(4, generator=g) + 80.0
            b[66:] -= 0.0 if low < -1e4 else 70 * torch.rand(62, generator=g)
            for topk in (1, 6, 16):
                with np.errstate(over="ignore"):
                    _check(esmoe, x, topk, b, scoring, True, grad=False, groups=groups, topk_groups=kept)


@pytest.mark.parametrize("t,e,topk,groups,topk_groups", [(9, 256, 8, 1, 1), (130, 256, 8, 8, 4), (5, 60, 7, 4, 3), (11, 64, 5, 64, 5), (17, 1024, 16, 8, 1),
                                                         (3, 36, 12, 3, 1), (6, 100, 10, 2, 2), (40, 512, 8, 16, 3), (21, 72, 4, 36, 3)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_gating_with_bias_and_groups(esmoe, t, e, topk, groups, topk_groups, scoring):
    bias = 0.3 * torch.randn(e, generator=torch.Generator().manual_seed(e))
    for masked in (0.0, 0.5):
        x = _logits(t, e, torch.float32, t, masked)
        _check(esmoe, x, topk, bias, scoring, True, 1.0, groups, topk_groups)
        _check(esmoe, x.to(torch.bfloat16), topk, None, scoring, False, 1.0, groups, topk_groups)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [False, True])
def test_masks_ties_and_extremes(esmoe, scoring, bias):
    inf, nan, low = float("inf"), float("nan"), torch.finfo(torch.float32).min
    x = torch.zeros((12, 70))
    x[1] = -inf                      # nothing left
    x[2], x[2, 69] = -inf, 0.5       # one left
    x[3], x[3, 5:8] = -inf, -200.0   # three, whose sigmoids are 0 in fp32
    x[4] = low                       # the type's lowest value is a logit like any other
    x[5], x[5, 30] = low, 0.0
    x[6, 66], x[6, 3] = nan, 4.0
    x[7, 1], x[7, 2] = -0.0, 0.0
    x[8, ::2] = -inf
    x[9] = torch.arange(70) % 7      # ties between lanes and within one
    x[10] = 90.0
    x[11, 9] = 150.0
    b = None
    if bias:
        b = torch.zeros(70)
        b[4], b[11] = -inf, 1.0      # an expert that is out by its bias
    for renormalize in (False, True):
        _check(esmoe, x, 6, b, scoring, renormalize, grad=not bias)
    y = torch.zeros((2, 70))
    y[0, 3], y[1, 3], y[1, 60] = inf, inf, nan
    ids, w = esmoe.es_topk_gating(y.cuda(), 3, None if b is None else b.cuda(), scoring)
    assert ((ids >= 0) & (ids < 70)).all() and ids[1, 0].item() == (60 if scoring == "sigmoid" or not bias else 0)
    if not bias:
        assert ids[0].tolist() == [3, 0, 1] and ids[1].tolist() == [60, 3, 0]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("experts", [60, 128, 200, 256, 300])
def test_order_at_the_ends_of_the_range(esmoe, dtype, experts):
    """NaN and the largest values at the first and last experts, values that differ in the last place of the type, masks by the type's lowest
    value beside ordinary logits, one expert far above all others."""
    info = torch.finfo(dtype)
    x = _logits(40, experts, dtype, experts)
    x[0, 0], x[1, -1], x[2, 0], x[2, -1] = float("nan"), float("nan"), float("nan"), float("nan")
    x[3, 0], x[4, -1], x[5, :] = info.max, info.max, info.min
    x[6, ::2] = info.min
    x[7, 1:] = info.min
    x[8] = 1.0 + info.eps * torch.arange(experts)
    x[9] = 1.0 + info.eps * torch.arange(experts).flip(0)
    x[10] = -1.0 - info.eps * torch.arange(experts)
    x[11] = info.tiny * torch.arange(experts)
    x[12, experts // 2] = 30000.0
    x[13:20] = x[13:20].round()
    bias = 0.1 * torch.randn(experts, generator=torch.Generator().manual_seed(3))
    groups = 4
    for scoring in ("softmax", "sigmoid"):
        for args in ((None, 1, 1), (bias, 1, 1), (None, groups, 2), (bias, groups, 3), (100 * bias, 1, 1), (1e-6 * bias, groups, 1)):
            _check(esmoe, x, 8, args[0], scoring, True, 1.0, args[1], args[2], grad=False)


def test_gradient_of_given_ids(esmoe):
    """Ids that no gating would give: one twice, ids of no expert; NaN gradients at places that do not count."""
    x = _logits(6, 40, torch.float32, 2)
    ids = torch.tensor([[3, 3, 7], [-1, 5, 40], [0, 39, 1 << 30], [-5, -1, -1], [1, 1, 1], [12, -1, 12]], dtype=torch.int32)
    g = torch.randn((6, 3), generator=torch.Generator().manual_seed(1))
    g[(ids < 0) | (ids >= 40)] = float("nan")
    for scoring in ("softmax", "sigmoid"):
        for renormalize in (False, True):
            d = esmoe.es_topk_gating_backward(g.cuda(), x.cuda(), ids.cuda(), scoring, renormalize, 2.0).double().cpu().numpy()
            want = O.gating_grad(g.double().numpy(), x.double().numpy(), ids.numpy(), scoring, renormalize, 2.0)
            mag = np.nansum(np.abs(g.double().numpy()), axis=1, keepdims=True) * 2.0
            assert (np.abs(d - want) <= 4 * _rel(x.double().numpy()) * mag + 1e-40).all()


def test_gradient_of_masked_rows(esmoe):
    x = _logits(5, 33, torch.float32, 4, 0.6)
    x[2] = float("-inf")
    for scoring in ("softmax", "sigmoid"):
        for renormalize in (False, True):
            ids, _ = esmoe.es_topk_gating(x.cuda(), 20, None, scoring, renormalize)
            d = esmoe.es_topk_gating_backward(torch.ones(5, 20, device="cuda"), x.cuda(), ids, scoring, renormalize)
            assert torch.isfinite(d).all() and (d[2] == 0).all() and (d.cpu()[torch.isneginf(x)] == 0).all()


def test_rows_apart_and_no_rows(esmoe):
    wide = _logits(19, 150, torch.bfloat16, 9).cuda()
    part = wide[:, 7:136]
    ids, w = esmoe.es_topk_gating(part, 5)
    same_ids, same_w = esmoe.es_topk_gating(part.contiguous(), 5)
    assert torch.equal(ids, same_ids) and torch.equal(w, same_w)
    g = torch.randn_like(w)
    assert torch.equal(esmoe.es_topk_gating_backward(g, part, ids, renormalize=False),
                       esmoe.es_topk_gating_backward(g, part.contiguous(), ids, renormalize=False))
    ids, w = esmoe.es_topk_gating(wide[:0], 5)
    assert ids.shape == w.shape == (0, 5)
    assert esmoe.es_topk_gating_backward(w, wide[:0], ids).shape == (0, 150)


def test_results_are_the_same_every_time(esmoe):
    x = _logits(4097, 256, torch.float32, 11).cuda()
    b = torch.zeros(256, device="cuda")
    first = esmoe.es_topk_gating(x, 8, b, "sigmoid", True, 2.5, 8, 4)
    g = esmoe.es_topk_gating_backward(first[1], x, first[0], "softmax", False)
    for _ in range(3):
        again = esmoe.es_topk_gating(x, 8, b, "sigmoid", True, 2.5, 8, 4)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
        assert torch.equal(g, esmoe.es_topk_gating_backward(first[1], x, first[0], "softmax", False))
    # a token's result does not hang on its neighbours
    alone = esmoe.es_topk_gating(x[4096:], 8, b, "sigmoid", True, 2.5, 8, 4)
    assert torch.equal(alone[0], first[0][4096:]) and torch.equal(alone[1], first[1][4096:])


def test_more_tokens_than_a_launch_takes(esmoe):
    """Over 2^24 tokens; one expert of four each, the weight an unnormalised sigmoid: values and gradients of a few known logits."""
    t = (1 << 24) + 37
    picked = torch.arange(t, device="cuda", dtype=torch.int32) * 7 % 5 % 4
    x = torch.zeros((t, 4), dtype=torch.bfloat16, device="cuda").scatter_(1, picked.long().unsqueeze(1), 2.0)
    ids, w = esmoe.es_topk_gating(x, 1, None, "sigmoid", False)
    p = torch.sigmoid(torch.tensor(2.0, dtype=torch.float64)).item()
    assert torch.equal(ids[:, 0], picked) and ((w.double() - p).abs() <= 4 * 2.0 ** -24).all()
    d = esmoe.es_topk_gating_backward(torch.ones_like(w), x, ids, "sigmoid", False)
    want = torch.tensor(p * (1 - p)).to(torch.bfloat16).item()
    assert (d.gather(1, picked.long().unsqueeze(1)).float() - want).abs().max() <= want * 2.0 ** -8
    assert torch.count_nonzero(d) == t


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups", [1, 8])
def test_a_token_is_the_same_in_any_batch(esmoe, scoring, groups):
    x = _logits(301, 256, torch.float32, 11).cuda()
    x[40] = x[41].round()   # (ties: decided in 64 bits)
    b = torch.zeros(256, device="cuda")
    ids, w = esmoe.es_topk_gating(x, 8, b, scoring, True, 2.5, groups, min(groups, 4))
    for t in (0, 1, 40, 41, 42, 43, 300):
        one = esmoe.es_topk_gating(x[t:t + 1], 8, b, scoring, True, 2.5, groups, min(groups, 4))
        assert torch.equal(one[0][0], ids[t]) and torch.equal(one[1][0], w[t])
    back = esmoe.es_topk_gating(x.flip(0), 8, b, scoring, True, 2.5, groups, min(groups, 4))
    assert torch.equal(back[0].flip(0), ids) and torch.equal(back[1].flip(0), w)


@pytest.mark.parametrize("scoring,biased", [("softmax", False), ("sigmoid", True), ("softmax", True)])
@pytest.mark.parametrize("groups,topk", [(1, 8), (8, 8), (1, 16), (4, 3)])
@pytest.mark.parametrize("experts", [64, 128, 256])
def test_close_calls(esmoe, scoring, biased, groups, topk, experts):
    """Logits a few units of the last place apart, in runs of neighbours and between groups: the order is the one of 64 bits."""
    gen = torch.Generator().manual_seed(experts + topk)
    t, inf = 4099, float("inf")
    x = torch.randint(-6, 7, (t, experts), generator=gen) / 2 + torch.randint(-3, 4, (t, experts), generator=gen) * 1.5 * 2.0 ** -22
    x[::3] = 2 * torch.randn((len(x[::3]), experts), generator=gen)
    x = x.cuda()
    b = (torch.randint(0, 2, (experts,), generator=gen) / 4 + torch.randint(0, 3, (experts,), generator=gen) * 2.0 ** -23).cuda() if biased else None
    keep = max(1, groups // 2)
    ids, _ = esmoe.es_topk_gating(x, topk, b, scoring, True, 1.0, groups, keep)
    xd = x.double()
    s = torch.softmax(xd, 1) if scoring == "softmax" else torch.sigmoid(xd)
    choice = x if groups == 1 and b is None else (s if b is None else s + b.double()).float()
    if groups > 1:
        g = choice.view(t, groups, -1)
        score = g.topk(2, dim=2).values.sum(2)
        kept = torch.sort(score, dim=1, descending=True, stable=True).indices[:, :keep]
        out = torch.ones_like(score, dtype=torch.bool).scatter_(1, kept, False)
        choice = g.masked_fill(out.unsqueeze(2), -inf).view(t, experts)
    want = torch.sort(choice, dim=1, descending=True, stable=True).indices[:, :topk]
    assert torch.equal(ids.long(), want)


def test_a_slice_as_bias_and_one_row_for_all(esmoe):
    x = _logits(9, 256, torch.float32, 3)
    b = 0.1 * torch.randn(257, generator=torch.Generator().manual_seed(4))
    _check(esmoe, x, 8, b[1:], "sigmoid", True, groups=8, topk_groups=3)
    same = x[:1].cuda().expand(6, 256)
    ids, w = esmoe.es_topk_gating(same, 8, b.cuda()[1:], "sigmoid", True, 1.0, 8, 3)
    one = esmoe.es_topk_gating(same[:1], 8, b.cuda()[1:], "sigmoid", True, 1.0, 8, 3)
    assert (ids == one[0]).all() and (w == one[1]).all()
    g = torch.ones_like(w)
    d = esmoe.es_topk_gating_backward(g, same, ids, "softmax", False)
    assert (d == d[:1]).all() and d.shape == (6, 256)
