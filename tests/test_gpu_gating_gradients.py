"""The gradient of the routing weights against the 64-bit oracle, every element within the rounding of its own terms.

Let R = 2 (d + x + 32) 2^-24 with d the spread and x the size of the logits that take part: what an exponential of a difference, a sum
over at most 1024 such terms in 22 levels, and a quotient are off by, relative.  A renormalised weight v and a softmax score are off by R,
v_j (g_j - sum v g) by v_j (|g_j| + sum v |g|) (2 R + 2^-20), whatever the difference cancels to; 1 - s and s (1 - s) of a sigmoid are
quotients by 1 + exp, off by R again.  A place's term has that bound; places of one id add up, each addition 2^-24 of the magnitudes.  Half a step of
the output's type on top."""
import numpy as np
import pytest
import torch

from oracle import moe_block as O

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0 ** -25}
# sixteen lanes a token up to 256 experts and 16 places, a wavefront a token beyond either
SHAPES = [(2051, 256, 8), (33, 60, 6), (129, 128, 16), (65, 130, 10), (9, 16, 16), (65, 300, 8), (7, 64, 64), (129, 256, 17), (33, 1024, 64), (5, 1000, 13),
          (17, 512, 1)]


def _bounds(x, ids, g, scoring, renormalize, scale):
    """-> error bound [T, E] before the last rounding."""
    out = np.zeros(x.shape)
    for i in range(len(x)):
        real = (ids[i] >= 0) & (ids[i] < x.shape[1])
        at, gi = ids[i][real], np.abs(g[i][real] * scale)
        if not at.size:
            continue
        s = O.scores(x[i], scoring)
        row = x[i] if scoring == "softmax" and not renormalize else x[i][at]
        finite = row[np.isfinite(row)]
        spread = min(finite.max() - finite.min(), 110.0)
        size = min(np.abs(finite).max(), 110.0) if scoring == "sigmoid" else 0.0
        r = 2 * (spread + size + 32) * 2.0 ** -24
        if renormalize:
            v = O.gating_weights(x[i][None], ids[i][None], scoring, True, 1.0)[0][real]
            term = v * (gi + (v * gi).sum())
            if scoring == "sigmoid":
                term = term / (1 + np.exp(x[i][at]))
        elif scoring == "sigmoid":
            term = s[at] / (1 + np.exp(x[i][at])) * gi
        else:   # dense: a sum of gradients at each expert, and what all have in common
            total = np.zeros(x.shape[1])
            np.add.at(total, at, gi)
            out[i] = s * (total + (s[at] * gi).sum()) * (2 * r + 2.0 ** -20 + at.size * 2.0 ** -23)
            continue
        many = np.zeros(x.shape[1])
        np.add.at(many, at, term)
        out[i] = many * (3 * r + 2.0 ** -20 + at.size * 2.0 ** -24)
    return out


def _check(es, x, ids, g, scoring, renormalize, scale, sharp=True):
    d = es.es_topk_gating_backward(g.cuda(), x.cuda(), ids.cuda(), scoring, renormalize, scale)
    assert d.dtype == x.dtype and d.shape == x.shape
    xd, gd, idn = x.double().numpy(), g.double().numpy(), ids.numpy()
    want = O.gating_grad(gd, xd, idn, scoring, renormalize, scale)
    err = _bounds(xd, idn, gd, scoring, renormalize, scale)
    bound = err + HALF_STEP[x.dtype] * (np.abs(want) + err) + TINY[x.dtype]
    got = d.double().cpu().numpy()
    bad = np.abs(got - want) > bound
    assert not bad.any(), (bad.sum(), np.argwhere(bad)[0], got[bad][:3], want[bad][:3], bound[bad][:3])
    some = np.abs(want) > 16 * TINY[x.dtype]
    if sharp and some.any():   # zeros, or any other wrong value, would not pass
        assert (bound[some] < np.abs(want[some]) / 8).mean() > 0.95
    return got


@pytest.mark.parametrize("t,e,topk", SHAPES)
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [False, True])
def test_gradients(esmoe, t, e, topk, scoring, renormalize):
    gen = torch.Generator().manual_seed(t + e)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        x = (2 * torch.randn((t, e), generator=gen) + torch.randn(e, generator=gen)).to(dtype)
        ids = esmoe.es_topk_gating(x.cuda(), topk, None, scoring)[0].cpu()
        # (one renormalised weight is 1 whatever its logit: its gradient is 0)
        got = _check(esmoe, x, ids, torch.randn((t, topk), generator=gen), scoring, renormalize, 2.5)
        assert topk > 1 or not renormalize or (got == 0).all()


@pytest.mark.parametrize("t,e,topk", [(301, 40, 3), (65, 256, 16), (65, 300, 8), (65, 256, 17), (33, 1024, 64), (65, 64, 64)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [False, True])
def test_ids_that_stand_twice_and_ids_of_no_expert(esmoe, t, e, topk, scoring, renormalize):
    gen = torch.Generator().manual_seed(t + topk)
    x = 2 * torch.randn((t, e), generator=gen)
    few = torch.randint(0, e, (t, max(1, topk // 3)), generator=gen)
    ids = few.gather(1, torch.randint(0, few.size(1), (t, topk), generator=gen)).int()
    foreign = torch.rand((t, topk), generator=gen) < 0.2
    ids[foreign] = torch.tensor([-1, e, -7, 1 << 30], dtype=torch.int32)[torch.randint(0, 4, (int(foreign.sum()),), generator=gen)]
    ids[0] = -1
    g = torch.randn((t, topk), generator=gen)
    g[foreign] = float("nan")   # (not read)
    g[0] = float("nan")
    assert (torch.sort(ids, dim=1).values.diff(dim=1) == 0).any()
    got = _check(esmoe, x, ids, g, scoring, renormalize, 1.5, sharp=False)
    assert (got[0] == 0).all() and np.isfinite(got).all()


@pytest.mark.parametrize("t,e,topk", [(65, 256, 8), (65, 300, 8)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [False, True])
def test_scores_near_their_ends(esmoe, t, e, topk, scoring, renormalize):
    """Sigmoids of 1 and softmax scores of nearly 1, with gradients as small as the rest that is left; masked experts have none."""
    gen = torch.Generator().manual_seed(e)
    x = 3 * torch.randn((t, e), generator=gen)
    x[:20] += 14
    x[20:40, ::7] += 25
    x[40:] = x[40:].masked_fill(torch.rand((t - 40, e), generator=gen) < 0.9, float("-inf"))
    ids = esmoe.es_topk_gating(x.cuda(), topk, None, scoring)[0].cpu()
    got = _check(esmoe, x, ids, torch.randn((t, topk), generator=gen), scoring, renormalize, 1.0, sharp=False)
    assert (got[torch.isneginf(x).numpy()] == 0).all()
