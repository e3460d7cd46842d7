"""Logits that tie or nearly do, with and without biases and groups: the ids are those of 64-bit scores rounded to fp32, ties to the lower
index.  Without a bias the scores follow the logits, except that different logits may share a score: sigmoids near 1, scores below
the normal range, logits a unit of the last place apart."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _rows(kind, t, e, gen):
    x = 2 * torch.randn((t, e), generator=gen)
    if kind == "equal":
        x = torch.randint(-2, 3, (t, 1), generator=gen).expand(t, e).float()
    elif kind == "two":          # most at one value, some above, some below: the cut falls into a run of equals
        x = (torch.randint(0, 12, (t, e), generator=gen) // 5).float()
    elif kind == "integers":
        x = x.round()
    elif kind == "saturated":    # sigmoids that round to 1 or to its neighbours
        x = 15 + 2.5 * torch.randn((t, e), generator=gen)
    elif kind == "peaked":       # one score near 1, the others over all magnitudes
        x = 25 * torch.randn((t, e), generator=gen)
    elif kind == "denormal":     # behind the largest by 75 to 115: scores from 2^-108 to below the smallest denormal
        x = -75 - 40 * torch.rand((t, e), generator=gen)
        x[:, ::32] = torch.randint(0, 2, (t, 1), generator=gen) - 1.0
    elif kind == "units":        # neighbours and next neighbours in fp32
        x = 1 + torch.randint(0, 3, (t, e), generator=gen) * 2.0 ** -23
    elif kind == "masked":
        x = x.round().masked_fill(torch.rand((t, e), generator=gen) < 0.8, float("-inf"))
    return x


def _want(x, topk, bias, scoring, groups, keep):
    t, e = x.shape
    xd = x.double()
    s = torch.sigmoid(xd) if scoring == "sigmoid" else torch.exp(xd - xd.amax(1, keepdim=True).nan_to_num(neginf=0.0))
    if scoring == "softmax":
        s = s / s.sum(1, keepdim=True)
    inf = float("-inf")
    choice = x.float() if bias is None and groups == 1 else (s if bias is None else s + bias.double()).float()
    choice = choice.masked_fill(x == inf, inf)
    if groups > 1:
        g = choice.view(t, groups, -1)
        best = g.topk(min(2, g.size(2)), dim=2).values
        score = best.masked_fill(best == inf, 0.0).sum(2).masked_fill(best[:, :, 0] == inf, inf)
        kept = torch.sort(score, dim=1, descending=True, stable=True).indices[:, :keep]
        out = torch.ones_like(score, dtype=torch.bool).scatter_(1, kept, False)
        choice = g.masked_fill(out.unsqueeze(2), inf).reshape(t, e)
    value, ids = torch.sort(choice, dim=1, descending=True, stable=True)
    return ids[:, :topk].masked_fill(value[:, :topk] == inf, -1)


@pytest.mark.parametrize("kind", ["equal", "two", "integers", "saturated", "peaked", "denormal", "units", "masked"])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("experts", [64, 128, 256, 192])
def test_ties(esmoe, experts, scoring, kind):
    gen = torch.Generator().manual_seed(experts)
    x32 = _rows(kind, 517, experts, gen)
    biases = [None, torch.zeros(experts), torch.randint(-1, 2, (experts,), generator=gen) / 8]
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        x = x32.to(dtype).cuda()
        for bias in biases:
            b = None if bias is None else bias.cuda()
            for groups, keep in ((1, 1), (4, 4), (4, 2), (8, 3)):
                for topk in (1, 5, 8, 15, 16):
                    ids, _ = esmoe.es_topk_gating(x, topk, b, scoring, True, 1.0, groups, keep)
                    # (all groups kept: no limit, but the choices are scores)
                    want = _want(x, topk, b, scoring, groups, keep)
                    bad = (ids.long() != want).any(1).nonzero().flatten().tolist()
                    assert not bad, (dtype, None if b is None else b[:4].tolist(), groups, keep, topk, len(bad), bad[0], ids[bad[0]].tolist(),
                                     want[bad[0]].tolist())
