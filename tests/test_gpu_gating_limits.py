"""Group limits that hang on the last bits: scores of two groups that the 64-bit definition makes equal, built so that every rounding of
an fp32 evaluation goes the other way.

With a bias of 16 a choice is a multiple of u = 2^-19 and a group's score one of 2u.  Group 0's choices lie just above half-way points
of the fp32 sum, group 1's just below, each within 2^-26 of its sigmoid, so that an fp32 sigmoid often lands on or past the half-way
point: each choice then is off by u, each sum of two by up to 4u after its own rounding, group 1 above and group 0 below the same
exact score.  A tie goes to group 0; an evaluation that trusts fp32 beyond 6u sees group 1 in front by up to 8u."""
import numpy as np
import pytest
import torch

from oracle import moe_block as O

pytestmark = pytest.mark.gpu

BIAS, UNIT = 16.0, 2.0 ** -19


def _beside(m, above):
    """The fp32 logit whose sigmoid lies next to m * 2^-20, above or below it."""
    p = m * 2.0 ** -20
    x = np.log(p / (1 - p)).astype(np.float32)
    s = lambda v: 1 / (1 + np.exp(-v.astype(np.float64)))
    for _ in range(4):
        x = np.where(above & (s(x) <= p), np.nextafter(x, np.float32(9)), np.where(~above & (s(x) >= p), np.nextafter(x, np.float32(-9)), x))
    assert ((s(x) > p) == above).all() and (np.abs(s(x) - p) < 2.0 ** -25).all()
    return x


def _tokens(t, seed):
    """-> logits [t, 4]: two experts of group 0, two of group 1.  f counts units above the bias; a half-way point is f + 1/2."""
    rng = np.random.default_rng(seed)
    odd = lambda: 2 * rng.integers(151000, 185000, t) + 1      # sigmoids of .576 to .706
    even = lambda: 2 * rng.integers(151000, 185000, t)
    high_odd, high_even = odd(), even()                        # (a tie to even goes up from an odd f, down from an even one)
    high_even += np.where((high_odd + high_even) % 4 == 1, 0, 2)
    low_even = even()
    low_odd = high_odd + high_even - 2 - (low_even + 1) - 1    # exact: f + 1 of either, two units below group 1's sum before its rounding
    f = np.stack([low_even, low_odd, high_odd, high_even], axis=1)
    keep = (low_odd > 300000) & (low_odd < 371000)
    f = f[keep]
    assert (f[:, 1] % 2 == 1).all() and keep.sum() > t // 2
    return _beside(2 * f + 1, np.array([True, True, False, False])[None, :] | np.zeros_like(f, bool))


@pytest.mark.parametrize("experts,groups", [(64, 8), (128, 8), (256, 8), (256, 32)])
def test_equal_scores_of_two_groups(esmoe, experts, groups):
    four = _tokens(6000, experts)
    width = experts // groups
    x = np.zeros((len(four), experts), np.float32)
    bias = np.zeros(experts, np.float32)
    at = [1, width - 1, width, 2 * width - 2]
    x[:, at], bias[at] = four, BIAS
    ids, w = esmoe.es_topk_gating(torch.from_numpy(x).cuda(), 2, torch.from_numpy(bias).cuda(), "sigmoid", True, 1.0, groups, 1)
    want, want_w = O.topk_gating(x, 2, bias, "sigmoid", True, 1.0, groups, 1)
    assert (want < width).all()   # all of them ties, and group 0's
    wrong = (ids.cpu().numpy() != want).any(axis=1)
    assert not wrong.any(), f"{wrong.sum()} of {len(x)}"
