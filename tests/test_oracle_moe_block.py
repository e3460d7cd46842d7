"""The 64-bit oracle of the operators around the grouped GEMMs: its gradients against differences of its own forward, its codes against
the weight quantiser of the package."""
import numpy as np
import pytest
import torch

from oracle import moe_block as O


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [False, True])
def test_gating_gradient_against_differences(scoring, renormalize):
    """Central differences of step h have an error of order h^2 (third derivatives here are below 10): 1e-8 at h = 1e-5, and the
    rounding of the forward, 1e-16 / h = 1e-11."""
    rng = np.random.default_rng(3)
    x = rng.normal(size=(4, 9)) * 2
    x[1, 3] = -np.inf
    ids = np.array([[0, 5, 2], [7, 1, -1], [4, 4, 8], [-1, -1, -1]], np.int32)   # a place without an expert, one id twice, none at all
    g = rng.normal(size=ids.shape)
    loss = lambda v: (g * O.gating_weights(v, ids, scoring, renormalize, 2.5)).sum()
    got = O.gating_grad(g, x, ids, scoring, renormalize, 2.5)
    h = 1e-5
    for i in range(x.shape[0]):
        for e in range(x.shape[1]):
            if np.isinf(x[i, e]):
                assert got[i, e] == 0
                continue
            up, down = x.copy(), x.copy()
            up[i, e] += h
            down[i, e] -= h
            assert abs((loss(up) - loss(down)) / (2 * h) - got[i, e]) < 1e-7


def test_gating_order():
    x = np.array([[1.0, 3.0, 3.0, np.nan, -np.inf, 2.0], [-np.inf] * 6, [-0.0, 0.0, -np.inf, -np.inf, -np.inf, -1.0]])
    ids, w = O.topk_gating(x, 4)
    assert ids.tolist() == [[3, 1, 2, 5], [-1] * 4, [0, 1, 5, -1]]
    assert np.isnan(w[0]).all() and (w[1] == 0).all() and w[2, 3] == 0 and abs(w[2].sum() - 1) < 1e-12
    # groups of two: sums 0.3 + 0.1, 0.35 + 0, 0.2 + 0.05 -> the first and the second stay
    p = np.log(np.array([[0.3, 0.1, 0.35, 1e-9, 0.2, 0.05]]))
    assert O.topk_gating(p, 3, groups=3, topk_groups=2)[0].tolist() == [[2, 0, 1]]


def test_combine_gradients_against_differences():
    """The combine is linear in either factor: differences of any step are exact up to rounding."""
    rng = np.random.default_rng(5)
    rows, dst, w, g = rng.normal(size=(5, 8)), np.array([0, 3, -1, 2, 9, 1]), rng.normal(size=(3, 2)), rng.normal(size=(3, 8))
    grad_rows, grad_w, _ = O.combine_grad(g, rows, dst, 2, w)
    loss = lambda r, v: (g * O.combine(r, dst, 2, v)[0]).sum()
    for r in range(5):
        for c in range(8):
            up = rows.copy()
            up[r, c] += 1.0
            want = loss(up, w) - loss(rows, w)
            assert abs(want - (0.0 if np.isnan(grad_rows[r, c]) else grad_rows[r, c])) < 1e-12
    for t in range(3):
        for j in range(2):
            up = w.copy()
            up[t, j] += 1.0
            assert abs(loss(rows, up) - loss(rows, w) - grad_w[t, j]) < 1e-12
    assert np.isnan(grad_rows[4]).all()   # (row 4 has no pair; dst 9 is no row)


def test_weight_quantiser_rounds_to_the_nearest_code():
    from expert_specialization_moe_amd import quant

    gen = torch.Generator().manual_seed(1)
    w = torch.randn((3, 16, 96), generator=gen) * torch.exp(4 * torch.randn((3, 16, 1), generator=gen))
    b, sf = quant.quant_weight_mxfp4(w)
    assert b.shape == (3, 16, 48) and sf.shape == (3, 16, 3) and b.dtype == sf.dtype == torch.uint8
    x = w.double().numpy().reshape(3, 16, 3, 32)
    amax = np.abs(x).max(axis=3)
    scale = np.ldexp(1.0, sf.numpy().astype(np.int64) - 127)
    assert (amax <= 6 * scale).all() and (amax > 3 * scale).all()   # the smallest power of two that holds the block
    back = O.dequant_mxfp4(b.numpy(), sf.numpy()).reshape(x.shape)
    grid = np.abs(x[..., None] / scale[..., None, None] - O.E2M1)
    assert np.allclose(np.abs(x - back) / scale[..., None], grid.min(axis=-1), rtol=0, atol=0)


def test_weight_quantiser_ties_zeros_and_extremes():
    from expert_specialization_moe_amd import quant

    ties = torch.zeros(1, 32)
    ties[0, :9] = torch.tensor([6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.75])
    b, sf = quant.quant_weight_mxfp4(ties)
    assert sf.item() == 127
    assert O.dequant_mxfp4(b.numpy(), sf.numpy())[0, :9].tolist() == [6.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, -1.0]
    for value, code in ((6.0 * 2.0 ** 10, 137), (6.1 * 2.0 ** 10, 138), (2.0 ** -149, 0), (3e38, 253)):
        b, sf = quant.quant_weight_mxfp4(torch.full((1, 32), value))
        assert sf.item() == code, value
    zero = quant.quant_weight_mxfp4(torch.zeros(2, 64, dtype=torch.bfloat16))
    assert (O.dequant_mxfp4(zero[0].numpy(), zero[1].numpy()) == 0).all()
    bad = torch.ones(1, 64)
    bad[0, 3] = float("inf")
    assert quant.quant_weight_mxfp4(bad)[1][0].tolist()[0] == 255
