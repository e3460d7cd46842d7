"""Calls of more rows or tokens than one launch's grid takes: what lies behind the first launch is right, and at its place."""
import numpy as np
import pytest
import torch

from oracle import moe_block as O

pytestmark = pytest.mark.gpu


def test_combine(esmoe):
    """Over 2^24 tokens of one piece (512 columns) each.  A token has one local pair: its product in fp32, rounded once more."""
    tokens, topk, rows = (1 << 24) + 5, 2, 1021
    gen = torch.Generator(device="cuda").manual_seed(1)
    y = torch.randn((rows, 8), generator=gen, device="cuda").to(torch.bfloat16)
    w = torch.randn((tokens, topk), generator=gen, device="cuda")
    at = torch.arange(tokens, device="cuda") * 7919 % rows
    which = torch.arange(tokens, device="cuda") % 3 % 2
    dst = torch.full((tokens, topk), -1, dtype=torch.int32, device="cuda").scatter_(1, which.unsqueeze(1), at.int().unsqueeze(1))
    out = esmoe.es_combine_rows(y, dst.view(-1), topk, w)
    want = (y[at].float() * w.gather(1, which.unsqueeze(1))).to(torch.bfloat16)
    assert torch.equal(out, want)


def test_combine_gradient(esmoe):
    """Over 2^25 pairs; the second of every token's two is another GPU's."""
    tokens, topk = (1 << 24) + 3, 2
    gen = torch.Generator(device="cuda").manual_seed(2)
    y, g = (torch.randn((tokens, 8), generator=gen, device="cuda").to(torch.float16) for _ in range(2))
    w = torch.randn((tokens, topk), generator=gen, device="cuda")
    dst = torch.full((tokens, topk), -1, dtype=torch.int32, device="cuda")
    dst[:, 0] = torch.arange(tokens - 1, -1, -1, device="cuda")
    into = torch.full_like(y, 9.0)
    grad_rows, grad_w = esmoe.es_combine_rows_backward(g, y, dst.view(-1), topk, w, into)
    # A product of fp16 and fp32 is exact in float64 (11 + 24 bits).  The kernel may round it to fp16 at once (the machine has such an
    # instruction) or to fp32 before: at most 2^-11 + 2^-24 + 2^-35 of it, below the normal range half of 2^-24 and 2^-24 of the product.
    exact = g.double() * w[:, :1].double()
    assert ((grad_rows.flip(0).double() - exact).abs() <= (2.0 ** -11 + 1.001 * 2.0 ** -24) * exact.abs() + 2.0 ** -25).all()
    terms = g.double() * y.flip(0).double()
    # eight products in a chain and a tree of 6 over lanes that hold nothing
    assert ((grad_w[:, 0].double() - terms.sum(1)).abs() <= 14 * 2.0 ** -24 * terms.abs().sum(1) + 1e-44).all()
    assert (grad_w[:, 1] == 0).all()


@pytest.mark.parametrize("k", [128, 1152])
def test_norm(esmoe, k):
    """Over 2^22 rows, a few thousand different ones over and over."""
    rows, period = (1 << 22) + 5, 4099
    gen = torch.Generator(device="cuda").manual_seed(k)
    base = torch.randn((period, k), generator=gen, device="cuda").to(torch.bfloat16)
    w = (1 + 0.2 * torch.randn(k, generator=gen, device="cuda")).to(torch.bfloat16)
    which = torch.arange(rows, device="cuda") % period
    q, scales, _, normed = esmoe.es_add_rms_norm_quant_1x128(base[which], w, 1e-6, return_normed=True)
    want = esmoe.es_add_rms_norm_quant_1x128(base, w, 1e-6, return_normed=True)
    for t in range(0, rows, 1 << 20):
        some = which[t:t + (1 << 20)]
        for a, b in ((q.view(torch.uint8), want[0].view(torch.uint8)), (scales, want[1]), (normed, want[3])):
            assert torch.equal(a[t:t + (1 << 20)], b[some])


def test_long_k_products(esmoe):
    """Over 128 units (of sixteen rows) of 2^20 weight rows with K beyond 8192: exact sums in a few columns, zeros in the others."""
    rows, n, k = 2048 + 17, 1 << 20, 8320
    rng = np.random.default_rng(5)
    b = torch.zeros((1, n, k // 2), dtype=torch.uint8, device="cuda")
    sf = torch.full((1, n, k // 32), 124, dtype=torch.uint8, device="cuda")
    at = torch.tensor([0, 1, 15, 16, 31, 32, n // 2 + 7, n - 33, n - 32, n - 17, n - 16, n - 1], device="cuda")
    codes = rng.integers(0, 256, (len(at), k // 2), dtype=np.uint8)
    b[0, at] = torch.from_numpy(codes).cuda()
    a = torch.from_numpy(rng.integers(-1, 2, (rows + 2, k))).to(torch.bfloat16).cuda()
    out = torch.full((rows + 2, n), 7.0, dtype=torch.bfloat16, device="cuda")
    ps, eo = torch.tensor([[rows, n, k]], dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    esmoe.es_mxfp4_grouped_mm(out, a, b.transpose(1, 2), sf.transpose(1, 2), ps, eo)
    w = torch.from_numpy(O.dequant_mxfp4(codes, np.full((len(at), k // 32), 124))).cuda()
    want = torch.matmul(a[:rows].double(), w.t().contiguous()).to(torch.bfloat16)
    assert torch.equal(out[:rows, at], want) and (out[rows:] == 7.0).all()
    assert sum(int(torch.count_nonzero(out[t:t + 256])) for t in range(0, rows - 17, 256)) + int(torch.count_nonzero(out[rows - 17:rows])) == int(
        torch.count_nonzero(want))
