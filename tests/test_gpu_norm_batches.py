"""A row of the residual norm has the same bytes in any batch, alone or beside however many others."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("k", [640, 1152, 2048, 4224, 7168, 8192, 12288, 20480, 32768])
def test_a_row_is_the_same_in_any_batch(esmoe, k, dtype):
    """Over the calls that put a row to 64, 256 and 1024 threads; rows of many sizes, so that sums of squares end on every last bit."""
    gen = torch.Generator().manual_seed(k)
    rows = 700
    x = (torch.randn((rows, k), generator=gen) * torch.exp2(torch.randint(-3, 4, (rows, 1), generator=gen))).to(dtype).cuda()
    r = torch.randn((rows, k), generator=gen).to(dtype).cuda()
    w = (1 + 0.3 * torch.randn(k, generator=gen)).to(dtype).cuda()
    whole = esmoe.es_add_rms_norm_quant_1x128(x, w, 1e-6, r, return_normed=True)
    for step in (1, 255, 256, 257):
        for t in range(0, rows, step if step > 1 else 29):
            some = slice(t, t + step)
            part = esmoe.es_add_rms_norm_quant_1x128(x[some], w, 1e-6, r[some], return_normed=True)
            for a, b in zip(whole, part):
                assert torch.equal(a[some].view(torch.uint8), b.view(torch.uint8)), (step, t)


@pytest.mark.parametrize("rows", [3, 300])
def test_squares_beyond_fp32_give_zeros(esmoe, rows):
    """A sum of squares above the largest fp32 number is infinite and its reciprocal root 0; other rows do not notice."""
    x = torch.ones((rows, 2048), dtype=torch.bfloat16, device="cuda")
    x[1] = 1e19   # 2048 squares of it: 2e41
    q, scales, _, normed = esmoe.es_add_rms_norm_quant_1x128(x, torch.ones(2048, dtype=torch.bfloat16, device="cuda"), 0.0, return_normed=True)
    keep = torch.arange(rows, device="cuda") != 1
    assert (normed[1] == 0).all() and (q[1].float() == 0).all() and (normed[keep] == 1).all() and (q[keep].float() == 448).all()
    # (the least scale: 1e-4 / 448 within two roundings)
    assert ((scales[1].double() * 448 / 1e-4 - 1).abs() <= 2.0 ** -22).all()
