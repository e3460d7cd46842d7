"""Residual addition, root-mean-square norm and 1x128 quantisation against the 64-bit oracle.

The new residual is one rounding of one fp32 sum: exactly torch's.  y is h * rstd * weight: the fp32 sum of K squares runs over at most
K / 32 fused additions per lane and a tree of 8 and more, its square root halves that, and the root, the division and two products add
2^-24 each: (K / 64 + 12) 2^-24 of y.  A scale is the largest |y| of its block times two more roundings.  A byte stands for y within half
a step of e4m3 (2^-4 of the value, 2^-10 scales near zero) of its quotient."""
import numpy as np
import pytest
import torch

from oracle import moe_block as O
from tests import helpers as H

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.bfloat16: 1e-40, torch.float16: 2.0 ** -25}


def _np(t):
    return t.double().cpu().numpy()


def _check(q, scales, normed, h, weight, eps):
    k, dtype = h.size(1), h.dtype
    y = O.rms_norm(_np(h), _np(weight), eps)
    rel = (k / 64 + 12) * 2.0 ** -24
    want = O.block_scales(y)
    assert (np.abs(_np(scales) - want) <= (rel + 2.0 ** -22) * want).all()
    back = _np(q.view(torch.float8_e4m3fn).float()).reshape(y.shape[0], -1, 128) * _np(scales)[:, :, None]
    yb = y.reshape(back.shape)
    assert (np.abs(back - yb) <= (2.0 ** -4 + 2.0 ** -18) * np.abs(yb) + 2.0 ** -10 * 1.001 * want[:, :, None]).all()
    if normed is not None:
        assert (np.abs(_np(normed) - y) <= (HALF_STEP[dtype] + 2 * rel) * np.abs(y) + TINY[dtype]).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,k", [(1, 128), (3, 256), (1, 7168), (5, 2048), (7, 2176), (2, 4096), (9, 4224), (4, 8192), (3, 8320), (2, 16384),
                                    (2, 16512), (1, 32768), (1027, 640)])
def test_norm(esmoe, rows, k, dtype):
    gen = torch.Generator().manual_seed(rows + k)
    x = torch.randn((rows, k), generator=gen).to(dtype)
    r = (3 * torch.randn((rows, k), generator=gen)).to(dtype)
    weight = (1 + 0.2 * torch.randn(k, generator=gen)).to(dtype)
    xd, rd, wd = x.cuda(), r.cuda(), weight.cuda()
    h = (x.float() + r.float()).to(dtype)
    q, scales, residual, normed = esmoe.es_add_rms_norm_quant_1x128(xd, wd, 1e-5, rd, return_normed=True)
    assert q.dtype == torch.float8_e4m3fn and scales.shape == (rows, k // 128)
    assert torch.equal(residual.cpu().view(torch.int16), h.view(torch.int16))
    assert torch.equal(xd.cpu(), x) and torch.equal(rd.cpu(), r)
    _check(q, scales, normed, h, weight, 1e-5)
    q2, s2, none, none2 = esmoe.es_add_rms_norm_quant_1x128(residual, wd, 1e-5)   # the same without an addition
    assert none is None and none2 is None and torch.equal(q2.view(torch.uint8), q.view(torch.uint8)) and torch.equal(s2, scales)


@pytest.mark.parametrize("into", ["input", "residual"])
def test_new_residual_in_place(esmoe, into):
    gen = torch.Generator(device="cuda").manual_seed(4)
    x, r = (torch.randn((33, 1280), generator=gen, device="cuda").to(torch.bfloat16) for _ in range(2))
    w = torch.ones(1280, dtype=torch.bfloat16, device="cuda")
    want = esmoe.es_add_rms_norm_quant_1x128(x, w, 1e-6, r, return_normed=True)
    place = x if into == "input" else r
    normed = torch.empty_like(x)
    got = esmoe.es_add_rms_norm_quant_1x128(x, w, 1e-6, r, place, normed)
    assert got[2].data_ptr() == place.data_ptr() and got[3].data_ptr() == normed.data_ptr()
    for a, b in zip(got, want):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_overlaps_are_refused(esmoe):
    buf = torch.zeros(4 * 256 + 128, dtype=torch.bfloat16, device="cuda")
    x, w = buf[:1024].view(4, 256), torch.ones(256, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(RuntimeError, match="not a part"):
        esmoe.es_add_rms_norm_quant_1x128(x, w, 1e-6, x.clone(), buf[128:].view(4, 256))
    with pytest.raises(RuntimeError, match="may not overlap"):
        esmoe.es_add_rms_norm_quant_1x128(x, w, 1e-6, normed=x)
    with pytest.raises(RuntimeError, match="may not overlap"):
        esmoe.es_add_rms_norm_quant_1x128(x, w, 1e-6, quant_output=buf[:512].view(torch.uint8).view(4, 256))
    both = torch.zeros_like(x)
    with pytest.raises(RuntimeError, match="each other"):
        esmoe.es_add_rms_norm_quant_1x128(x, w, 1e-6, x.clone(), both, both)
    with pytest.raises(RuntimeError, match="each other"):
        esmoe.es_add_rms_norm_quant_1x128(x, w, 1e-6, normed=both, quant_output=both.view(-1)[:512].view(torch.uint8).view(4, 256))


def test_zero_rows_tiny_rows_and_large_ones(esmoe):
    x = torch.zeros((6, 512), dtype=torch.bfloat16)
    x[1] = 1e-30
    x[2, 7] = 1e-3
    x[3] = 3e4
    x[4, :128] = 1.0                 # blocks of zeros beside others: least scale, zero bytes
    x[5] = torch.randn(512, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16) * 1e17   # (512 squares stay below the largest fp32)
    w = torch.linspace(0.5, 1.5, 512).to(torch.bfloat16)
    q, scales, _, normed = esmoe.es_add_rms_norm_quant_1x128(x.cuda(), w.cuda(), 1e-6, return_normed=True)
    _check(q, scales, normed, x, w, 1e-6)
    assert (q[0].float() == 0).all() and (q[4, 128:].float() == 0).all()
    q, scales, _, _ = esmoe.es_add_rms_norm_quant_1x128(x[2:].cuda(), w.cuda(), 0.0)
    _check(q, scales, None, x[2:], w, 0.0)


def test_nan_shows_in_its_row_alone(esmoe):
    x = torch.randn((3, 384), generator=torch.Generator().manual_seed(2)).to(torch.float16)
    clean = esmoe.es_add_rms_norm_quant_1x128(x.cuda(), torch.ones(384, dtype=torch.float16, device="cuda"), return_normed=True)
    x[1, 200] = float("nan")
    q, scales, _, normed = esmoe.es_add_rms_norm_quant_1x128(x.cuda(), torch.ones(384, dtype=torch.float16, device="cuda"), return_normed=True)
    assert torch.isnan(normed[1]).all() and torch.isnan(scales[1]).all() and torch.isnan(q[1].float()).all()
    for a, b in ((q.view(torch.uint8), clean[0].view(torch.uint8)), (scales, clean[1]), (normed, clean[3])):
        assert torch.equal(a[0], b[0]) and torch.equal(a[2], b[2])


def test_bytes_are_the_quantisers(esmoe):
    """With values that the norm leaves exact in 16 bits (a row of +-2^j with rstd a power of two), the bytes and scales are those of
    es_fp8_quant_act_1x128."""
    gen = torch.Generator().manual_seed(3)
    x = torch.where(torch.rand((4, 1024), generator=gen) < 0.5, -4.0, 4.0)
    w = torch.exp2(torch.randint(-6, 3, (1024,), generator=gen).float())
    q, scales, _, normed = esmoe.es_add_rms_norm_quant_1x128(x.to(torch.bfloat16).cuda(), w.to(torch.bfloat16).cuda(), 0.0, return_normed=True)
    assert torch.equal(normed.float().cpu(), x / 4 * w)
    want_q, want_s = esmoe.es_fp8_quant_act_1x128(normed)
    assert torch.equal(q.view(torch.uint8), want_q.view(torch.uint8)) and torch.equal(scales, want_s)


@pytest.mark.parametrize("rows,k", [(65537, 512), (9001, 7168), (40001, 1024)])
def test_rows_beyond_the_cache_give_the_bytes_of_small_calls(esmoe, rows, k):
    gen = torch.Generator().manual_seed(3)
    x, r = (torch.randn((rows, k), generator=gen).to(torch.bfloat16).cuda() for _ in range(2))
    w = torch.randn(k, generator=gen).to(torch.bfloat16).cuda()
    assert 9 * rows * k > 2 ** 28
    for residual, normed in ((r, True), (None, False)):
        whole = esmoe.es_add_rms_norm_quant_1x128(x, w, 1e-6, residual, return_normed=normed)
        for t in (*range(0, rows - 2999, 2999), rows - 2999):   # (256 rows or fewer are summed in another order)
            part = esmoe.es_add_rms_norm_quant_1x128(x[t:t + 2999], w, 1e-6, None if residual is None else residual[t:t + 2999],
                                                     return_normed=normed)
            for a, b in zip(whole, part):
                assert (a is None) == (b is None)
                if a is not None:
                    a = a[t:t + 2999]
                    assert torch.equal(a.view(torch.uint8) if a.element_size() == 1 else a, b.view(torch.uint8) if b.element_size() == 1 else b)


def test_no_rows_and_offsets_past_32_bits(esmoe):
    w = torch.ones(8192, dtype=torch.bfloat16, device="cuda")
    assert esmoe.es_add_rms_norm_quant_1x128(torch.zeros((0, 8192), dtype=torch.bfloat16, device="cuda"), w)[0].shape == (0, 8192)
    rows = 270000   # 2.2e9 elements
    x = torch.zeros((rows, 8192), dtype=torch.bfloat16, device="cuda")
    last = torch.randn((2, 8192), generator=torch.Generator().manual_seed(6)).to(torch.bfloat16)
    x[-2:] = last.cuda()
    q, scales, _, _ = esmoe.es_add_rms_norm_quant_1x128(x, w)
    _check(q[-2:], scales[-2:], None, last, w.cpu(), 1e-6)
    assert (scales[:-2] == scales[0, 0]).all()


def test_c_abi(esmoe):
    from expert_specialization_moe_amd import _native

    x = torch.randn((5, 256), generator=torch.Generator().manual_seed(2)).to(torch.float16).cuda()
    w = torch.ones(256, dtype=torch.float16, device="cuda")
    out = [torch.empty_like(x), torch.empty_like(x), torch.empty((5, 256), dtype=torch.uint8, device="cuda"), torch.empty((5, 2), device="cuda")]
    rc = _native.lib.esmoe_add_rms_norm_quant_1x128(H.ptr(x), 1, H.ptr(x), H.ptr(w), 1e-6, 5, 256, *[H.ptr(t) for t in out], H.stream_ptr())
    assert rc == 0, _native.last_error()
    q, scales, residual, normed = esmoe.es_add_rms_norm_quant_1x128(x, w, 1e-6, x, return_normed=True)
    for a, b in zip(out, (residual, normed, q.view(torch.uint8), scales)):
        assert torch.equal(a, b)
