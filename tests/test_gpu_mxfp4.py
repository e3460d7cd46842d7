"""Grouped products with 4-bit weights against the 64-bit oracle.

A sum of K products in fp32: 32 products per matrix instruction in whatever order and with at worst a full step of 2^-23 each, then K / 32
fused additions over four wavefronts and two more: (32 + K / 32 + 4) 2^-23 * sum |terms|, and half a step of the output type.  SwiGLU: its
slope in the gate is below 1.1 and in the up factor below |silu|; its own exponential, reciprocal and products add 2^-20 of the value."""
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


def _operands(rows, n, k, dtype, seed, spare=2, std=0.05):
    from expert_specialization_moe_amd import quant

    gen = torch.Generator().manual_seed(seed)
    b, sf = quant.quant_weight_mxfp4(std * torch.randn((len(rows), n, k), generator=gen))
    a = torch.randn((sum(rows) + spare, k), generator=gen).to(dtype)
    return a, b, sf


def _run(es, a, b, sf, rows, swiglu, offsets=None, fill=55.0):
    n = b.size(1)
    offsets = np.concatenate([[0], np.cumsum(rows)[:-1]]) if offsets is None else offsets
    ps = torch.tensor([[m, n, a.size(1)] for m in rows], dtype=torch.int32, device="cuda")
    eo = torch.tensor(np.asarray(offsets), dtype=torch.int32, device="cuda")
    out = torch.full((a.size(0), n // 2 if swiglu else n), fill, dtype=a.dtype, device="cuda")
    f = es.es_mxfp4_grouped_mm_swiglu if swiglu else es.es_mxfp4_grouped_mm
    f(out, a.cuda(), b.cuda().transpose(1, 2), sf.cuda().transpose(1, 2), ps, eo)
    torch.cuda.synchronize()
    return out


def _check(out, a, b, sf, rows, swiglu, offsets=None, fill=55.0):
    k, dtype = a.size(1), a.dtype
    offsets = np.concatenate([[0], np.cumsum(rows)[:-1]]) if offsets is None else offsets
    want, mag = O.mxfp4_mm(_np(a), b.numpy(), sf.numpy(), rows, offsets)
    err = (32 + k / 32 + 4) * 2.0 ** -23 * mag
    if swiglu:
        half = b.size(1) // 2
        g, u, eg, eu = want[:, :half], want[:, half:], err[:, :half], err[:, half:]
        want = O.swiglu(g, u)
        err = 1.1 * eg * (np.abs(u) + eu) + (np.abs(g) + eg) * eu + 2.0 ** -20 * np.abs(want)
    none = np.isnan(want)
    got = _np(out)
    assert (got[none] == fill).all()   # rows of no expert are left as they were
    bound = err + HALF_STEP[dtype] * (np.abs(want) + err) + TINY[dtype]
    # (from half a step above the type's largest number on, a value rounds to infinity)
    top = torch.finfo(dtype).max * (1 + HALF_STEP[dtype] / 2)
    with np.errstate(invalid="ignore"):
        over = np.isinf(got) & (got * want > 0) & (np.abs(want) + err >= top)
        ok = (np.abs(got - want) <= bound) | over
    assert ok[~none].all()


CASES = [([1], 32, 128), ([1], 64, 256), ([3, 0, 5], 96, 384), ([1] * 8, 256, 512), ([0, 0, 16, 0, 17, 1, 15], 64, 640), ([64, 65, 2], 32, 1024),
         ([33, 0, 48, 100], 160, 128), ([2, 1], 4096, 7168), ([1, 0, 4], 7168, 2048), ([0, 7], 128, 32768), ([200], 32, 256)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("swiglu", [False, True])
@pytest.mark.parametrize("rows,n,k", CASES)
def test_grouped_mm(esmoe, rows, n, k, swiglu, dtype):
    a, b, sf = _operands(rows, n, k, dtype, n + k)
    _check(_run(esmoe, a, b, sf, rows, swiglu), a, b, sf, rows, swiglu)


def test_sixteen_columns_and_odd_tiles(esmoe):
    for n in (16, 48, 80):
        a, b, sf = _operands([5, 18], n, 384, torch.bfloat16, n)
        _check(_run(esmoe, a, b, sf, [5, 18], False), a, b, sf, [5, 18], False)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,n,k", [([5, 18], 16, 8320), ([1], 48, 12288), ([3, 0, 33], 80, 14336), ([1] * 70, 32, 8448)])
def test_long_k(esmoe, rows, n, k, dtype):
    """Past what a workgroup's registers hold of `a`; an odd number of column tiles, more than 64 experts, scales far apart."""
    a, b, sf = _operands(rows, n, k, dtype, n + k)
    sf[:, :, 3], sf[:, :, -1] = 2, 150
    _check(_run(esmoe, a, b, sf, rows, False), a, b, sf, rows, False)
    if n % 32 == 0:
        sf[:, :, -1] = 120
        _check(_run(esmoe, a, b, sf, rows, True), a, b, sf, rows, True)
    sf[-1, n // 2, 7] = 255   # NaN: its column, in its expert's rows
    out = _run(esmoe, a, b, sf, rows, False).cpu()
    first = sum(rows) - rows[-1]
    assert out[first:sum(rows), n // 2].isnan().all() and out.isnan().sum() == rows[-1]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_every_code_exactly(esmoe, dtype):
    """Integer activations and every 4-bit code with scales 2^-1 .. 2^2: all sums are exact in fp32, the output their rounding."""
    rng = np.random.default_rng(1)
    rows, n, k = [3, 17, 0, 1], 64, 512
    a = torch.from_numpy(rng.integers(-4, 5, (sum(rows), k))).to(dtype)
    b = torch.from_numpy(rng.integers(0, 256, (4, n, k // 2), dtype=np.uint8))
    sf = torch.from_numpy(rng.integers(126, 130, (4, n, k // 32), dtype=np.uint8))
    out = _run(esmoe, a, b, sf, rows, False)
    want, _ = O.mxfp4_mm(_np(a), b.numpy(), sf.numpy(), rows, [0, 3, 20, 20])
    assert torch.equal(out.cpu(), torch.from_numpy(want).to(dtype))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_one_column_at_a_time(esmoe, dtype):
    """A single non-zero activation picks one weight: every place of K, and the row it is in, at its own scale."""
    k, n = 256, 32
    a = torch.eye(k).to(dtype)
    rng = np.random.default_rng(2)
    b = torch.from_numpy(rng.integers(0, 256, (1, n, k // 2), dtype=np.uint8))
    sf = torch.from_numpy((120 + rng.integers(0, 12, (1, n, k // 32))).astype(np.uint8))
    out = _run(esmoe, a, b, sf, [k], False)
    assert np.array_equal(_np(out), O.dequant_mxfp4(b.numpy(), sf.numpy())[0].T)


def test_scales_over_their_whole_range(esmoe):
    """Codes 0 (2^-127) to 254, and 255, which is NaN; activations that bring the products back into range."""
    codes = [0, 1, 2, 40, 100, 127, 154, 200, 253, 254]
    k, n = 128, 16
    for code in codes:
        a = torch.zeros((2, k), dtype=torch.bfloat16)
        a[0] = 2.0 ** max(min(127 - code, 100), -100)   # (32 products have to be finite before they are scaled)
        b = torch.randint(0, 256, (1, n, k // 2), dtype=torch.uint8, generator=torch.Generator().manual_seed(code))
        sf = torch.full((1, n, k // 32), code, dtype=torch.uint8)
        out = _run(esmoe, a, b, sf, [2], False)
        _check(out, a, b, sf, [2], False)
        assert (out[1] == 0).all()
    sf = torch.full((1, n, 4), 127, dtype=torch.uint8)
    sf[0, 5, 2] = 255
    a = torch.ones((1, k), dtype=torch.bfloat16)
    out = _run(esmoe, a, b, sf, [1], False)
    assert torch.isnan(out[0, 5]) and torch.isfinite(out[0, torch.arange(n) != 5]).all()


@pytest.mark.parametrize("swiglu", [False, True])
def test_half_precision_scales(esmoe, swiglu):
    """fp16 activations with scales where an e2m1 value is an fp16 number (codes 104 to 140) and beyond on either side."""
    k, n = 256, 64
    for code in (60, 90, 103, 104, 105, 112, 127, 139, 140, 141, 150):
        a = torch.full((3, k), 2.0 ** max(min(127 - code, 14), -13), dtype=torch.float16)
        a[1] *= -0.75
        b = torch.randint(0, 256, (1, n, k // 2), dtype=torch.uint8, generator=torch.Generator().manual_seed(code))
        sf = torch.full((1, n, k // 32), code, dtype=torch.uint8)
        _check(_run(esmoe, a, b, sf, [3], swiglu), a, b, sf, [3], swiglu)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,swiglu", [(48, False), (64, True)])
def test_far_scales_in_some_places(esmoe, n, swiglu, dtype):
    """Single blocks with scales far from all others, in some tiles, beside ordinary ones; the activations bring their products into range."""
    k, rows = 1152, [5, 0, 19]
    a, b, sf = _operands(rows, n, k, dtype, 11)
    far = 2.0 ** (-100 if dtype == torch.bfloat16 else -12)
    sf[0, 3, 1] = 253 if dtype == torch.bfloat16 else 145
    sf[2, n - 1, 35] = 254 if dtype == torch.bfloat16 else 141
    sf[2, n // 2, 0] = 2
    for block in (1, 35):
        a[:, 32 * block:32 * block + 32] = far * torch.sign(a[:, 32 * block:32 * block + 32])
    _check(_run(esmoe, a, b, sf, rows, swiglu), a, b, sf, rows, swiglu)


def test_a_nan_row_is_alone(esmoe):
    rows = [4, 20]
    a, b, sf = _operands(rows, 64, 256, torch.float16, 5)
    clean = _run(esmoe, a, b, sf, rows, False)
    a[2, 100], a[7, 3] = float("nan"), float("inf")
    out = _run(esmoe, a, b, sf, rows, False)
    keep = torch.ones(out.size(0), dtype=torch.bool)
    keep[[2, 7]] = False
    assert torch.isnan(out[2]).all() and not torch.isfinite(out[7]).all() and torch.equal(out[keep.cuda()], clean[keep.cuda()])


def test_many_experts_few_rows(esmoe):
    rng = np.random.default_rng(4)
    for experts in (64, 65, 200, 1024):
        rows = [0] * experts
        for e in rng.choice(experts, 9, replace=False):
            rows[e] = int(rng.integers(1, 20))
        rows[-1] = 2
        a, b, sf = _operands(rows, 32, 128, torch.bfloat16, experts)
        _check(_run(esmoe, a, b, sf, rows, True), a, b, sf, rows, True)


def test_metadata_outside_the_tensors(esmoe):
    """Negative counts, offsets outside the rows and counts that run past them reach no memory outside the tensors."""
    a, b, sf = _operands([4, 4, 4, 4], 32, 128, torch.bfloat16, 7, spare=0)
    out = _run(esmoe, a, b, sf, [-3, 4, 100, 5], False, offsets=[0, 4, 12, 16])
    _check(out, a, b, sf, [0, 4, 4, 0], False, offsets=[0, 4, 12, 0])
    out = _run(esmoe, a, b, sf, [2, 2 ** 31 - 1, 3, 1], False, offsets=[-1, 2 ** 31 - 1, 8, 2])
    _check(out, a, b, sf, [0, 0, 3, 1], False, offsets=[0, 0, 8, 2])
    out = _run(esmoe, a, b, sf, [0, 0, 0, 0], True)
    assert (out == 55.0).all()


def test_rows_do_not_hang_on_their_neighbours(esmoe):
    """The bytes of a row are the same alone, beside other rows of its expert and in another place of the list."""
    a, b, sf = _operands([40, 3], 128, 1024, torch.bfloat16, 9, spare=0)
    out = _run(esmoe, a, b, sf, [40, 3], False)
    alone = _run(esmoe, a[17:18], b[:1], sf[:1], [1], False)
    assert torch.equal(alone[0], out[17])
    swapped = _run(esmoe, torch.cat([a[40:], a[:40]]), b.flip(0), sf.flip(0), [3, 40], False)
    assert torch.equal(swapped[:3], out[40:]) and torch.equal(swapped[3:], out[:40])


def test_weights_past_32_bits(esmoe):
    """[E, N, K/2] of more than 4 GB: the last expert's."""
    e, n, k = 66, 8192, 16384
    b = torch.zeros((e, n, k // 2), dtype=torch.uint8, device="cuda")
    sf = torch.full((e, n, k // 32), 127, dtype=torch.uint8, device="cuda")
    rng = np.random.default_rng(3)
    tail = torch.from_numpy(rng.integers(0, 256, (32, k // 2), dtype=np.uint8))
    b[-1, -32:] = tail.cuda()
    a = torch.from_numpy(rng.integers(-2, 3, (2, k))).to(torch.bfloat16)
    out = torch.empty((2, n), dtype=torch.bfloat16, device="cuda")
    ps = torch.zeros((e, 3), dtype=torch.int32, device="cuda")
    ps[-1, 0] = 2
    esmoe.es_mxfp4_grouped_mm(out, a.cuda(), b.transpose(1, 2), sf.transpose(1, 2), ps, torch.zeros(e, dtype=torch.int32, device="cuda"))
    want = _np(a) @ O.dequant_mxfp4(tail.numpy(), np.full((32, k // 32), 127)).T
    assert torch.equal(out[:, -32:].cpu(), torch.from_numpy(want).to(torch.bfloat16)) and (out[:, :-32] == 0).all()


def test_c_abi(esmoe):
    from expert_specialization_moe_amd import _native

    a, b, sf = (t.cuda() for t in _operands([2, 3], 64, 256, torch.float16, 1, spare=0))
    ps = torch.tensor([[2, 64, 256], [3, 64, 256]], dtype=torch.int32, device="cuda")
    eo = torch.tensor([0, 2], dtype=torch.int32, device="cuda")
    for swiglu in (0, 1):
        out = torch.empty((5, 32 if swiglu else 64), dtype=torch.float16, device="cuda")
        rc = _native.lib.esmoe_mxfp4_grouped_mm(H.ptr(out), 1, H.ptr(a), H.ptr(b), H.ptr(sf), H.ptr(ps), H.ptr(eo), 2, 5, 64, 256, swiglu, H.stream_ptr())
        assert rc == 0, _native.last_error()
        assert torch.equal(out, _run(esmoe, a.cpu(), b.cpu(), sf.cpu(), [2, 3], bool(swiglu)))
