"""Grouped products in 8-bit integers and their quantiser.

The product's sum is exact in int32; then the conversion to fp32 and two products, half a step of 2^-24 each (three in all, and the sum of the
two SwiGLU factors' errors as in the 16-bit form), and half a step of the output type."""
import numpy as np
import pytest
import torch

from oracle import expert_mm as O
from tests.test_gpu_expert_mm import check, meta

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def operands(rows, n, k, seed, spare=3):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    total = sum(rows) + spare
    a = torch.randint(-128, 128, (total, k), generator=gen, device="cuda", dtype=torch.int8)
    b = torch.randint(-128, 128, (len(rows), n, k), generator=gen, device="cuda", dtype=torch.int8)
    sa = torch.rand((total,), generator=gen, device="cuda") * 0.02 + 1e-4
    sb = torch.rand((len(rows), n), generator=gen, device="cuda") * 0.003 / k ** 0.5 + 1e-6
    return a, b, sa, sb


def exact(a, b, sa, sb, rows, offsets):
    want, _ = O.grouped_mm(a, b, rows, offsets)
    scale = torch.full_like(want, float("nan"))
    for e, off, m in O.spans(rows, offsets, a.size(0)):
        scale[off:off + m] = torch.outer(sa[off:off + m].double(), sb[e].double())
    return want * scale


def run(es, a, b, sa, sb, rows, offsets, swiglu, dtype, fill=55.0):
    n, k = b.size(1), a.size(1)
    out = torch.full((a.size(0), n // 2 if swiglu else n), fill, dtype=dtype, device="cuda")
    f = es.es_int8_scaled_grouped_mm_swiglu if swiglu else es.es_int8_scaled_grouped_mm
    f(out, a, b.transpose(1, 2), sa, sb, *meta(rows, offsets, n, k))
    return out


ROWS = [[1], [17, 0, 3], [64, 65, 63], [0, 127, 128, 129, 0, 1], [255, 256, 257], [5, 600, 0, 40], [1] * 20, [0, 0, 0]]
SIZES = [(16, 16), (48, 64), (256, 128), (272, 144), (720, 1040), (1296, 192)]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("n,k", SIZES)
@pytest.mark.parametrize("rows", ROWS, ids=str)
def test_grouped_mm(esmoe, rows, n, k, dtype):
    a, b, sa, sb = operands(rows, n, k, n + k)
    offsets = O.offsets_of(rows)
    want = exact(a, b, sa, sb, rows, offsets)
    none = want[:, 0].isnan()
    err = 3 * 2.0 ** -24 * want.abs()
    check(run(esmoe, a, b, sa, sb, rows, offsets, False, dtype), want, err, none, 55.0)
    (g, u), (eg, eu) = want.chunk(2, dim=1), err.chunk(2, dim=1)
    h = O.swiglu(g, u)
    check(run(esmoe, a, b, sa, sb, rows, offsets, True, dtype), h, 1.1 * eg * (u.abs() + eu) + (g.abs() + eg) * eu + 2.0 ** -20 * h.abs(), none, 55.0)


@pytest.mark.parametrize("swiglu", [False, True])
@pytest.mark.parametrize("rows,n,k", [([4100, 0, 70], 272, 144), ([1, 0] * 300, 16, 48), ([2, 700, 0, 513], 2320, 4096), ([16], 1000, 208), ([2] * 8, 2048, 528),
                                      ([33, 1, 0, 64], 4112, 144), ([97, 0, 5], 2064, 4112), ([3000, 1, 0, 1300], 544, 4096), ([30, 0, 21] * 80, 528, 208),
                                      ([1] * 9 + [0] * 60, 4096, 1024), ([2, 0, 3] * 11, 4096, 2048), ([30, 0, 77] * 11, 4096, 2048)], ids=range(12))
def test_many_tiles_and_few_rows(esmoe, rows, n, k, swiglu):
    """Each kernel and each of its shapes; sums are exact: the same bytes from all.  The scales' products are two roundings."""
    a, b, sa, sb = operands(rows, n, k, n + k)
    offsets = O.offsets_of(rows)
    if swiglu and n % 16:
        with pytest.raises(RuntimeError):
            run(esmoe, a, b, sa, sb, rows, offsets, swiglu, BF)
        return
    got = run(esmoe, a, b, sa, sb, rows, offsets, swiglu, BF)
    want = exact(a, b, sa, sb, rows, offsets)
    none = want[:, 0].isnan()
    err = 3 * 2.0 ** -24 * want.abs()
    if swiglu:
        (g, u), (eg, eu) = want.chunk(2, dim=1), err.chunk(2, dim=1)
        want = O.swiglu(g, u)
        err = 1.1 * eg * (u.abs() + eu) + (g.abs() + eg) * eu + 2.0 ** -20 * want.abs()
    check(got, want, err, none, 55.0)


def test_largest_sums(esmoe):
    """All values at their ends and the longest K: sums of 2^30, each exact."""
    k = 65536
    a = torch.full((3, k), -128, dtype=torch.int8, device="cuda")
    b = torch.full((1, 16, k), -128, dtype=torch.int8, device="cuda")
    b[0, 1], b[0, 2, ::2], b[0, 3, -1] = 127, 127, -127
    sa, sb = torch.ones(3, device="cuda"), torch.full((1, 16), 2.0 ** -16, device="cuda")
    out = run(esmoe, a, b, sa, sb, [3], [0], False, BF)
    want = (a.double() @ b[0].double().t() * 2.0 ** -16).to(BF)
    assert torch.equal(out, want)


def test_scales_of_zero_infinity_and_nan(esmoe):
    rows, n, k = [40, 30], 48, 64
    a, b, sa, sb = operands(rows, n, k, 5)
    sa[3], sa[5], sb[1, 7] = 0.0, float("nan"), float("inf")
    b[1, 7] = 1
    out = run(esmoe, a, b, sa, sb, rows, [0, 40], False, BF)
    assert (out[3] == 0).all() and out[5].isnan().all() and not out[40:70, 7].isfinite().any()
    assert out.isfinite().sum() == 73 * n - n - 30


def test_other_streams_and_graphs(esmoe):
    rows, n, k = [100, 0, 260], 160, 144
    a, b, sa, sb = operands(rows, n, k, 6, spare=0)
    m = meta(rows, O.offsets_of(rows), n, k)
    out = torch.empty((360, n // 2), dtype=BF, device="cuda")
    x = torch.randn((360, k), device="cuda").to(BF)

    def step():
        esmoe.es_int8_quant(x, a, sa)
        esmoe.es_int8_scaled_grouped_mm_swiglu(out, a, b.transpose(1, 2), sa, sb, *m)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(4):
        x.copy_(torch.randn(x.shape, device="cuda") * (i + 1))
        step()
        want = out.clone()
        out.fill_(55.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.view(torch.int16), want.view(torch.int16)), i


# ---------------------------------------------------------------------------- the quantiser
def check_quant(es, x):
    q, scales = es.es_int8_quant(x)
    want, s = O.int8_quant(x)
    assert q.dtype == torch.int8 and q.shape == x.shape and scales.shape == x.shape[:-1]
    assert torch.equal(q, want)
    # (one division, correctly rounded)
    assert torch.equal(scales, s.float()) or torch.equal(scales.nan_to_num(-1), s.float().nan_to_num(-1))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("rows,k", [(1, 16), (3, 32), (5, 528), (2, 1024), (7, 2064), (3, 4096), (300, 7168), (2, 16400), (1, 65536), (1000, 160), (0, 64)])
def test_quant(esmoe, rows, k, dtype):
    gen = torch.Generator(device="cuda").manual_seed(rows + k)
    check_quant(esmoe, (torch.randn((rows, k), generator=gen, device="cuda") * torch.exp(2 * torch.randn((rows, 1), generator=gen, device="cuda"))).to(dtype))


@pytest.mark.parametrize("dtype", [BF, HF])
def test_quant_of_every_value(esmoe, dtype):
    """Every finite pattern of the type against maxima of every mantissa: all ties and all their neighbours."""
    bits = torch.arange(0, 1 << 16, device="cuda", dtype=torch.int32).to(torch.int16).view(dtype)
    bits = bits[bits.isfinite()]
    bits = bits[: bits.numel() // 16 * 16]
    mantissas = 128 if dtype == BF else 1024
    tops = (1 + torch.arange(mantissas, device="cuda") / mantissas).to(dtype)
    for scale in (2.0, 2.0 ** -6, 2.0 ** 9):
        for top in (tops * scale).split(64):
            x = bits.repeat(top.numel(), 1)
            x = torch.where(x.abs() > top[:, None], torch.zeros_like(x), x)
            x[:, -1] = top
            if x.size(1) > 65536:
                x = x[:, -65536:]
            check_quant(esmoe, x.contiguous())


@pytest.mark.parametrize("dtype", [BF, HF])
def test_quant_of_rows_out_of_the_ordinary(esmoe, dtype):
    x = torch.randn((8, 272), device="cuda").to(dtype)
    tiny = torch.finfo(dtype).smallest_normal
    x[0] = 0
    x[1, 5] = float("inf")
    x[2, 7] = float("nan")
    x[3] = torch.randint(-9, 10, (272,), device="cuda").to(dtype) * torch.tensor(tiny / 64, device="cuda").to(dtype)   # subnormal
    x[4] *= torch.finfo(dtype).max / 8
    x[5] = -0.0
    x[6, 0] = torch.finfo(dtype).max
    check_quant(esmoe, x)
    q, scales = esmoe.es_int8_quant(x)
    assert scales[0] == 0 and scales[5] == 0 and scales[1:3].isnan().all() and not q[:3].any()


def test_quant_of_weights_and_into_given_tensors(esmoe):
    w = torch.randn((3, 40, 80), device="cuda").to(BF)
    check_quant(esmoe, w)
    q, s = torch.empty((3, 40, 80), dtype=torch.int8, device="cuda"), torch.empty((3, 40), device="cuda")
    got = esmoe.es_int8_quant(w, q, s)
    assert got[0] is q and got[1] is s and torch.equal(q, esmoe.es_int8_quant(w)[0])


def test_an_mlp_in_int8(esmoe):
    """Quantise, gate_up with SwiGLU, quantise, down: against the 64-bit products of the unquantised operands, within the quantisers' steps."""
    rows, hidden, inter = [33, 0, 140, 2], 256, 160
    gen = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn((175, hidden), generator=gen, device="cuda").to(BF)
    w13 = (0.06 * torch.randn((4, 2 * inter, hidden), generator=gen, device="cuda")).to(BF)
    w2 = (0.08 * torch.randn((4, hidden, inter), generator=gen, device="cuda")).to(BF)
    offsets = O.offsets_of(rows)
    (q13, s13), (q2, s2) = esmoe.es_int8_quant(w13), esmoe.es_int8_quant(w2)
    qx, sx = esmoe.es_int8_quant(x)
    h = run(esmoe, qx, q13, sx, s13, rows, offsets, True, BF)
    qh, sh = esmoe.es_int8_quant(h)
    y = run(esmoe, qh, q2, sh, s2, rows, offsets, False, BF)
    # every step against its own inputs: the chain is what a program runs
    check(y, exact(qh, q2, sh, s2, rows, offsets), 3 * 2.0 ** -24 * exact(qh, q2, sh, s2, rows, offsets).abs())
    want = O.grouped_mm(O.swiglu(*O.grouped_mm(x, w13, rows, offsets)[0].chunk(2, dim=1)), w2, rows, offsets)[0]
    assert float((y.double() - want).norm() / want.norm()) < 0.05
