"""The experts' products in 16 bits and their gradients against the 64-bit oracle.

A sum of K products in fp32: 32 products per matrix instruction in whatever order and with at worst a full step of 2^-23 each, then K / 32
additions: (32 + K / 32 + 4) 2^-23 * sum |terms|, and half a step of the output type.  SwiGLU: its slope in the gate is below 1.1 and in the
up factor below |silu|; its own exponential, reciprocal and products add 2^-20 of the value.  Its gradient, from the stored projections:
2^-20 of its terms' magnitudes and half a step of the type, and that error goes through the two products behind it."""
import numpy as np
import pytest
import torch

from oracle import expert_mm as O

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def sum_error(depth, mag):
    return (32 + depth / 32 + 4) * 2.0 ** -23 * mag


def meta(rows, offsets, n, k):
    return (torch.tensor([[m, n, k] for m in rows], dtype=torch.int32, device="cuda"), torch.tensor(offsets, dtype=torch.int32, device="cuda"))


def operands(rows, n, k, dtype, seed, spare=3, std=0.1):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(s, generator=gen, device="cuda")
    return rand(sum(rows) + spare, k).to(dtype), (std * rand(len(rows), n, k)).to(dtype), rand(sum(rows) + spare, n).to(dtype)


def check(got, want, err, none=None, fill=None):
    """Every element within its bound; rows of no expert as they were."""
    if none is not None:
        assert (got[none] == fill).all()
        got, want, err = got[~none], want[~none], err[~none]
    bound = O.out_bound(want, err, got.dtype)
    bad = ~((got.double() - want).abs() <= bound)
    assert not bad.any(), (int(bad.sum()), float(((got.double() - want).abs() / bound).max()))


def run_forward(es, a, b, rows, offsets, swiglu, gate_up=False, fill=55.0):
    n, k = b.size(1), a.size(1)
    out = torch.full((a.size(0), n // 2 if swiglu else n), fill, dtype=a.dtype, device="cuda")
    gu = torch.full((a.size(0), n), fill, dtype=a.dtype, device="cuda") if gate_up else None
    if swiglu:
        es.es_grouped_mm_swiglu(out, a, b.transpose(1, 2), *meta(rows, offsets, n, k), gate_up=gu)
    else:
        es.es_grouped_mm(out, a, b.transpose(1, 2), *meta(rows, offsets, n, k))
    return (out, gu) if gate_up else out


def check_forward(es, a, b, rows, offsets=None, fill=55.0):
    offsets = O.offsets_of(rows) if offsets is None else offsets
    want, mag = O.grouped_mm(a, b, rows, offsets)
    none = want[:, 0].isnan()
    err = sum_error(a.size(1), mag)
    check(run_forward(es, a, b, rows, offsets, False), want, err, none, fill)
    if b.size(1) % 16:
        return
    out, gate_up = run_forward(es, a, b, rows, offsets, True, True)
    check(gate_up, want, err, none, fill)
    (g, u), (eg, eu) = want.chunk(2, dim=1), err.chunk(2, dim=1)
    h = O.swiglu(g, u)
    check(out, h, 1.1 * eg * (u.abs() + eu) + (g.abs() + eg) * eu + 2.0 ** -20 * h.abs(), none, fill)
    # (without the projections: the same bytes)
    assert torch.equal(run_forward(es, a, b, rows, offsets, True).view(torch.int16), out.view(torch.int16))


ROWS = [[1], [17, 0, 3], [64, 65, 63], [0, 127, 128, 129, 0, 1], [255, 256, 257], [5, 600, 0, 40], [1] * 20, [0, 0, 0]]
SIZES = [(16, 8), (48, 64), (256, 128), (272, 136), (512, 520), (720, 72), (144, 1032), (1296, 192)]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("n,k", SIZES)
@pytest.mark.parametrize("rows", ROWS, ids=str)
def test_forward(esmoe, rows, n, k, dtype):
    a, b, _ = operands(rows, n, k, dtype, n + k)
    check_forward(esmoe, a, b, rows)


def ragged(experts, most, seed):
    """Rows of many experts, a third of them without any."""
    g = np.random.default_rng(seed)
    return [int(m) if g.random() < 0.67 else 0 for m in g.integers(1, most + 1, experts)]


# Tiles for all CUs or many rows: the large kernel; long rows of whole 4096 bytes begin their sums at different steps there.
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("rows,n,k", [(ragged(600, 3, 1), 16, 72), (ragged(1024, 5, 2), 24, 16), ([4100, 0, 70], 272, 136), ([3000, 1, 0, 1300], 48, 2048),
                                      (ragged(300, 40, 3), 32, 2048), ([2, 700, 0, 513], 2320, 2048), ([1] * 40, 2048, 4096)], ids=range(7))
def test_forward_of_many_tiles(esmoe, rows, n, k, dtype):
    a, b, _ = operands(rows, n, k, dtype, n + k)
    check_forward(esmoe, a, b, rows)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("rows,n,k", [(ragged(600, 40, 4), 528, 72), ([3000, 1, 0, 1300], 520, 2048), ([4100, 0, 70], 544, 200), ([1500, 0, 1700, 33], 784, 4096)], ids=range(4))
def test_many_rows(esmoe, rows, n, k, dtype):
    """More than the kernel of few rows takes, forward and gradients, with sums that end inside a step."""
    a, b, d = operands(rows, n, k, dtype, n + k)
    check_forward(esmoe, a, b, rows)
    offsets = O.offsets_of(rows)
    for d, a, b in ((d, a, b), (a, d, b.transpose(1, 2).contiguous())):   # (and the other way round)
        n, k = b.shape[1:]
        ga_want, ga_mag, _, gb_want, gb_mag, _ = O.grouped_mm_grads(d, a, b, rows, offsets)
        ga, gb = esmoe.es_grouped_mm_backward(d, a, b.transpose(1, 2), *meta(rows, offsets, n, k))
        check(ga, ga_want, sum_error(n, ga_mag), ga_want[:, 0].isnan(), 0.0)
        check(gb.transpose(1, 2), gb_want, sum_error(max(rows), gb_mag))


# Over 256 MB of weights in rows of whole lines, which are read past the caches: few rows (one tile of rows, two; half as wide items and whole ones) and many
@pytest.mark.parametrize("rows,n,k,dtype", [([1] * 8 + [0] * 60, 2048, 1024, BF), ([2, 0, 3] * 11, 2048, 2048, HF), ([20, 31, 11] * 11, 2048, 2048, BF), ([40, 0, 77] * 11, 2048, 2048, HF),
                                            ([1] * 10 + [0] * 7, 4096, 2048, HF), ([9, 40, 0] * 6, 4096, 2048, BF)], ids=range(6))
def test_streamed_weights(esmoe, rows, n, k, dtype):
    a, b, d = operands(rows, n, k, dtype, n + k)
    offsets = O.offsets_of(rows)
    check_forward(esmoe, a, b, rows)
    ga_want, ga_mag, _, _, _, _ = O.grouped_mm_grads(d, a, b, rows, offsets)
    ga, _ = esmoe.es_grouped_mm_backward(d, a, b.transpose(1, 2), *meta(rows, offsets, n, k), need_grad_b=False)
    check(ga, ga_want, sum_error(n, ga_mag), ga_want[:, 0].isnan(), 0.0)


# 300 tiles and 357 of 256 CUs: the last round's in quarters and in halves, by columns and (SwiGLU of more than 64 rows) by rows
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("rows,n,k", [([2] * 100, 528, 72), ([2] * 119, 528, 72), ([100, 0, 66] * 50, 528, 136), ([70] * 119, 528, 64),
                                      ([30] * 100, 528, 72), ([30] * 119, 528, 72)], ids=range(6))
def test_a_last_round_in_parts(esmoe, rows, n, k, dtype):
    a, b, _ = operands(rows, n, k, dtype, n + k)
    check_forward(esmoe, a, b, rows)
    n, k = k, n
    a, b, d = operands(rows, n, k, dtype, n + k)
    offsets = O.offsets_of(rows)
    ga_want, ga_mag, _, gb_want, gb_mag, _ = O.grouped_mm_grads(d, a, b, rows, offsets)
    ga, gb = esmoe.es_grouped_mm_backward(d, a, b.transpose(1, 2), *meta(rows, offsets, n, k))
    check(ga, ga_want, sum_error(n, ga_mag), ga_want[:, 0].isnan(), 0.0)
    check(gb.transpose(1, 2), gb_want, sum_error(max(rows), gb_mag))


# ... and few of both: one row tile or two, items of 16, 32 and 64 columns, units of an expert with more rows than one
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("rows,n,k", [([16], 1000, 200), ([3, 0, 13], 264, 1032), ([1] * 9, 4096, 264), ([2] * 8, 2048, 520), ([17], 520, 264), ([33, 1, 0, 64], 4104, 136),
                                      ([97, 0, 5], 2064, 2056), ([1], 8, 8), ([0, 0, 1], 16, 16384)], ids=range(9))
def test_forward_of_few_rows(esmoe, rows, n, k, dtype):
    a, b, _ = operands(rows, n, k, dtype, n + k)
    check_forward(esmoe, a, b, rows)


@pytest.mark.parametrize("n", [8, 24, 40, 264, 1000])
def test_columns_that_fill_no_tile(esmoe, n):
    rows = [3, 130, 0, 260]
    a, b, _ = operands(rows, n, 88, BF, n)
    check_forward(esmoe, a, b, rows)


def test_long_sums(esmoe):
    rows = [2, 70]
    a, b, _ = operands(rows, 32, 28672, BF, 1)
    check_forward(esmoe, a, b, rows)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("n,k", SIZES)
@pytest.mark.parametrize("rows", ROWS, ids=str)
def test_gradients(esmoe, rows, n, k, dtype):
    a, b, d = operands(rows, n, k, dtype, n + k + 1)
    offsets = O.offsets_of(rows)
    ga_want, ga_mag, _, gb_want, gb_mag, _ = O.grouped_mm_grads(d, a, b, rows, offsets)
    none = ga_want[:, 0].isnan()
    ga = torch.full_like(a, 55.0)
    gb = torch.full_like(b, 55.0)
    got = esmoe.es_grouped_mm_backward(d, a, b.transpose(1, 2), *meta(rows, offsets, n, k), grad_a=ga, grad_b=gb.transpose(1, 2))
    assert got[0] is ga and got[1].data_ptr() == gb.data_ptr()
    check(ga, ga_want, sum_error(n, ga_mag), none, 55.0)
    check(gb, gb_want, sum_error(max(rows), gb_mag))
    assert (gb[[e for e, m in enumerate(rows) if m == 0]] == 0).all()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("rows,n,k", [([17, 0, 3], 48, 64), ([130, 1, 300], 272, 136), ([64, 5], 720, 520), ([0, 0], 16, 8)])
def test_swiglu_gradients(esmoe, rows, n, k, dtype):
    a, b, gate_up = operands(rows, n, k, dtype, n + k + 2)
    gen = torch.Generator(device="cuda").manual_seed(9)
    d = torch.randn((a.size(0), n // 2), generator=gen, device="cuda").to(dtype)
    gate_up *= 3
    offsets = O.offsets_of(rows)
    dgu = O.swiglu_grad(d, gate_up)
    g, u = gate_up.double().chunk(2, dim=1)
    terms = torch.cat([d.double().abs() * u.abs() * (1 + g.abs()), d.double().abs() * g.abs()], dim=1)
    dgu_err = 2.0 ** -20 * terms
    dgu_err = O.out_bound(dgu, dgu_err, dtype)
    ga_want, ga_mag, ga_err, gb_want, gb_mag, gb_err = O.grouped_mm_grads(dgu, a, b, rows, offsets, dgu_err)
    ga, gb = esmoe.es_grouped_mm_swiglu_backward(d, a, b.transpose(1, 2), gate_up, *meta(rows, offsets, n, k))
    none = ga_want[:, 0].isnan()
    check(ga, ga_want, sum_error(n, ga_mag + ga_err) + ga_err, none, 0.0)
    check(gb.transpose(1, 2), gb_want, sum_error(max(rows), gb_mag + gb_err) + gb_err)


def test_gradients_are_the_differences_of_the_output(esmoe):
    """<grad_a, da> + <grad_b, db> against (loss(+h) - loss(-h)) / 2h of the 64-bit forward, along random directions."""
    rows, n, k = [30, 0, 7], 64, 48
    a, b, d = operands(rows, n, k, HF, 5, spare=0)
    offsets = O.offsets_of(rows)
    d = d[:, :n // 2].contiguous()
    _, gate_up = run_forward(esmoe, a, b, rows, offsets, True, True)
    ga, gb = esmoe.es_grouped_mm_swiglu_backward(d, a, b.transpose(1, 2), gate_up, *meta(rows, offsets, n, k))
    loss = lambda x, w: float((O.swiglu(*O.grouped_mm(x, w, rows, offsets)[0].chunk(2, dim=1)) * d.double()).sum())
    gen = torch.Generator(device="cuda").manual_seed(6)
    for _ in range(4):
        da, db = (torch.randn(t.shape, generator=gen, device="cuda", dtype=torch.float64) for t in (a, b))
        h = 1e-5
        diff = (loss(a.double() + h * da, b.double() + h * db) - loss(a.double() - h * da, b.double() - h * db)) / (2 * h)
        got = float((ga.double() * da).sum() + (gb.transpose(1, 2).double() * db).sum())
        # fp16 roundings of gate_up, its gradient and the result, each half a step of independent terms: eight times that of the norm
        scale = float(((ga.double() ** 2).sum() + (gb.double() ** 2).sum()) ** 0.5)
        assert abs(got - diff) <= 8 * 3 * 2.0 ** -11 * scale


def test_one_gradient_alone(esmoe):
    rows, n, k = [30, 0, 70], 64, 48
    a, b, d = operands(rows, n, k, BF, 7)
    m = meta(rows, O.offsets_of(rows), n, k)
    both = esmoe.es_grouped_mm_backward(d, a, b.transpose(1, 2), *m)
    ga, none = esmoe.es_grouped_mm_backward(d, a, b.transpose(1, 2), *m, need_grad_b=False)
    assert none is None and torch.equal(ga, both[0])
    none, gb = esmoe.es_grouped_mm_backward(d, a, b.transpose(1, 2), *m, need_grad_a=False)
    assert none is None and torch.equal(gb, both[1])


def test_no_rows(esmoe):
    """Empty tensors: nothing to multiply, and the weights' gradient is zero."""
    n, k = 64, 48
    a, b, d = operands([0, 0], n, k, BF, 8, spare=0)
    m = meta([0, 0], [0, 0], n, k)
    out = torch.empty((0, n), dtype=BF, device="cuda")
    esmoe.es_grouped_mm(out, a, b.transpose(1, 2), *m)
    gb = torch.full_like(b, 55.0)
    esmoe.es_grouped_mm_backward(d, a, b.transpose(1, 2), *m, grad_b=gb.transpose(1, 2))
    assert (gb == 0).all()


def test_gaps_and_any_order(esmoe):
    """Experts' rows in any order with rows of nobody between them."""
    rows, offsets, n, k = [20, 5, 0, 140], [150, 180, 7, 3], 80, 72
    gen = torch.Generator(device="cuda").manual_seed(3)
    a = torch.randn((190, k), generator=gen, device="cuda").to(BF)
    b = torch.randn((4, n, k), generator=gen, device="cuda").to(BF)
    d = torch.randn((190, n), generator=gen, device="cuda").to(BF)
    a[143:150] = float("nan")   # nobody's
    check_forward(esmoe, a, b, rows, offsets)
    ga_want, ga_mag, _, gb_want, gb_mag, _ = O.grouped_mm_grads(d, a, b, rows, offsets)
    ga, gb = esmoe.es_grouped_mm_backward(d, a, b.transpose(1, 2), *meta(rows, offsets, n, k))
    check(ga, ga_want, sum_error(n, ga_mag), ga_want[:, 0].isnan(), 0.0)
    check(gb.transpose(1, 2), gb_want, sum_error(140, gb_mag))


def test_metadata_that_leave_the_tensor(esmoe):
    """Counts and offsets are cut at the tensor's rows; negative ones are none."""
    rows, offsets, n, k = [50, -3, 1 << 30, 9], [60, 0, 90, -1], 64, 64
    a, b, d = operands([100], n, k, BF, 4, spare=0)
    b = b.repeat(4, 1, 1)
    cut = [40, 0, 10, 0]
    want, mag = O.grouped_mm(a, b, rows, offsets)
    out = run_forward(esmoe, a, b, rows, offsets, False)
    mine = slice(60, 90)
    check(out[mine], want[mine], sum_error(k, mag)[mine])
    assert (out[:60] == 55.0).all()
    gb = esmoe.es_grouped_mm_backward(d, a, b.transpose(1, 2), *meta(rows, offsets, n, k), need_grad_a=False)[1].transpose(1, 2)
    _, _, _, gb_want, gb_mag, _ = O.grouped_mm_grads(d, a, b, cut, [60, 0, 90, 0])
    check(gb, gb_want, sum_error(40, gb_mag))


def test_many_claims_on_the_same_rows(esmoe):
    """1024 experts that all claim all rows: nothing outside the tensors is touched, and the call ends."""
    a, b, _ = operands([300], 16, 16, BF, 4, spare=0)
    b = b.repeat(1024, 1, 1)
    out = run_forward(esmoe, a, b, [300] * 1024, [0] * 1024, False)
    torch.cuda.synchronize()
    assert (out != 55.0).all()


def test_nan_and_infinity_stay_where_they_are(esmoe):
    rows, n, k = [140, 70, 0], 80, 72
    a, b, d = operands(rows, n, k, BF, 11)
    base = run_forward(esmoe, a, b, rows, O.offsets_of(rows), False)
    m = meta(rows, O.offsets_of(rows), n, k)
    ga0, gb0 = esmoe.es_grouped_mm_backward(d, a, b.transpose(1, 2), *m)
    a2, b2, d2 = a.clone(), b.clone(), d.clone()
    a2[5, 3], b2[1, 79, 71], d2[7, 8] = float("nan"), float("inf"), float("nan")
    a2[-1], d2[-1] = float("nan"), float("inf")   # behind the last expert's rows
    b2[2] = float("nan")                          # of an expert without rows
    out = run_forward(esmoe, a2, b2, rows, O.offsets_of(rows), False)
    hit = torch.zeros_like(out, dtype=torch.bool)
    hit[5], hit[140:210, 79] = True, True
    assert not out[hit].isfinite().any() and torch.equal(out[~hit], base[~hit])
    ga, gb = esmoe.es_grouped_mm_backward(d2, a2, b2.transpose(1, 2), *m)
    hit = torch.zeros_like(ga, dtype=torch.bool)
    hit[7], hit[140:210, 71] = True, True
    assert not ga[hit].isfinite().any() and torch.equal(ga[~hit], ga0[~hit])
    hit = torch.zeros_like(gb0, dtype=torch.bool)
    hit[0, 3, :], hit[0, :, 8] = True, True
    assert not gb[hit].isfinite().any() and torch.equal(gb[~hit], gb0[~hit])


@pytest.mark.parametrize("swiglu", [False, True])
def test_a_row_is_the_same_in_any_batch(esmoe, swiglu):
    """What stands beside a row in its expert, and which experts are beside it, does not change its bytes."""
    n, k = 320, 264
    a, b, _ = operands([700, 40], n, k, BF, 12, spare=0)
    whole = run_forward(esmoe, a, b, [700, 40], [0, 700], swiglu)
    for m in (1, 5, 64, 100, 130, 300):
        part = run_forward(esmoe, a[:m].contiguous(), b[:1].contiguous(), [m], [0], swiglu)
        assert torch.equal(part.view(torch.int16), whole[:m].view(torch.int16)), m


def test_same_bytes_every_time(esmoe):
    rows, n, k = [300, 1, 80, 513], 272, 200
    a, b, d = operands(rows, n, k, BF, 13)
    m = meta(rows, O.offsets_of(rows), n, k)
    first = esmoe.es_grouped_mm_backward(d, a, b.transpose(1, 2), *m)
    for _ in range(3):
        again = esmoe.es_grouped_mm_backward(d, a, b.transpose(1, 2), *m)
        assert all(torch.equal(x.view(torch.int16), y.view(torch.int16)) for x, y in zip(first, again))


def test_another_stream(esmoe):
    """The call runs on the current stream, in order with what that stream does before and after it."""
    rows, n, k = [500, 200], 512, 512
    a, b, _ = operands(rows, n, k, BF, 14, spare=0)
    want = run_forward(esmoe, a, b, rows, O.offsets_of(rows), True)
    m = meta(rows, O.offsets_of(rows), n, k)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        late = torch.zeros_like(a)
        big = torch.randn((4096, 4096), device="cuda")
        for _ in range(4):
            big = big @ big * 1e-3
        late.copy_(a)
        out = torch.empty_like(want)
        esmoe.es_grouped_mm_swiglu(out, late, b.transpose(1, 2), *m)
        got = out.clone()
        late.zero_()
    s.synchronize()
    assert torch.equal(got.view(torch.int16), want.view(torch.int16))


def test_captured_and_replayed(esmoe):
    """A training step in a graph, replayed on new values between eager calls; metadata are read anew by every replay."""
    rows, n, k = [100, 0, 260], 160, 136
    a, b, _ = operands(rows, n, k, BF, 15, spare=0)
    ps, eo = meta(rows, O.offsets_of(rows), n, k)
    d = torch.randn((360, n // 2), device="cuda").to(BF)
    h, gu = torch.empty_like(d), torch.empty((360, n), dtype=BF, device="cuda")
    ga, gb = torch.empty_like(a), torch.empty_like(b)

    def step():
        esmoe.es_grouped_mm_swiglu(h, a, b.transpose(1, 2), ps, eo, gate_up=gu)
        esmoe.es_grouped_mm_swiglu_backward(d, a, b.transpose(1, 2), gu, ps, eo, grad_a=ga, grad_b=gb.transpose(1, 2))

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(4):
        gen = torch.Generator(device="cuda").manual_seed(i)
        a.copy_(torch.randn(a.shape, generator=gen, device="cuda"))
        split = [360 - 30 * i, 10 * i, 20 * i]
        ps[:, 0] = torch.tensor(split, dtype=torch.int32)
        eo.copy_(torch.tensor(O.offsets_of(split), dtype=torch.int32))
        step()
        want = [t.clone() for t in (h, gu, ga, gb)]
        for t in (h, gu, ga, gb):
            t.fill_(55.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x.view(torch.int16), y.view(torch.int16)) for x, y in zip(want, (h, gu, ga, gb))), i


def test_offsets_beyond_31_bits(esmoe):
    """More than 2^31 elements of weights and of their gradient, and 2^32 bytes of rows: the last expert's and the last rows."""
    e, n, k = 5, 16384, 32768
    b = torch.zeros((e, n, k), dtype=BF, device="cuda")
    rows = [0, 0, 0, 0, 66]
    gen = torch.Generator(device="cuda").manual_seed(16)
    a = torch.zeros((66000, k), dtype=BF, device="cuda")
    a[-66:] = torch.randn((66, k), generator=gen, device="cuda")
    b[4, -40:] = 0.1 * torch.randn((40, k), generator=gen, device="cuda")
    m = meta(rows, [0, 0, 0, 0, 66000 - 66], n, k)
    out = torch.zeros((66000, n), dtype=BF, device="cuda")
    esmoe.es_grouped_mm(out, a, b.transpose(1, 2), *m)
    x, w = a[-66:].double(), b[4, -40:].double()
    check(out[-66:, -40:], x @ w.t(), sum_error(k, x.abs() @ w.abs().t()))
    assert (out[:-66] == 0).all() and (out[-66:, :-40] == 0).all()
    d = out
    d[-66:] = torch.randn((66, n), generator=gen, device="cuda").to(BF)
    ga, gb = torch.zeros_like(a), torch.empty_like(b)
    esmoe.es_grouped_mm_backward(d, a, b.transpose(1, 2), *m, grad_a=ga, grad_b=gb.transpose(1, 2))
    y = d[-66:].double()
    check(ga[-66:], y[:, -40:] @ w, sum_error(n, y[:, -40:].abs() @ w.abs()))
    check(gb[4, -300:], y[:, -300:].t() @ x, sum_error(66, y[:, -300:].abs().t() @ x.abs()))
    assert not gb[:4].any()
