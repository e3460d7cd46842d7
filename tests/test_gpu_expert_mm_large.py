"""Properties of the experts' products at sizes that the large kernel (expert_mm.hip) multiplies in every form used here, which each test asks the
rule for: gaps, metadata that leave the tensor or claim the same rows, NaN neighbours, repeatability, streams, graphs, SwiGLU's gradients and int8.
(test_gpu_expert_mm.py and test_gpu_int8.py have the same properties at sizes that the kernels of few rows take; a row's bytes are the same in any batch
within one kernel.)  Bounds as derived in those two files."""
import pytest
import torch

from oracle import expert_mm as O
from tests.mm_kernel_choice import FORWARD, ROWS, SWIGLU, WEIGHTS, only_large
from tests.test_gpu_expert_mm import check, check_forward, meta, operands, run_forward, sum_error
from tests.test_gpu_experts_training import Layer
from tests.test_gpu_int8 import exact as int8_exact, operands as int8_operands, run as int8_run

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16

# weight rows of two times 4096 bytes, whose sums begin at different steps; and rows that fill no step, experts of all heights
WHOLE = ([1500, 0, 1700, 33], 784, 4096)
RAGGED = ([300, 0, 517, 33, 256, 1, 700, 0, 64, 190, 257, 128], 784, 1048)
CASES = [WHOLE, RAGGED]
IDS = ["whole", "ragged"]


def same(x, y):
    return torch.equal(x.contiguous().view(torch.int16), y.contiguous().view(torch.int16))


def backward(es, a, b, d, rows, offsets, **grads):
    return es.es_grouped_mm_backward(d, a, b.transpose(1, 2), *meta(rows, offsets, b.size(1), a.size(1)), **grads)


def check_backward(es, a, b, d, rows, offsets):
    """Into given tensors: rows of no expert stay, an expert without rows gets zeros."""
    n, k = b.shape[1:]
    ga_want, ga_mag, _, gb_want, gb_mag, _ = O.grouped_mm_grads(d, a, b, rows, offsets)
    ga, gb = torch.full_like(a, 55.0), torch.full_like(b, 55.0)
    backward(es, a, b, d, rows, offsets, grad_a=ga, grad_b=gb.transpose(1, 2))
    check(ga, ga_want, sum_error(n, ga_mag), ga_want[:, 0].isnan(), 55.0)
    check(gb, gb_want, sum_error(max(rows), gb_mag))
    assert not gb[[e for e, m in enumerate(rows) if m == 0]].any()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("rows,n,k", CASES, ids=IDS)
def test_values(esmoe, rows, n, k, dtype):
    a, b, d = operands(rows, n, k, dtype, n + k)
    assert only_large(len(rows), a.size(0), n, k)
    check_forward(esmoe, a, b, rows)
    check_backward(esmoe, a, b, d, rows, O.offsets_of(rows))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("rows,n,k", CASES, ids=IDS)
def test_swiglu_gradients(esmoe, rows, n, k, dtype):
    a, b, gate_up = operands(rows, n, k, dtype, n + k + 2)
    assert only_large(len(rows), a.size(0), n, k, (ROWS, WEIGHTS))
    gen = torch.Generator(device="cuda").manual_seed(9)
    d = torch.randn((a.size(0), n // 2), generator=gen, device="cuda").to(dtype)
    gate_up *= 3
    offsets = O.offsets_of(rows)
    dgu = O.swiglu_grad(d, gate_up)
    g, u = gate_up.double().chunk(2, dim=1)
    terms = torch.cat([d.double().abs() * u.abs() * (1 + g.abs()), d.double().abs() * g.abs()], dim=1)
    dgu_err = O.out_bound(dgu, 2.0 ** -20 * terms, dtype)
    ga_want, ga_mag, ga_err, gb_want, gb_mag, gb_err = O.grouped_mm_grads(dgu, a, b, rows, offsets, dgu_err)
    ga, gb = esmoe.es_grouped_mm_swiglu_backward(d, a, b.transpose(1, 2), gate_up, *meta(rows, offsets, n, k))
    check(ga, ga_want, sum_error(n, ga_mag + ga_err) + ga_err, ga_want[:, 0].isnan(), 0.0)
    check(gb.transpose(1, 2), gb_want, sum_error(max(rows), gb_mag + gb_err) + gb_err)


@pytest.mark.parametrize("n,k", [(784, 4096), (784, 2056)])
def test_gaps_and_any_order(esmoe, n, k):
    """Experts' rows in any order with rows of nobody between them."""
    rows, offsets, total = [300, 700, 0, 1333, 5, 257], [1700, 2010, 7, 20, 1400, 2730], 3000
    gen = torch.Generator(device="cuda").manual_seed(3)
    a, d = (torch.randn((total, w), generator=gen, device="cuda").to(BF) for w in (k, n))
    b = (0.1 * torch.randn((len(rows), n, k), generator=gen, device="cuda")).to(BF)
    assert only_large(len(rows), total, n, k)
    for nobody in (slice(0, 20), slice(1353, 1400), slice(1405, 1700), slice(2000, 2010), slice(2710, 2730), slice(2987, 3000)):
        a[nobody], d[nobody] = float("nan"), float("inf")
    check_forward(esmoe, a, b, rows, offsets)
    check_backward(esmoe, a, b, d, rows, offsets)


def test_metadata_that_leave_the_tensor(esmoe):
    """Counts and offsets are cut at the tensor's rows; negative ones are none."""
    n, k, total = 784, 4096, 3000
    rows, offsets = [900, -3, 1 << 30, 9, (1 << 31) - 1, 17], [0, 0, 900, -1, total, (1 << 31) - 1]
    a, b, d = operands([total], n, k, BF, 4, spare=0)
    b = torch.cat([b * (i + 1) / 4 for i in range(len(rows))])
    assert only_large(len(rows), total, n, k)
    cut, at = [900, 0, total - 900, 0, 0, 0], [0, 0, 900, 0, 0, 0]
    want, mag = O.grouped_mm(a, b, cut, at)
    check(run_forward(esmoe, a, b, rows, offsets, False), want, sum_error(k, mag))
    ga_want, ga_mag, _, gb_want, gb_mag, _ = O.grouped_mm_grads(d, a, b, cut, at)
    ga, gb = backward(esmoe, a, b, d, rows, offsets)
    check(ga, ga_want, sum_error(n, ga_mag))
    check(gb.transpose(1, 2), gb_want, sum_error(total, gb_mag))


def test_many_claims_on_the_same_rows(esmoe):
    """64 experts of the same weights that all claim all rows: every row gets that product, every expert the whole gradient."""
    n, k, total, experts = 2064, 2056, 1100, 64
    a, b, d = operands([total], n, k, BF, 5, spare=0)
    assert only_large(experts, total, n, k)
    want, mag = O.grouped_mm(a, b, [total], [0])
    ga_want, ga_mag, _, gb_want, gb_mag, _ = O.grouped_mm_grads(d, a, b, [total], [0])
    b = b.repeat(experts, 1, 1)
    check(run_forward(esmoe, a, b, [total] * experts, [0] * experts, False), want, sum_error(k, mag))
    assert run_forward(esmoe, a, b, [total] * experts, [0] * experts, True).isfinite().all()
    ga, gb = backward(esmoe, a, b, d, [total] * experts, [0] * experts)
    check(ga, ga_want, sum_error(n, ga_mag))
    gb = gb.transpose(1, 2)
    check(gb[0], gb_want[0], sum_error(total, gb_mag[0]))
    assert all(same(g, gb[0]) for g in gb)


@pytest.mark.parametrize("rows,n,k", CASES, ids=IDS)
def test_nan_and_infinity_stay_where_they_are(esmoe, rows, n, k):
    a, b, d = operands(rows, n, k, BF, 11)
    assert only_large(len(rows), a.size(0), n, k)
    offsets, half = O.offsets_of(rows), n // 2
    base, base_h = (run_forward(esmoe, a, b, rows, offsets, swiglu) for swiglu in (False, True))
    ga0, gb0 = backward(esmoe, a, b, d, rows, offsets)
    a2, b2, d2 = a.clone(), b.clone(), d.clone()
    mine = slice(offsets[2], offsets[2] + rows[2])
    a2[5, 3], b2[2, n - 1, k - 1], d2[7, 8] = float("nan"), float("inf"), float("nan")
    a2[-1], d2[-1] = float("nan"), float("inf")   # behind the last expert's rows
    b2[1] = float("nan")                          # of an expert without rows
    out, h = (run_forward(esmoe, a2, b2, rows, offsets, swiglu) for swiglu in (False, True))
    hit = torch.zeros_like(out, dtype=torch.bool)
    hit[5], hit[mine, n - 1] = True, True
    assert not out[hit].isfinite().any() and same(out[~hit], base[~hit])
    hit = torch.zeros_like(h, dtype=torch.bool)
    hit[5], hit[mine, half - 1] = True, True
    assert not h[hit].isfinite().any() and same(h[~hit], base_h[~hit])
    ga, gb = backward(esmoe, a2, b2, d2, rows, offsets)
    hit = torch.zeros_like(ga, dtype=torch.bool)
    hit[7], hit[mine, k - 1] = True, True
    assert not ga[hit].isfinite().any() and same(ga[~hit], ga0[~hit])
    hit = torch.zeros_like(gb0, dtype=torch.bool)
    hit[0, 3, :], hit[0, :, 8] = True, True
    assert not gb[hit].isfinite().any() and same(gb[~hit], gb0[~hit])


@pytest.mark.parametrize("swiglu", [False, True])
@pytest.mark.parametrize("n,k", [(4096, 2048), (4096, 1032)])
def test_a_row_is_the_same_beside_any_others(esmoe, n, k, swiglu):
    """How many rows its expert has besides it, how they are divided into tiles and what the other experts have does not change a row's bytes."""
    a, b, _ = operands([2000, 500], n, k, BF, 12, spare=0)
    kind = SWIGLU if swiglu else FORWARD
    assert only_large(2, 2500, n, k, (kind,))
    whole = run_forward(esmoe, a, b, [2000, 500], [0, 2000], swiglu)
    for m, other in ((2000, 0), (2000, 40), (1999, 500), (1300, 257), (1025, 0), (1024, 500), (777, 333), (600, 0)):
        assert only_large(2, m + other, n, k, (kind,))
        rows = torch.cat([a[:m], a[2000:2000 + other]])
        part = run_forward(esmoe, rows, b, [m, other], [0, m], swiglu)
        assert same(part[:m], whole[:m]) and same(part[m:], whole[2000:2000 + other]), (m, other)


def test_a_rows_gradient_is_the_same_beside_any_others(esmoe):
    n, k = 1032, 4096
    _, b, d = operands([2000, 500], n, k, BF, 12, spare=0)
    zeros = lambda m: torch.zeros((m, k), dtype=BF, device="cuda")
    whole, _ = backward(esmoe, zeros(2500), b, d, [2000, 500], [0, 2000], need_grad_b=False)
    for m, other in ((2000, 0), (1999, 500), (1300, 257), (1025, 0), (777, 333), (600, 0)):
        assert only_large(2, m + other, n, k, (ROWS,))
        rows = torch.cat([d[:m], d[2000:2000 + other]])
        part, _ = backward(esmoe, zeros(m + other), b, rows, [m, other], [0, m], need_grad_b=False)
        assert same(part[:m], whole[:m]) and same(part[m:], whole[2000:2000 + other]), (m, other)


@pytest.mark.parametrize("rows,n,k", CASES, ids=IDS)
def test_same_bytes_every_time(esmoe, rows, n, k):
    a, b, d = operands(rows, n, k, BF, 13)
    assert only_large(len(rows), a.size(0), n, k)
    offsets = O.offsets_of(rows)

    def all_forms():
        return [run_forward(esmoe, a, b, rows, offsets, False), *run_forward(esmoe, a, b, rows, offsets, True, True), *backward(esmoe, a, b, d, rows, offsets)]

    first = all_forms()
    for _ in range(4):
        assert all(same(x, y) for x, y in zip(first, all_forms()))


def test_another_stream(esmoe):
    """The calls run on the current stream, in order with what that stream does before and after them."""
    rows, n, k = RAGGED
    a, b, d = operands(rows, n, k, BF, 14, spare=0)
    assert only_large(len(rows), a.size(0), n, k)
    offsets = O.offsets_of(rows)
    want = [run_forward(esmoe, a, b, rows, offsets, True), *backward(esmoe, a, b, d, rows, offsets)]
    m = meta(rows, offsets, n, k)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        late, late_d = torch.zeros_like(a), torch.zeros_like(d)
        big = torch.randn((4096, 4096), device="cuda")
        for _ in range(4):
            big = big @ big * 1e-3
        late.copy_(a)
        late_d.copy_(d)
        out = torch.empty_like(want[0])
        esmoe.es_grouped_mm_swiglu(out, late, b.transpose(1, 2), *m)
        ga, gb = esmoe.es_grouped_mm_backward(late_d, late, b.transpose(1, 2), *m)
        got = [out.clone(), ga.clone(), gb.clone()]
        for t in (late, late_d, out, ga, gb):
            t.zero_()
    s.synchronize()
    assert all(same(x, y) for x, y in zip(got, want))


def test_captured_and_replayed(esmoe):
    """A training step in a graph, replayed on new values between eager calls; metadata are read anew by every replay."""
    n, k, total, experts = 784, 1048, 2446, 12
    a, b, _ = operands([total], n, k, BF, 15, spare=0)
    b = torch.cat([b * (i + 4) / 8 for i in range(experts)])
    assert only_large(experts, total, n, k)
    ps, eo = meta([total] + [0] * (experts - 1), [0] * experts, n, k)
    d = torch.randn((total, n // 2), device="cuda").to(BF)
    h, gu = torch.zeros_like(d), torch.zeros((total, n), dtype=BF, device="cuda")
    ga, gb = torch.zeros_like(a), torch.zeros_like(b)

    def step():
        esmoe.es_grouped_mm_swiglu(h, a, b.transpose(1, 2), ps, eo, gate_up=gu)
        esmoe.es_grouped_mm_swiglu_backward(d, a, b.transpose(1, 2), gu, ps, eo, grad_a=ga, grad_b=gb.transpose(1, 2))

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    splits = [[2446] + [0] * 11, [200] * 11 + [246], [0, 1, 2000, 0, 63, 129, 0, 0, 5, 0, 0, 248], [300, 0, 517, 33, 256, 1, 700, 0, 64, 190, 257, 128]]
    for i, split in enumerate(splits):
        assert sum(split) == total
        gen = torch.Generator(device="cuda").manual_seed(i)
        a.copy_(torch.randn(a.shape, generator=gen, device="cuda"))
        ps[:, 0] = torch.tensor(split, dtype=torch.int32)
        eo.copy_(torch.tensor(O.offsets_of(split), dtype=torch.int32))
        step()
        want = [t.clone() for t in (h, gu, ga, gb)]
        for t in (h, gu, ga, gb):
            t.fill_(55.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(same(x, y) for x, y in zip(want, (h, gu, ga, gb))), i


@pytest.mark.parametrize("dtype", [BF, HF])
def test_a_training_step(esmoe, dtype):
    """The layer of test_gpu_experts_training.py and its bound, at a size whose products are all the large kernel's."""
    tokens, experts, topk, hidden, inter = 1500, 16, 2, 1024, 520
    assert only_large(experts, tokens * topk, 2 * inter, hidden, (SWIGLU, ROWS, WEIGHTS)) and only_large(experts, tokens * topk, hidden, inter, (FORWARD, ROWS, WEIGHTS))
    layer = Layer(tokens, experts, topk, hidden, inter, dtype, 7)
    got = layer.step(esmoe)
    half = torch.finfo(dtype).eps / 2
    for name, g, w in zip(("output", "tokens", "logits", "w13", "w2"), got, layer.exact()):
        assert float((g.double() - w).norm()) <= 8 * half * float(w.norm()), name


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("n,k", [(8, 136), (24, 776), (264, 8), (520, 264), (784, 520)])
def test_weights_gradient_of_many_experts(esmoe, n, k, dtype):
    """Sums of every length in steps of 64, from none on, columns and rows that end inside a tile's sixteens."""
    rows = ([0, 1, 7, 63, 64, 65, 127, 128, 129, 200] * 30)[:300 if n * k < 100000 else 60]
    a, b, d = operands(rows, n, k, dtype, n + k + 3)
    assert only_large(len(rows), a.size(0), n, k, (WEIGHTS,))
    _, _, _, want, mag, _ = O.grouped_mm_grads(d, a, b, rows, O.offsets_of(rows))
    gb = torch.full_like(b, 55.0)
    backward(esmoe, a, b, d, rows, O.offsets_of(rows), grad_b=gb.transpose(1, 2), need_grad_a=False)
    check(gb, want, sum_error(200, mag))


# ---------------------------------------------------------------------------- 8-bit integers
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("rows,n,k", [WHOLE, RAGGED[:2] + (1040,)], ids=IDS)
def test_int8_values(esmoe, rows, n, k, dtype):
    a, b, sa, sb = int8_operands(rows, n, k, n + k)
    assert only_large(len(rows), a.size(0), n, k, (FORWARD, SWIGLU))
    offsets = O.offsets_of(rows)
    want = int8_exact(a, b, sa, sb, rows, offsets)
    none = want[:, 0].isnan()
    err = 3 * 2.0 ** -24 * want.abs()
    check(int8_run(esmoe, a, b, sa, sb, rows, offsets, False, dtype), want, err, none, 55.0)
    (g, u), (eg, eu) = want.chunk(2, dim=1), err.chunk(2, dim=1)
    h = O.swiglu(g, u)
    check(int8_run(esmoe, a, b, sa, sb, rows, offsets, True, dtype), h, 1.1 * eg * (u.abs() + eu) + (g.abs() + eg) * eu + 2.0 ** -20 * h.abs(), none, 55.0)


def test_int8_scales_of_zero_infinity_and_nan(esmoe):
    rows, n, k = [1400, 1600], 784, 1040
    a, b, sa, sb = int8_operands(rows, n, k, 5)
    assert only_large(2, a.size(0), n, k, (FORWARD,))
    offsets = O.offsets_of(rows)
    base = int8_run(esmoe, a, b, sa, sb, rows, offsets, False, BF)
    sa[3], sa[5], sb[1, 7] = 0.0, float("nan"), float("inf")
    b[1, 7] = 1
    a[1400:3000, 0] = 127   # (that channel of ones: sums of 127 + 1039)
    a[1400:3000, 1:] = 1
    want = int8_run(esmoe, a, b, sa, sb, rows, offsets, False, BF)
    assert (want[3] == 0).all() and want[5].isnan().all() and want[1400:3000, 7].isinf().all()
    keep = [i for i in range(1400) if i not in (3, 5)]
    assert same(want[keep], base[keep]) and want[1400:3000, [i for i in range(n) if i != 7]].isfinite().all()


def test_int8_captured_and_replayed(esmoe):
    rows, n, k = [1100, 0, 1900], 784, 1040
    a, b, sa, sb = int8_operands(rows, n, k, 6, spare=0)
    assert only_large(3, 3000, n, k, (SWIGLU,))
    m = meta(rows, O.offsets_of(rows), n, k)
    out = torch.empty((3000, n // 2), dtype=BF, device="cuda")
    x = torch.randn((3000, k), device="cuda").to(BF)

    def step():
        esmoe.es_int8_quant(x, a, sa)
        esmoe.es_int8_scaled_grouped_mm_swiglu(out, a, b.transpose(1, 2), sa, sb, *m)

    step()
    torch.cuda.synchronize()
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
        assert same(out, want), i
