"""The norm over many gradients and their clipping.

Squares and sums are 64-bit: the norm is the fp32 rounding of the exact one (and 2^-40 for the order of the sum); a clipped gradient is its
value times an fp32 factor (half a step off), in fp32 (another half), rounded to its type."""
import pytest
import torch

from oracle import expert_mm as O

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def make(shapes, seed=0, scale=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return [(scale * torch.randn(s, generator=gen, device="cuda")).to(t) for s, t in shapes]


def check(es, grads, max_norm, eps=1e-6):
    want, factor = O.clip(grads, max_norm, eps)
    norm = es.es_grad_norm(grads)
    assert norm.dtype == F32 and norm.dim() == 0
    if want > torch.finfo(F32).max * (1 + 2.0 ** -24):   # (no fp32 number: 1300 gradients of up to 3e38 have one of 3.2e39)
        assert norm.isinf()
    else:
        assert abs(float(norm) - want) <= (2.0 ** -24 + 2.0 ** -40) * want + 1e-45
    before = [g.clone() for g in grads]
    outputs = [torch.full_like(g, 55.0) for g in grads]
    n2 = es.es_clip_grad_norm(grads, max_norm, eps, outputs=outputs)
    assert float(n2) == float(norm)
    assert all(torch.equal(g, b) for g, b in zip(grads, before))   # inputs are left as they were
    n3 = es.es_clip_grad_norm(grads, max_norm, eps)
    assert float(n3) == float(norm)
    for g, b, o in zip(grads, before, outputs):
        assert torch.equal(g.contiguous().view(-1).view(torch.uint8), o.contiguous().view(-1).view(torch.uint8))
        exact = b.double() * factor
        if factor == 1.0:
            assert torch.equal(g, b)
        assert ((g.double() - exact).abs() <= O.out_bound(exact, 2 * 2.0 ** -24 * exact.abs() + 1e-45, g.dtype)).all()


LISTS = [[((1,), F32)], [((7,), BF), ((3, 5), HF), ((2,), F32)], [((8192,), BF), ((8193,), HF), ((8191,), F32), ((0,), BF), ((40000,), BF)],
         [((0, 4), F32), ((), F32)], [((17, 33), t) for t in (BF, HF, F32)] * 70, [((3, 500, 1001), BF), ((1001,), F32), ((2, 1000, 999), HF)]]


@pytest.mark.parametrize("shapes", LISTS, ids=range(len(LISTS)))
@pytest.mark.parametrize("max_norm", [0.5, 1e9, 0.0])
def test_norm_and_clip(esmoe, shapes, max_norm):
    check(esmoe, make(shapes), max_norm)


def test_many_elements(esmoe):
    """More chunks than workgroups, tensors that end inside them."""
    check(esmoe, make([((5, 2049, 2047), BF), ((11,), F32), ((3, 1 << 20), F32), ((9000001,), HF)]), 1.0)


def test_more_than_31_bits_of_elements(esmoe):
    g = torch.zeros((1 << 31) + 12345, dtype=BF, device="cuda")
    g[-3:], g[0] = 2.0, 2.0
    assert float(esmoe.es_grad_norm([g])) == 4.0
    assert float(esmoe.es_clip_grad_norm([g], 1.0, 0.0)) == 4.0
    assert (g[-3:] == 0.5).all() and g[0] == 0.5 and g[1 << 31] == 0


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("shift", range(1, 9))
def test_any_alignment(esmoe, dtype, shift):
    """Slices of one flat buffer: what stands around them is not read into the norm, nor written."""
    flat = torch.full((70000,), float("nan"), dtype=dtype, device="cuda")
    cuts = [(shift, 5), (100 + shift, 9001), (20000 - shift, 8 * shift), (30000 + 3 * shift, 16384 + shift)]
    gen = torch.Generator(device="cuda").manual_seed(shift)
    for at, n in cuts:
        flat[at:at + n] = torch.randn(n, generator=gen, device="cuda").to(dtype)
    nans = flat.isnan()
    check(esmoe, [flat[at:at + n] for at, n in cuts], 1.0)
    assert torch.equal(flat.isnan(), nans)


def test_transposed_and_permuted_views(esmoe):
    """Dense memory in any order, as the products' weight gradients are."""
    base = make([((4, 30, 50), BF), ((6, 7, 8), F32)], 3)
    check(esmoe, [base[0].transpose(1, 2), base[1].permute(2, 0, 1)], 0.25)


def test_large_and_small_values(esmoe):
    """Squares beyond fp32 in either direction."""
    for scale in (1e30, 1e-30, 3e38, 1e-40):
        g = make([((1000,), F32), ((300,), BF)], 4)
        g = [(x / x.abs().max().float() * scale).to(x.dtype) for x in g]
        check(esmoe, g, scale * 0.5, 0.0)


def test_norm_beyond_fp32(esmoe):
    """The norm itself is infinite in fp32; the factor is not 0."""
    g = torch.full((10000,), 1e38, device="cuda")
    assert torch.isinf(esmoe.es_grad_norm([g]))
    esmoe.es_clip_grad_norm([g], 100.0, 0.0)
    assert ((g - 1.0).abs() <= 4 * 2.0 ** -24).all()


def test_nan_and_infinity(esmoe):
    for bad, rest in ((float("nan"), float("nan")), (float("inf"), 0.0)):
        g = make([((100,), F32), ((50,), BF)], 5)
        g[0][3] = bad
        norm = esmoe.es_clip_grad_norm(g, 1.0)
        assert norm.isnan() if bad != bad else norm.isinf()
        assert g[0][3].isnan() and (g[1].isnan().all() if rest != rest else (g[1] == 0).all())
    g = make([((100,), F32)], 6)
    before = g[0].clone()
    assert float(esmoe.es_clip_grad_norm(g, float("inf"))) == float(esmoe.es_grad_norm(g)) and torch.equal(g[0], before)


def test_zero_gradients(esmoe):
    g = [torch.zeros(100, device="cuda"), torch.zeros((3, 3), dtype=BF, device="cuda")]
    assert float(esmoe.es_clip_grad_norm(g, 1.0)) == 0.0 and not g[0].any()
    e = [torch.zeros(0, device="cuda")]
    assert float(esmoe.es_clip_grad_norm(e, 1.0)) == 0.0 and float(esmoe.es_grad_norm(e)) == 0.0


@pytest.mark.parametrize("eps", [0.0, 1e-3, 25.0])
def test_eps(esmoe, eps):
    """Beside a norm of about its size."""
    check(esmoe, make([((300,), F32), ((20, 17), BF)], 11), 10.0, eps)


def test_a_given_norm(esmoe):
    """The norm over several ranks: the gradients of each are scaled by the same factor."""
    g = make([((100,), F32), ((50,), BF)], 7)
    total = (esmoe.es_grad_norm(g) ** 2 * 4).sqrt()
    want = [x.float() * (1.0 / (total + 1e-6)) for x in g]
    assert torch.equal(esmoe.es_clip_grad_norm(g, 1.0, norm=total), total)
    assert all(((x.float() - w).abs() <= O.out_bound(w.double(), 3 * 2.0 ** -24 * w.abs().double(), x.dtype)).all() for x, w in zip(g, want))


def test_a_given_norm_of_nothing(esmoe):
    total = torch.tensor(3.0, device="cuda")
    for _ in range(3):
        assert float(esmoe.es_clip_grad_norm([torch.zeros(0, device="cuda")], 1.0, norm=total)) == 3.0


def test_one_by_one_or_together(esmoe):
    """Over a hundred tensors (several launches) against the same memory as one."""
    flat = torch.randn(300 * 64, device="cuda")
    parts = list(flat.split(64))
    a, b = esmoe.es_grad_norm(parts), esmoe.es_grad_norm([flat])
    assert abs(float(a) - float(b)) <= 2.0 ** -23 * float(b)
    assert all(float(esmoe.es_grad_norm(parts)) == float(a) for _ in range(3))


def test_captured_and_replayed(esmoe):
    g = make([((64, 1000), BF), ((999,), F32)] + [((5,), F32)] * 100, 8)
    out = [torch.empty_like(x) for x in g]
    esmoe.es_clip_grad_norm(g, 1.0, outputs=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = esmoe.es_clip_grad_norm(g, 1.0, outputs=out)
    for i in range(4):
        for j, x in enumerate(g):
            x.copy_(torch.randn(x.shape, device="cuda") * (0.001 if i == 2 else i + 1))
        n = esmoe.es_clip_grad_norm(g, 1.0, outputs=out)
        want = [x.clone() for x in out]
        for x in out:
            x.fill_(55.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert float(norm) == float(n) and all(torch.equal(x, w) for x, w in zip(out, want)), i


def test_two_calls_at_once(esmoe):
    """Each call has partial sums of its own."""
    a, b = make([((3000, 1000), BF)], 9), make([((2000, 3000), F32)], 10)
    wa, wb = float(esmoe.es_grad_norm(a)), float(esmoe.es_grad_norm(b))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        with torch.cuda.stream(s):
            na = esmoe.es_grad_norm(a)
        nb = esmoe.es_grad_norm(b)
        torch.cuda.synchronize()
        assert float(na) == wa and float(nb) == wb
