"""SwiGLU's gradient where factors are large and the result is not, and the range of the type that it is rounded to.

grad_gate = d * u * s * (1 + g * (1 - s)), grad_up = d * g * s, s = sigmoid(g).  Seen through the rows' gradient of weights that are the identity:
its sums are one term and zeros.  The exponential's argument is off by 2^-23 of itself, which is |g| * 2^-23 of s; the exponential, the reciprocal and
the products add a few roundings: (|g| + 16) * 2^-22 of the value in all where 1 + g * (1 - s) does not cancel (|g| > 4), then half a step of the type."""
import pytest
import torch

from oracle import expert_mm as O
from tests.test_gpu_expert_mm import meta

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def gradient(es, d, gate, up):
    """(grad_gate, grad_up) of [rows, 8] tensors."""
    rows = d.size(0)
    gate_up = torch.cat([gate, up], dim=1).contiguous()
    b = torch.eye(16, dtype=d.dtype, device="cuda")[None].contiguous()
    a = torch.zeros((rows, 16), dtype=d.dtype, device="cuda")
    ga, _ = es.es_grouped_mm_swiglu_backward(d, a, b.transpose(1, 2), gate_up, *meta([rows], [0], 16, 16), need_grad_b=False)
    return ga[:, :8], ga[:, 8:]


def check_gradient(got, d, gate, up):
    want = O.swiglu_grad(d, torch.cat([gate, up], dim=1))
    g = torch.cat([gate, gate], dim=1).double().abs()
    assert (g > 4).all()
    bound = O.out_bound(want, (g + 16) * 2.0 ** -22 * want.abs(), d.dtype)
    assert ((torch.cat(got, dim=1).double() - want).abs() <= bound).all()


def test_factors_whose_product_leaves_fp32(esmoe):
    """d * u beyond 3.4e38 next to a sigmoid that brings it back: bf16 holds such numbers."""
    cases = [(2.0 ** 100, 2.0 ** 40, -60.0), (2.0 ** 127, 2.0 ** 20, -40.0), (2.0 ** 70, -2.0 ** 70, -50.0), (-2.0 ** 20, 2.0 ** 127, -45.0),
             (2.0 ** 126, 2.0 ** 60, -80.0), (1.5, -2.25, 7.0), (2.0 ** -90, 2.0 ** 100, -30.0), (2.0 ** -70, 2.0 ** -50, 9.0)]
    d, up, gate = (torch.tensor(x, device="cuda").to(BF)[None].contiguous() for x in zip(*cases))
    check_gradient(gradient(esmoe, d, gate, up), d, gate, up)


def test_what_fp16_holds(esmoe):
    """The gradient of gate_up is rounded to the tensors' type in front of its products: from 65520 on it is infinite in fp16, below 2^-25 zero, and
    between, down from 2^-14, it has steps of 2^-24."""
    gate = torch.full((6, 8), 32.0, device="cuda").to(HF)   # (its sigmoid is 1 in fp32: grad_up = 32 d; grad_gate = d u)
    gate[3:] = -14.0                                        # (sigmoid 8.3e-7: grad_up = -1.16e-5 d, grad_gate = -1.08e-5 d u)
    d, up = torch.ones_like(gate), torch.ones_like(gate)
    d[0], d[1], d[2] = 2047.0, 2048.0, -4096.0
    d[3], d[4], d[5] = 2.0 ** -10, 0.5, 2.0 ** -2
    up[4:] = 3.0
    g, u = gradient(esmoe, d, gate, up)
    assert (u[0] == 65504).all() and (g[0] == 2047).all()
    assert not u[1:3].isfinite().any()
    assert (u[3] == 0).all() and (g[3] == 0).all()
    check_gradient((g[4:], u[4:]), d[4:], gate[4:], up[4:])
    assert (u[4] == round(-14 * 0.5 / (1 + 2.718281828459045 ** 14) * 2 ** 24) * 2.0 ** -24).all()


def test_grad_output_chooses_the_range(esmoe):
    """Gradients are linear in grad_output: one times 2^12 gives them times 2^12, where fp16 holds them, with the bits that it would have lost."""
    rows, n, k = [130, 0, 70], 64, 48
    gen = torch.Generator(device="cuda").manual_seed(3)
    rand = lambda *s: torch.randn(s, generator=gen, device="cuda")
    a, b, gate_up = rand(200, k).to(HF), (0.1 * rand(3, n, k)).to(HF), rand(200, n).to(HF)
    small = (rand(200, n // 2) * 2.0 ** -17).to(HF)
    offsets = O.offsets_of(rows)
    m = meta(rows, offsets, n, k)
    dgu = O.swiglu_grad(small, gate_up)
    want_a, _, _, want_b, _, _ = O.grouped_mm_grads(dgu, a, b, rows, offsets)
    scale = 2.0 ** 12
    ga, gb = esmoe.es_grouped_mm_swiglu_backward(small * scale, a, b.transpose(1, 2), gate_up, *m)
    for got, want in ((ga, want_a), (gb.transpose(1, 2), want_b)):
        got = (got.double() / scale)[~want.isnan()], want[~want.isnan()]
        # two roundings, of the gradient of gate_up and of the result, half a step each of values that agree at worst
        assert float((got[0] - got[1]).norm()) <= 2 * 2.0 ** -11 * 1.01 * float(got[1].norm())


def test_projections_that_fp16_does_not_hold(esmoe):
    """A stored infinity is a finite sum beyond 65504.  Far below zero silu and its slope are zero, and a row without a gradient has none whatever
    its projections: no NaN comes of either.  Forward and backward in one."""
    k = 16
    a = torch.ones((4, k), device="cuda").to(HF)
    w = torch.zeros((1, 32, k), device="cuda").to(HF)
    w[0, :8], w[0, 16:24] = -4400.0, 0.0625         # gate -70400, up 1
    w[0, 8:16], w[0, 24:] = 4400.0, 4400.0          # gate and up 70400
    a[2:] = 2.0 ** -8                               # gates of -275 and 275, up 2^-8 and 275: all held
    m = meta([4], [0], 32, k)
    h, gate_up = torch.empty((4, 16), dtype=HF, device="cuda"), torch.empty((4, 32), dtype=HF, device="cuda")
    esmoe.es_grouped_mm_swiglu(h, a, w.transpose(1, 2), *m, gate_up=gate_up)
    assert gate_up[:2, :8].isinf().all() and gate_up[:2, 8:16].isinf().all() and (h[:, :8] == 0).all()
    d = torch.zeros_like(h)
    d[0, :8], d[2, :8], d[3, 8:] = 1.0, 1.0, 2.0 ** -8
    ga, gb = esmoe.es_grouped_mm_swiglu_backward(d, a, w.transpose(1, 2), gate_up, *m)
    # rows 0 and 2: sigmoid(-275) and less; row 1: no gradient; row 3: grad_gate = 275 / 256, grad_up = 275 / 256, times weights of 4400
    assert (ga[:3] == 0).all()
    want = torch.full((k,), 8 * 2 * 275 / 256 * 4400, dtype=torch.float64, device="cuda")
    assert want[0] > 65520 and ga[3].isinf().all()
    gb = gb.transpose(1, 2)[0]
    assert (gb[:8] == 0).all() and (gb[16:24] == 0).all()
    one = 275 / 256 * 2.0 ** -8
    assert ((gb[8:16].double() - one).abs() <= 2 * 2.0 ** -11 * one).all() and ((gb[24:].double() - one).abs() <= 2 * 2.0 ** -11 * one).all()
