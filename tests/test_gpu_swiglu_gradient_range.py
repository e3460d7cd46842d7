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
