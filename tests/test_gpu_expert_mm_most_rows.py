"""The experts' products at the largest number of rows that a call may have, 2^31 - 1: offsets beyond 2^32 elements and an expert whose rows, rounded
up to whole units, pass 31 bits.  Bounds as in test_gpu_expert_mm.py."""
import pytest
import torch

from tests.test_gpu_expert_mm import check, meta, sum_error

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
MOST, N, K, CHUNK = (1 << 31) - 1, 8, 8, 1 << 26


def test_forward_and_rows_gradient(esmoe):
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 190 << 30:
        pytest.skip("three tensors of 34 GB, and what they are compared by")
    rows, offsets = [MOST - 5, 5], [0, MOST - 5]
    gen = torch.Generator(device="cuda").manual_seed(1)
    a = torch.empty((MOST, K), dtype=BF, device="cuda")
    for part in a.split(CHUNK):
        part.normal_(generator=gen)
    b = torch.randn((2, N, K), generator=gen, device="cuda").to(BF)
    m = meta(rows, offsets, N, K)
    out = torch.full((MOST, N), 55.0, dtype=BF, device="cuda")
    esmoe.es_grouped_mm(out, a, b.transpose(1, 2), *m)

    def compare(got, given, weights, depth):   # weights [2, columns, depth]
        for first in range(0, MOST - 5, CHUNK):
            at = slice(first, min(first + CHUNK, MOST - 5))
            x, w = given[at].double(), weights[0].double()
            check(got[at], x @ w.t(), sum_error(depth, x.abs() @ w.abs().t()))
        x, w = given[-5:].double(), weights[1].double()
        check(got[-5:], x @ w.t(), sum_error(depth, x.abs() @ w.abs().t()))

    compare(out, a, b, K)
    grad_a = torch.full((MOST, K), 55.0, dtype=BF, device="cuda")
    esmoe.es_grouped_mm_backward(out, a, b.transpose(1, 2), *m, grad_a=grad_a, need_grad_b=False)
    compare(grad_a, out, b.transpose(1, 2), N)
    del a, out, grad_a
    torch.cuda.empty_cache()
