"""Several experts that claim the same rows: the grouped products with 4-bit weights touch no memory outside these and end."""
import numpy as np
import pytest
import torch

from oracle import moe_block as O

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("k", [256, 8320])
@pytest.mark.parametrize("experts,total", [(3, 20), (70, 37), (2, 5)])
def test_experts_that_claim_all_rows(esmoe, experts, total, k):
    """All experts hold the same weights, so it does not matter whose product a row gets; sums of integers are exact."""
    rng = np.random.default_rng(experts)
    n, spare = 48, 3
    a = torch.from_numpy(rng.integers(-2, 3, (total + spare, k))).to(torch.bfloat16).cuda()
    b = torch.from_numpy(rng.integers(0, 256, (1, n, k // 2), dtype=np.uint8)).expand(experts, -1, -1).contiguous().cuda()
    sf = torch.full((experts, n, k // 32), 127, dtype=torch.uint8, device="cuda")
    ps = torch.tensor([[total, n, k]] * experts, dtype=torch.int32, device="cuda")
    behind = torch.full((total + spare + 1, n), 55.0, dtype=torch.bfloat16, device="cuda")
    out = behind[:-1]
    esmoe.es_mxfp4_grouped_mm(out, a, b.transpose(1, 2), sf.transpose(1, 2), ps, torch.zeros(experts, dtype=torch.int32, device="cuda"))
    want = a[:total].double().cpu().numpy() @ O.dequant_mxfp4(b[0].cpu().numpy(), sf[0].cpu().numpy()).T
    assert torch.equal(out[:total].cpu(), torch.from_numpy(want).to(torch.bfloat16))
    assert (behind[total:] == 55.0).all()
