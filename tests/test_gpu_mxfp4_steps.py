"""Grouped products with 4-bit weights where a workgroup runs through several steps (a step: two tiles of sixteen weight rows), from one
unit to the next and over the 64 experts that a wavefront looks at together; every instance of the streaming kernel, one to four pairs
of K chunks a wavefront.

Activations are -1, 0 and 1 and scales 2^-5 to 2^-3: a sum is a multiple of 2^-6 below 2^18, exact in fp32 in any order, so the plain
product is the float64 one rounded once.  With SwiGLU the sums are exact too; the sigmoid's exponential adds |gate| 2^-23 of the value
(the rounding of its argument) and the reciprocal and the products a few units of 2^-24: (|gate| + 8) 2^-23, and half a step of the output."""
import numpy as np
import pytest
import torch

from oracle import moe_block as O

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.bfloat16: 1e-33, torch.float16: 2.0 ** -25}   # (gates below -88: 1 + exp(88) is infinite in fp32 and the value, below 1e-34, is 0)
FAR = {torch.bfloat16: 254, torch.float16: 200}   # a scale that the 16-bit type cannot take in: its step is done again
ZERO_BLOCK = 3                                    # activations of this block are 0: far and NaN scales stand here


def _grid(k):
    """Workgroups that the launch starts where there are steps enough, and pairs of chunks per wavefront."""
    pairs = (k // 128 + 1) // 2
    each = (pairs + 7) // 8
    waves = (pairs + each - 1) // each
    per_cu = {1: 16, 2: 12, 3: 8, 4: 8}[each] // waves
    return torch.cuda.get_device_properties(0).multi_processor_count * per_cu, each


def _weights(b, sf):
    """float64 [N, K] of one expert, on the device."""
    table = torch.from_numpy(O.E2M1).cuda()
    v = torch.stack([table[(b & 15).long()], table[(b >> 4).long()]], dim=-1).view(b.size(0), -1, 32)
    scale = torch.exp2(sf.double() - 127).masked_fill(sf == 255, float("nan"))
    return (v * scale.unsqueeze(2)).view(b.size(0), -1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("swiglu", [False, True])
@pytest.mark.parametrize("k,pairs", [(128, 1), (1152, 1), (2048, 1), (2176, 2), (4096, 2), (4224, 3), (5248, 3), (6272, 4), (7168, 4), (8064, 4), (8192, 4)])
def test_several_steps_a_workgroup(esmoe, k, pairs, swiglu, dtype):
    gen = torch.Generator(device="cuda").manual_seed(k)
    rng = np.random.default_rng(k)
    grid, each = _grid(k)
    assert each == pairs
    experts = 150
    rows = rng.integers(1, 40, experts) * (rng.random(experts) < 0.4)
    rows[[0, 63, 64, 128, 149]] = 1, 17, 3, 16, 33
    units = int(((rows + 15) // 16).sum())
    steps = int(np.ceil(3.3 * grid / units))
    n = 32 * steps if swiglu else 32 * steps - 16   # plain: an odd number of tiles, the last step has one
    assert units * steps > 3 * grid and (units * steps) % grid   # what this test is about: three or four steps each
    ri = lambda lo, hi, *shape: torch.randint(lo, hi, shape, generator=gen, device="cuda")
    total = int(rows.sum())
    a = ri(-1, 2, total + 5, k).to(dtype)
    a.view(total + 5, k // 32, 32)[:, ZERO_BLOCK] = 0
    b = ri(0, 256, experts, n, k // 2).to(torch.uint8)
    sf = ri(122, 125, experts, n, k // 32).to(torch.uint8)
    far = torch.rand((experts, n), generator=gen, device="cuda") < 0.01   # about every fourth step
    sf[:, :, ZERO_BLOCK][far] = FAR[dtype]
    last, nan_row = experts - 1, n // 2 + 5
    sf[last, nan_row, ZERO_BLOCK] = 255
    offsets = np.concatenate([[0], np.cumsum(rows)[:-1]])
    ps = torch.tensor([[int(m), n, k] for m in rows], dtype=torch.int32, device="cuda")
    out = torch.full((total + 5, n // 2 if swiglu else n), 55.0, dtype=dtype, device="cuda")
    f = esmoe.es_mxfp4_grouped_mm_swiglu if swiglu else esmoe.es_mxfp4_grouped_mm
    f(out, a, b.transpose(1, 2), sf.transpose(1, 2), ps, torch.tensor(offsets, dtype=torch.int32, device="cuda"))
    assert (out[total:] == 55.0).all()
    for e, (m, off) in enumerate(zip(rows, offsets)):
        if m == 0:
            continue
        want = torch.matmul(a[off:off + m].double(), _weights(b[e], sf[e]).t().contiguous())
        got = out[off:off + m]
        nan = torch.zeros(n, dtype=torch.bool, device="cuda")
        if e == last:
            nan[nan_row] = True
        if swiglu:
            gate, up = want[:, :n // 2], want[:, n // 2:]
            nan = nan[:n // 2] | nan[n // 2:]
            want = gate / (1 + torch.exp(-gate)) * up
            err = (gate.abs() + 8) * 2.0 ** -23 * want.abs()
            ok = (got.double() - want).abs() <= err + HALF_STEP[dtype] * (want.abs() + err) + TINY[dtype]
        else:
            ok = got == want.to(dtype)
        assert ok[:, ~nan].all(), (e, int(m), (~ok).nonzero()[:4].tolist())
        assert torch.isnan(got[:, nan]).all() and int(nan.sum()) == (e == last)


def test_weights_past_32_bits_stream(esmoe):
    """More than 4 GB of weights: the last expert's, one step behind another."""
    e, n, k = 66, 16384, 8192
    b = torch.zeros((e, n, k // 2), dtype=torch.uint8, device="cuda")
    sf = torch.full((e, n, k // 32), 127, dtype=torch.uint8, device="cuda")
    rng = np.random.default_rng(3)
    tail = torch.from_numpy(rng.integers(0, 256, (48, k // 2), dtype=np.uint8)).cuda()
    b[-1, -48:] = tail
    a = torch.from_numpy(rng.integers(-1, 2, (18, k))).to(torch.bfloat16).cuda()
    out = torch.empty((18, n), dtype=torch.bfloat16, device="cuda")
    ps = torch.zeros((e, 3), dtype=torch.int32, device="cuda")
    ps[-1, 0] = 18
    esmoe.es_mxfp4_grouped_mm(out, a, b.transpose(1, 2), sf.transpose(1, 2), ps, torch.zeros(e, dtype=torch.int32, device="cuda"))
    want = torch.matmul(a.double(), _weights(tail, sf[-1, -48:]).t().contiguous())
    assert torch.equal(out[:, -48:], want.to(torch.bfloat16)) and (out[:, :-48] == 0).all()
