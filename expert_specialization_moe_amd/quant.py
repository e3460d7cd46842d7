"""Torch-side quantisers that prepare operands for the grouped GEMMs (run on any device).

They produce the tensors the reference's callers build with its test helpers
(test/test_es_grouped_gemm.py:36-59): e4m3fn data with fp32 scales per 1x128
block of an activation row and per 128x128 block of a weight matrix.  They are
input preparation, not part of the measured path.
"""
import torch

FP8_MAX = 448.0


def quant_act_1x128(x: torch.Tensor):
    """[M, K] (K % 128 == 0) -> (e4m3fn [M, K], fp32 scales [M, K/128])."""
    assert x.dim() == 2 and x.size(1) % 128 == 0
    m, k = x.shape
    xv = x.view(m, k // 128, 128)
    amax = xv.abs().float().amax(dim=2).clamp(1e-4)
    q = (xv * (FP8_MAX / amax.unsqueeze(2))).to(torch.float8_e4m3fn)
    return q.view(m, k), amax / FP8_MAX


def quant_weight_128x128(w: torch.Tensor):
    """[..., N, K] (both % 128 == 0) -> (e4m3fn [..., N, K], fp32 scales [..., N/128, K/128])."""
    assert w.size(-1) % 128 == 0 and w.size(-2) % 128 == 0
    lead = w.shape[:-2]
    n, k = w.shape[-2:]
    wv = w.reshape(*lead, n // 128, 128, k // 128, 128)
    amax = wv.abs().float().amax(dim=(-3, -1), keepdim=True).clamp(1e-4)
    q = (wv * (FP8_MAX / amax)).to(torch.float8_e4m3fn)
    return q.reshape(*lead, n, k), (amax / FP8_MAX).reshape(*lead, n // 128, k // 128)


def quant_weight_mxfp4(w: torch.Tensor):
    """[..., N, K] (K % 32 == 0) -> (uint8 [..., N, K/2], E8M0 uint8 [..., N, K/32]) for es_mxfp4_grouped_mm, once per weight.

    A block of 32 along K has the scale 2^(code - 127), the smallest power of two from amax / 6 on, and values rounded to the nearest
    e2m1 (0, .5, 1, 1.5, 2, 3, 4, 6 and their negatives; a tie goes to the even code).  The even column of a byte is its low half.
    A block without a finite amax gets the scale NaN (255).
    """
    assert w.size(-1) % 32 == 0
    lead, k = w.shape[:-1], w.size(-1)
    v = w.float().reshape(*lead, k // 32, 32)
    amax = v.abs().amax(dim=-1)
    mant, exp = torch.frexp(amax)               # amax = mant 2^exp, mant in [.5, 1); 6 = .75 * 2^3
    exp = (exp - 3 + (mant > 0.75).to(exp.dtype)).clamp(-127, 127)
    v = torch.ldexp(v, -exp.unsqueeze(-1)).reshape(*lead, k)
    mag = v.abs()
    code = torch.zeros(mag.shape, dtype=torch.uint8, device=w.device)
    # half-way values go down where the lower code is even, up where it is odd
    for edge, even_below in ((0.25, True), (0.75, False), (1.25, True), (1.75, False), (2.5, True), (3.5, False), (5.0, True)):
        code += (mag > edge) if even_below else (mag >= edge)
    code |= torch.signbit(v).to(torch.uint8) << 3
    sf = torch.where(torch.isfinite(amax), exp + 127, 255).to(torch.uint8)
    return (code[..., 0::2] | (code[..., 1::2] << 4)).contiguous(), sf
