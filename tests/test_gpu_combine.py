"""The weighted way back from the experts and its gradients against the 64-bit oracle.

An output is off by half a step of its type and by topk fp32 roundings of the running sum: 2^-24 * topk * sum |terms|.  A dot product of H
terms runs over at most H / 512 additions per lane times eight, a tree of 6 and one of 2: (H / 64 + 16) 2^-24 * sum |terms|."""

import numpy as np
import pytest
import torch

from oracle import moe_block as O
from tests import helpers as H

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.bfloat16: 1e-40, torch.float16: 2.0 ** -25}


def _case(tokens, topk, hidden, dtype, seed, remote=0.3, spare=3):
    """Pairs packed in a random order, some of them remote, rows behind the last one that belong to nobody."""
    rng = np.random.default_rng(seed)
    dst = np.full(tokens * topk, -1, np.int32)
    here = np.flatnonzero(rng.random(dst.size) >= remote)
    dst[here] = rng.permutation(here.size)
    gen = torch.Generator().manual_seed(seed)
    rows = torch.randn((here.size + spare, hidden), generator=gen).to(dtype)
    weights = torch.randn((tokens, topk), generator=gen)
    grad = torch.randn((tokens, hidden), generator=gen).to(dtype)
    return rows, torch.from_numpy(dst), weights, grad


def _np(t):
    return t.double().cpu().numpy()


CASES = [(1, 1, 8, 0.0), (1, 8, 7168, 0.0), (5, 3, 136, 0.3), (4, 8, 4104, 0.9), (63, 2, 520, 0.3), (3, 64, 512, 0.3), (3, 70, 72, 0.3),
         (2, 130, 1032, 0.5), (301, 8, 2048, 0.75), (7, 1, 14336, 0.3), (9, 6, 512, 1.0)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,topk,hidden,remote", CASES)
def test_combine(esmoe, tokens, topk, hidden, remote, dtype):
    rows, dst, weights, _ = _case(tokens, topk, hidden, dtype, tokens + topk, remote)
    for w in (weights, None):
        out = esmoe.es_combine_rows(rows.cuda(), dst.cuda(), topk, None if w is None else w.cuda())
        want, mag = O.combine(_np(rows), dst.numpy(), topk, None if w is None else _np(w))
        bound = HALF_STEP[dtype] * np.abs(want) + (topk + 1) * 2.0 ** -24 * mag + TINY[dtype]
        assert out.dtype == dtype and (np.abs(_np(out) - want) <= bound).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,topk,hidden,remote", CASES)
def test_combine_gradient(esmoe, tokens, topk, hidden, remote, dtype):
    rows, dst, weights, grad = _case(tokens, topk, hidden, dtype, tokens + topk, remote)
    into = torch.full_like(rows, 77.0).cuda()
    got_rows, got_w = esmoe.es_combine_rows_backward(grad.cuda(), rows.cuda(), dst.cuda(), topk, weights.cuda(), into)
    assert got_rows.data_ptr() == into.data_ptr() and got_w.shape == weights.shape and got_w.dtype == torch.float32
    want_rows, want_w, mag = O.combine_grad(_np(grad), _np(rows), dst.numpy(), topk, _np(weights))
    none = np.isnan(want_rows)
    assert (_np(got_rows)[none] == 77.0).all()   # rows without a pair are left as they were
    want_rows = np.where(none, 77.0, want_rows)
    bound = (HALF_STEP[dtype] + 2.0 ** -24) * np.abs(want_rows) + TINY[dtype]
    assert (np.abs(_np(got_rows) - want_rows) <= bound).all()
    assert (np.abs(_np(got_w) - want_w) <= (hidden / 64 + 16) * 2.0 ** -24 * mag).all()
    fresh, again = esmoe.es_combine_rows_backward(grad.cuda(), rows.cuda(), dst.cuda(), topk, weights.cuda())
    assert torch.equal(again, got_w) and (_np(fresh)[none] == 0).all() and np.array_equal(_np(fresh)[~none], _np(got_rows)[~none])


def test_pairs_that_are_left_out_touch_nothing(esmoe):
    """Rows of nobody and weights of remote pairs hold NaN; indexes outside the rows count as remote."""
    rows, dst, weights, grad = _case(6, 4, 256, torch.bfloat16, 3)
    rows[-3:] = float("nan")
    flat = weights.view(-1)
    flat[dst < 0] = float("nan")
    far = dst.clone()
    far[dst < 0] = torch.tensor([-1, rows.size(0), 2 ** 31 - 1, -2 ** 31], dtype=torch.int32).repeat(6)[:(dst < 0).sum()]
    want, mag = O.combine(_np(rows), far.numpy(), 4, np.nan_to_num(_np(weights)))
    out = esmoe.es_combine_rows(rows.cuda(), far.cuda(), 4, weights.cuda())
    assert (np.abs(_np(out) - want) <= 2.0 ** -8 * np.abs(want) + 5 * 2.0 ** -24 * mag).all()
    into = torch.zeros_like(rows).cuda()
    _, gw = esmoe.es_combine_rows_backward(grad.cuda(), rows.cuda(), far.cuda(), 4, weights.cuda(), into)
    assert torch.isfinite(gw).all() and (gw.view(-1).cpu()[dst < 0] == 0).all() and torch.isfinite(into).all() and (into[-3:] == 0).all()


def test_it_is_the_gradient_of_the_row_packing(esmoe):
    """<permute(x), g> = <x, combine(g)> for all x and g: with small integers both sides are exact."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    ids = torch.randint(0, 12, (37, 5), generator=gen, device="cuda", dtype=torch.int32)   # experts 10 and 11 are remote
    _, offsets, _, dst = esmoe.es_route_metadata(ids, 0, 10, 64, 128)
    total = int(offsets[-1].item())
    x = torch.randint(-3, 4, (37, 264), generator=gen, device="cuda").to(torch.bfloat16)
    g = torch.randint(-3, 4, (total, 264), generator=gen, device="cuda").to(torch.bfloat16)
    packed = torch.zeros_like(g)
    esmoe.es_permute_rows(x, dst, 5, packed)
    back = esmoe.es_combine_rows(g, dst, 5)
    assert (packed.double() * g.double()).sum() == (x.double() * back.double()).sum()


def test_offsets_past_32_bits(esmoe):
    """A packed tensor of more than 2^31 elements (5.1 GB): rows at its end."""
    hidden, rows = 8192, 310000
    big = torch.empty((rows, hidden), dtype=torch.float16, device="cuda")
    at = torch.tensor([rows - 1, 0, 262144, rows - 2], dtype=torch.int32)
    gen = torch.Generator().manual_seed(2)
    vals = torch.randn((4, hidden), generator=gen).to(torch.float16)
    big[at.long().cuda()] = vals.cuda()
    weights, grad = torch.randn((2, 2), generator=gen), torch.randn((2, hidden), generator=gen).to(torch.float16)
    order = np.arange(4)
    out = esmoe.es_combine_rows(big, at.cuda(), 2, weights.cuda())
    want, mag = O.combine(_np(vals), order, 2, _np(weights))
    assert (np.abs(_np(out) - want) <= 2.0 ** -11 * np.abs(want) + 3 * 2.0 ** -24 * mag + 2.0 ** -25).all()
    into = torch.empty_like(big)
    _, gw = esmoe.es_combine_rows_backward(grad.cuda(), big, at.cuda(), 2, weights.cuda(), into)
    want_rows, want_w, mag = O.combine_grad(_np(grad), _np(vals), order, 2, _np(weights))
    assert (np.abs(_np(into[at.long().cuda()]) - want_rows) <= (2.0 ** -11 + 2.0 ** -24) * np.abs(want_rows) + 2.0 ** -25).all()
    assert (np.abs(_np(gw) - want_w) <= (hidden / 64 + 16) * 2.0 ** -24 * mag).all()


def test_rows_beyond_the_cache_give_the_bytes_of_small_calls(esmoe):
    """More than 256 MB of rows and gradients, ragged, some pairs remote, against the same tokens a few at a time."""
    for tokens, topk, hidden in ((2503, 8, 8184), (40007, 3, 1160)):
        rows, dst, weights, grad = (t.cuda() for t in _case(tokens, topk, hidden, torch.bfloat16, 8, 0.1))
        assert rows.numel() * 2 > 2 ** 28 // 2
        for w in (weights, None):
            whole = esmoe.es_combine_rows(rows, dst, topk, w)
            for t in range(0, tokens, 997):
                part = slice(t, min(t + 997, tokens))
                assert torch.equal(whole[part], esmoe.es_combine_rows(rows, dst[part.start * topk:part.stop * topk], topk, None if w is None else w[part]))
        into, small = torch.full_like(rows, 7.0), torch.full_like(rows, 7.0)
        _, gw = esmoe.es_combine_rows_backward(grad, rows, dst, topk, weights, into)
        for t in range(0, tokens, 997):
            part = slice(t, min(t + 997, tokens))
            _, g = esmoe.es_combine_rows_backward(grad[part], rows, dst[part.start * topk:part.stop * topk], topk, weights[part], small)
            assert torch.equal(gw[part], g)
        assert torch.equal(into, small)


def test_empty_calls_and_overlaps(esmoe):
    rows = torch.zeros((4, 64), dtype=torch.bfloat16, device="cuda")
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    assert esmoe.es_combine_rows(rows, none, 3).shape == (0, 64)
    far = torch.full((6,), -1, dtype=torch.int32, device="cuda")
    assert (esmoe.es_combine_rows(rows[:0], far, 2, torch.ones(3, 2, device="cuda")) == 0).all()   # no local row at all
    gr, gw = esmoe.es_combine_rows_backward(torch.ones((3, 64), dtype=torch.bfloat16, device="cuda"), rows[:0], far, 2, torch.ones(3, 2, device="cuda"))
    assert gr.shape == (0, 64) and (gw == 0).all()
    dst = torch.arange(4, dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="may not overlap"):
        esmoe.es_combine_rows(rows, dst, 1, None, rows)
    with pytest.raises(RuntimeError, match="may not overlap"):
        esmoe.es_combine_rows_backward(rows, rows.clone(), dst, 1, torch.ones(4, 1, device="cuda"), rows)
    w = torch.ones(4, 1, device="cuda")
    with pytest.raises(RuntimeError, match="may not overlap"):
        esmoe.es_combine_rows_backward(rows, rows.clone(), dst, 1, w, grad_weights=w)
    out = torch.zeros_like(rows)
    with pytest.raises(RuntimeError, match="may not overlap"):
        esmoe.es_combine_rows(rows, dst, 1, out.view(-1).view(torch.float32)[4:8], out)


def test_c_abi(esmoe):
    from expert_specialization_moe_amd import _native

    rows, dst, weights, grad = (t.cuda() for t in _case(5, 3, 256, torch.float16, 8))
    out, gin, gw = torch.empty((5, 256), dtype=torch.float16, device="cuda"), torch.zeros_like(rows), torch.empty((5, 3), device="cuda")
    rc = _native.lib.esmoe_combine_rows(H.ptr(rows), 1, H.ptr(dst), H.ptr(weights), 15, 3, rows.size(0), 256, H.ptr(out), H.stream_ptr())
    assert rc == 0, _native.last_error()
    rc = _native.lib.esmoe_combine_rows_backward(H.ptr(grad), H.ptr(rows), 1, H.ptr(dst), H.ptr(weights), 15, 3, rows.size(0), 256, H.ptr(gin),
                                                 H.ptr(gw), H.stream_ptr())
    assert rc == 0, _native.last_error()
    assert torch.equal(out, esmoe.es_combine_rows(rows, dst, 3, weights))
    want = esmoe.es_combine_rows_backward(grad, rows, dst, 3, weights)
    assert torch.equal(gin, want[0]) and torch.equal(gw, want[1])
