"""The operators around the grouped GEMMs reject bad arguments before any launch: through torch (CPU tensors: the checks run, then
the call is refused for want of a device) and through the C ABI."""
import ctypes

import pytest
import torch

BF = torch.bfloat16


def _refused(match, f, *args, **kw):
    with torch.no_grad(), pytest.raises(RuntimeError, match=match):
        f(*args, **kw)


def test_gating_refusals(esmoe):
    x = torch.zeros(3, 16)
    _refused("no CPU implementation", esmoe.es_topk_gating, x, 4)
    _refused("no CPU implementation", esmoe.es_topk_gating, x.to(BF), 4, torch.zeros(16), "sigmoid", False, 2.5, 4, 2)
    _refused("no CPU implementation", esmoe.es_topk_gating, torch.zeros(3, 20)[:, 2:18], 16)   # rows apart are fine
    _refused("2D", esmoe.es_topk_gating, x[0], 4)
    _refused("row major", esmoe.es_topk_gating, torch.zeros(16, 3).t(), 4)
    _refused("float32, bfloat16 or half", esmoe.es_topk_gating, x.double(), 4)
    _refused("topk must be", esmoe.es_topk_gating, x, 17)
    _refused("topk must be", esmoe.es_topk_gating, x, 0)
    _refused("topk must be", esmoe.es_topk_gating, torch.zeros(1, 100), 65)
    _refused("Number of experts", esmoe.es_topk_gating, torch.zeros(1, 1025), 4)
    _refused("bias must be", esmoe.es_topk_gating, x, 4, torch.zeros(15))
    _refused("bias must be", esmoe.es_topk_gating, x, 4, torch.zeros(16, dtype=BF))
    _refused("num_groups", esmoe.es_topk_gating, x, 4, num_groups=3)
    _refused("topk_groups", esmoe.es_topk_gating, x, 4, num_groups=4, topk_groups=5)
    _refused("more than the experts", esmoe.es_topk_gating, x, 5, num_groups=4, topk_groups=1)
    _refused("scale must be finite", esmoe.es_topk_gating, x, 4, scale=float("inf"))
    with pytest.raises(ValueError, match="scoring"):
        esmoe.es_topk_gating(x, 4, scoring="tanh")
    with pytest.raises(RuntimeError, match="not differentiable by autograd"):
        esmoe.es_topk_gating(x.clone().requires_grad_(), 4)
    g, ids = torch.zeros(3, 4), torch.zeros(3, 4, dtype=torch.int32)
    _refused("no CPU implementation", esmoe.es_topk_gating_backward, g, x, ids)
    _refused("topk_ids must be", esmoe.es_topk_gating_backward, g, x, ids.long())
    _refused("a row per row", esmoe.es_topk_gating_backward, g, x[:2], ids)
    _refused("grad_weights must be", esmoe.es_topk_gating_backward, g[:, :3], x, ids)
    _refused("grad_weights must be", esmoe.es_topk_gating_backward, g.half(), x, ids)


def test_combine_refusals(esmoe):
    y, dst, w = torch.zeros(6, 16, dtype=BF), torch.zeros(8, dtype=torch.int32), torch.zeros(4, 2)
    _refused("no CPU implementation", esmoe.es_combine_rows, y, dst, 2, w)
    _refused("no CPU implementation", esmoe.es_combine_rows, y, dst, 2)
    _refused("bfloat16 or half", esmoe.es_combine_rows, y.float(), dst, 2, w)
    _refused("contiguous 2D", esmoe.es_combine_rows, torch.zeros(6, 32, dtype=BF)[:, :16], dst, 2, w)
    _refused("16 bytes", esmoe.es_combine_rows, torch.zeros(6, 12, dtype=BF), dst, 2, w)
    _refused("int32", esmoe.es_combine_rows, y, dst.long(), 2, w)
    _refused("tokens \\* topk", esmoe.es_combine_rows, y, dst, 3, w)
    _refused("tokens \\* topk", esmoe.es_combine_rows, y, dst, 0, w)
    _refused("weights must be", esmoe.es_combine_rows, y, dst, 2, w[:3])
    _refused("weights must be", esmoe.es_combine_rows, y, dst, 2, w.half())
    _refused("output must be", esmoe.es_combine_rows, y, dst, 2, w, torch.zeros(4, 16))
    _refused("output must be", esmoe.es_combine_rows, y, dst, 2, w, torch.zeros(5, 16, dtype=BF))
    with pytest.raises(RuntimeError, match="not differentiable by autograd"):
        esmoe.es_combine_rows(y, dst, 2, w.clone().requires_grad_())
    g = torch.zeros(4, 16, dtype=BF)
    _refused("no CPU implementation", esmoe.es_combine_rows_backward, g, y, dst, 2, w)
    _refused("grad_output must be", esmoe.es_combine_rows_backward, g[:3], y, dst, 2, w)
    _refused("grad_output must be", esmoe.es_combine_rows_backward, g.half(), y, dst, 2, w)
    _refused("grad_input must be", esmoe.es_combine_rows_backward, g, y, dst, 2, w, torch.zeros(5, 16, dtype=BF))
    _refused("grad_weights must be", esmoe.es_combine_rows_backward, g, y, dst, 2, w, None, torch.zeros(7))


def test_norm_refusals(esmoe):
    f = esmoe.es_add_rms_norm_quant_1x128
    x, w = torch.zeros(3, 256, dtype=BF), torch.ones(256, dtype=BF)
    _refused("no CPU implementation", f, x, w)
    _refused("no CPU implementation", f, x, w, 1e-6, x.clone(), return_normed=True)
    _refused("contiguous 2D", f, torch.zeros(3, 512, dtype=BF)[:, :256], w)
    _refused("kFloat16 or kBFloat16", f, x.float(), w.float())
    _refused("k must align", f, torch.zeros(3, 192, dtype=BF), w[:192])
    _refused("k must align", f, torch.zeros(1, 32896, dtype=BF), torch.zeros(32896, dtype=BF))
    _refused("weight must be", f, x, w.half())
    _refused("weight must be", f, x, w[:128])
    _refused("eps must be", f, x, w, -1.0)
    _refused("eps must be", f, x, w, float("nan"))
    _refused("input's shape and dtype", f, x, w, 1e-6, x[:2])
    _refused("input's shape and dtype", f, x, w, 1e-6, x.half())
    _refused("go together", f, x, w, 1e-6, None, x.clone())
    _refused("quant_output must be", f, x, w, quant_output=torch.zeros(3, 128, dtype=torch.uint8))
    _refused("scales must be", f, x, w, scales=torch.zeros(3, 3))
    with pytest.raises(RuntimeError, match="not differentiable by autograd"):
        f(x, w.clone().requires_grad_())


@pytest.mark.parametrize("swiglu", [False, True])
def test_mxfp4_refusals(esmoe, swiglu):
    f = esmoe.es_mxfp4_grouped_mm_swiglu if swiglu else esmoe.es_mxfp4_grouped_mm
    e, n, k, rows = 2, 64, 256, 5
    good = dict(output=torch.zeros(rows, n // 2 if swiglu else n, dtype=BF), a=torch.zeros(rows, k, dtype=BF),
                b=torch.zeros(e, n, k // 2, dtype=torch.uint8).transpose(1, 2), sfb=torch.zeros(e, n, k // 32, dtype=torch.uint8).transpose(1, 2),
                problem_sizes=torch.tensor([[3, n, k], [2, n, k]], dtype=torch.int32), expert_offsets=torch.tensor([0, 3], dtype=torch.int32))
    call = lambda match, **kw: _refused(match, f, *dict(good, **kw).values())
    call("no CPU implementation")
    call("bfloat16 or half", a=good["a"].float())
    call("packed row-major", a=torch.zeros(rows, 2 * k, dtype=BF)[:, :k])
    call("multiple of 128", a=torch.zeros(rows, 192, dtype=BF))
    call("k/2, n", b=torch.zeros(e, n, k, dtype=torch.uint8).transpose(1, 2))
    call("column-major", b=torch.zeros(e, k // 2, n, dtype=torch.uint8))
    call("n must be", b=torch.zeros(e, 24, k // 2, dtype=torch.uint8).transpose(1, 2))
    call("sfb must be", sfb=torch.zeros(e, k // 32, n, dtype=torch.uint8))
    call("sfb must be", sfb=torch.zeros(e, n, k // 16, dtype=torch.uint8).transpose(1, 2))
    call("output must be", output=good["output"].half())
    call("output must be", output=torch.zeros(rows, n + 16, dtype=BF))
    call("must match expert_offsets", expert_offsets=torch.zeros(3, dtype=torch.int32))
    call("int32", problem_sizes=good["problem_sizes"].long())
    with pytest.raises(RuntimeError, match="not differentiable by autograd"):
        f(*dict(good, a=good["a"].clone().requires_grad_()).values())


def test_c_abi_refusals(esmoe):
    from expert_specialization_moe_amd import _native

    lib = _native.lib
    buf = (ctypes.c_char * 4096)()
    base = ctypes.addressof(buf)
    p = ctypes.c_void_p(base + 16 - base % 16)
    odd = ctypes.c_void_p(p.value + 8)

    def bad(match, rc):
        assert rc == -1 and match in _native.last_error(), (rc, _native.last_error())

    gate = lib.esmoe_topk_gating
    bad("logits_dtype", gate(p, 3, 16, p, 4, 16, 4, 0, 1, 1.0, 1, 1, p, p, None))
    bad("num_experts", gate(p, 2, 16, p, 4, 1025, 4, 0, 1, 1.0, 1, 1, p, p, None))
    bad("topk", gate(p, 2, 16, p, 4, 16, 17, 0, 1, 1.0, 1, 1, p, p, None))
    bad("scoring", gate(p, 2, 16, p, 4, 16, 4, 2, 1, 1.0, 1, 1, p, p, None))
    bad("tokens", gate(p, 2, 16, p, 1 << 30, 16, 4, 0, 1, 1.0, 1, 1, p, p, None))
    bad("row stride", gate(p, 2, -1, p, 4, 16, 4, 0, 1, 1.0, 1, 1, p, p, None))
    bad("scale", gate(p, 2, 16, p, 4, 16, 4, 0, 1, float("nan"), 1, 1, p, p, None))
    bad("num_groups", gate(p, 2, 16, p, 4, 16, 4, 0, 1, 1.0, 5, 1, p, p, None))
    bad("topk_groups", gate(p, 2, 16, p, 4, 16, 4, 0, 1, 1.0, 4, 0, p, p, None))
    bad("null", gate(None, 2, 16, p, 4, 16, 4, 0, 1, 1.0, 1, 1, p, p, None))
    assert gate(None, 2, 16, None, 0, 16, 4, 0, 1, 1.0, 1, 1, None, None, None) == 0
    bad("null", lib.esmoe_topk_gating_backward(p, p, 2, 16, None, 4, 16, 4, 0, 1, 1.0, p, None))
    assert lib.esmoe_topk_gating_backward(None, None, 2, 16, None, 0, 16, 4, 0, 1, 1.0, None, None) == 0
    comb = lib.esmoe_combine_rows
    bad("dtype", comb(p, 2, p, p, 8, 2, 6, 16, p, None))
    bad("num_pairs", comb(p, 0, p, p, 7, 2, 6, 16, p, None))
    bad("rows", comb(p, 0, p, p, 8, 2, -1, 16, p, None))
    bad("hidden", comb(p, 0, p, p, 8, 2, 6, 12, p, None))
    bad("aligned", comb(odd, 0, p, p, 8, 2, 6, 16, p, None))
    bad("null", comb(p, 0, None, p, 8, 2, 6, 16, p, None))
    assert comb(None, 0, None, None, 0, 2, 0, 16, None, None) == 0
    back = lib.esmoe_combine_rows_backward
    bad("null", back(p, p, 0, p, None, 8, 2, 6, 16, p, p, None))
    bad("aligned", back(p, p, 0, p, p, 8, 2, 6, 16, odd, p, None))
    norm = lib.esmoe_add_rms_norm_quant_1x128
    bad("k must", norm(p, 0, p, p, 1e-6, 4, 100, p, p, p, p, None))
    bad("in_dtype", norm(p, 2, p, p, 1e-6, 4, 128, p, p, p, p, None))
    bad("eps", norm(p, 0, p, p, -1.0, 4, 128, p, p, p, p, None))
    bad("go together", norm(p, 0, p, p, 1e-6, 4, 128, None, p, p, p, None))
    bad("aligned", norm(p, 0, None, odd, 1e-6, 4, 128, None, None, p, p, None))
    assert norm(None, 0, None, None, 1e-6, 0, 128, None, None, None, None, None) == 0
    mm = lib.esmoe_mxfp4_grouped_mm
    bad("dtype", mm(p, 2, p, p, p, p, p, 4, 8, 64, 128, 0, None))
    bad("num_experts", mm(p, 0, p, p, p, p, p, 0, 8, 64, 128, 0, None))
    bad("total_rows", mm(p, 0, p, p, p, p, p, 4, -1, 64, 128, 0, None))
    bad("k must", mm(p, 0, p, p, p, p, p, 4, 8, 64, 96, 0, None))
    bad("n must", mm(p, 0, p, p, p, p, p, 4, 8, 48, 128, 1, None))
    bad("aligned", mm(p, 0, odd, p, p, p, p, 4, 8, 64, 128, 0, None))
    bad("null", mm(p, 0, p, p, None, p, p, 4, 8, 64, 128, 0, None))
    assert mm(None, 0, None, None, None, None, None, 4, 0, 64, 128, 0, None) == 0
