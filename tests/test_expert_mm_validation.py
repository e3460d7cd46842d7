"""The experts' products, their gradients, the int8 quantiser and the clipping of gradients reject bad arguments before any launch: through
torch (CPU tensors: the checks run, then the call is refused for want of a device) and through the C ABI."""
import ctypes

import pytest
import torch
import torch.autograd.forward_ad as fwd

BF, HF, I8 = torch.bfloat16, torch.float16, torch.int8


def _refused(match, f, *args, **kw):
    with torch.no_grad(), pytest.raises(RuntimeError, match=match):
        f(*args, **kw)


def _meta(n=32, k=48, rows=(3, 2)):
    return (torch.tensor([[m, n, k] for m in rows], dtype=torch.int32), torch.tensor([0, rows[0]], dtype=torch.int32))


def _b(e=2, n=32, k=48, dtype=BF):
    return torch.zeros(e, n, k, dtype=dtype).transpose(1, 2)


NO_GPU = "no CPU implementation"


def test_product_refusals(esmoe):
    f, a, out, m = esmoe.es_grouped_mm, torch.zeros(5, 48, dtype=BF), torch.zeros(5, 32, dtype=BF), _meta()
    _refused(NO_GPU, f, out, a, _b(), *m)
    _refused(NO_GPU, f, out.half(), a.half(), _b(dtype=HF), *m)
    _refused("bfloat16 or half", f, out.float(), a.float(), _b(dtype=torch.float32), *m)
    _refused("of a's dtype", f, out, a, _b(dtype=HF), *m)
    _refused("output must be", f, out.half(), a, _b(), *m)
    _refused("output must be", f, out[:4], a, _b(), *m)
    _refused("output must be", f, torch.zeros(5, 64, dtype=BF)[:, :32], a, _b(), *m)
    _refused("packed row-major", f, out, torch.zeros(5, 96, dtype=BF)[:, :48], _b(), *m)
    _refused("packed row-major", f, out, a[0], _b(), *m)
    _refused("k must be a multiple of 8", f, out, torch.zeros(5, 52, dtype=BF), _b(k=52), *m)
    _refused("k must be a multiple of 8", f, out, torch.zeros(5, 0, dtype=BF), _b(k=0), *m)
    _refused("n must be a multiple of 8", f, torch.zeros(5, 36, dtype=BF), a, _b(n=36), *m)
    _refused("column-major", f, out, a, _b().contiguous(), *m)
    _refused("column-major", f, out, a, torch.zeros(2, 32, 96, dtype=BF)[:, :, :48].transpose(1, 2), *m)
    _refused("column-major", f, out, a, torch.zeros(4, 32, 48, dtype=BF)[::2].transpose(1, 2), *m)
    _refused("\\(num_experts, k, n\\)", f, out, a, _b(e=3), *m)
    _refused("\\(num_experts, k, n\\)", f, out, a, _b()[0], *m)
    _refused("problem_sizes must have", f, out, a, _b(), m[0][:, :2], m[1])
    _refused("must match expert_offsets", f, out, a, _b(), m[0], m[1][:1])
    _refused("int32", f, out, a, _b(), m[0].long(), m[1])
    _refused("int32", f, out, a, _b(), m[0], m[1].long())
    _refused("contiguous", f, out, a, _b(), torch.zeros(4, 3, dtype=torch.int32)[::2], m[1])
    big = torch.zeros(1025, 3, dtype=torch.int32), torch.zeros(1025, dtype=torch.int32)
    _refused("cannot exceed 1024", f, torch.zeros(5, 8, dtype=BF), torch.zeros(5, 8, dtype=BF), _b(1025, 8, 8), *big)
    s = esmoe.es_grouped_mm_swiglu
    h = torch.zeros(5, 16, dtype=BF)
    _refused(NO_GPU, s, h, a, _b(), *m)
    _refused(NO_GPU, s, h, a, _b(), *m, gate_up=out)
    _refused("output must be", s, out, a, _b(), *m)
    _refused("gate_up must be", s, h, a, _b(), *m, gate_up=h)
    _refused("of 16 with SwiGLU", s, torch.zeros(5, 12, dtype=BF), a, _b(n=24), *m)


def test_gradient_refusals(esmoe):
    f, a, d, m = esmoe.es_grouped_mm_backward, torch.zeros(5, 48, dtype=BF), torch.zeros(5, 32, dtype=BF), _meta()
    _refused(NO_GPU, f, d, a, _b(), *m)
    _refused(NO_GPU, f, d, a, _b(), *m, grad_a=torch.zeros(5, 48, dtype=BF), grad_b=_b())
    _refused(NO_GPU, f, d, a, _b(), *m, need_grad_a=False, need_grad_b=False)
    _refused("grad_output must be", f, d[:, :16], a, _b(), *m)
    _refused("grad_output must be", f, d.half(), a, _b(), *m)
    _refused("grad_a must be", f, d, a, _b(), *m, grad_a=torch.zeros(4, 48, dtype=BF))
    _refused("grad_a must be", f, d, a, _b(), *m, grad_a=torch.zeros(5, 48))
    _refused("grad_b must be", f, d, a, _b(), *m, grad_b=_b().contiguous())
    _refused("grad_b must be", f, d, a, _b(), *m, grad_b=_b(dtype=HF))
    _refused("grad_b must be", f, d, a, _b(), *m, grad_b=_b(e=1))
    _refused("\\(num_experts, k, n\\)", f, d, a, _b()[0], *m)
    s, dh = esmoe.es_grouped_mm_swiglu_backward, torch.zeros(5, 16, dtype=BF)
    _refused(NO_GPU, s, dh, a, _b(), d, *m)
    _refused("gate_up must be", s, dh, a, _b(), dh, *m)
    _refused("grad_output must be", s, d, a, _b(), d, *m)


def test_int8_refusals(esmoe):
    f, m = esmoe.es_int8_scaled_grouped_mm, _meta()
    a, out, sa, sb = torch.zeros(5, 48, dtype=I8), torch.zeros(5, 32, dtype=BF), torch.zeros(5), torch.zeros(2, 32)
    _refused(NO_GPU, f, out, a, _b(dtype=I8), sa, sb, *m)
    _refused(NO_GPU, esmoe.es_int8_scaled_grouped_mm_swiglu, out[:, :16].contiguous(), a, _b(dtype=I8), sa, sb, *m)
    _refused("a must be int8", f, out, a.to(torch.uint8), _b(dtype=I8), sa, sb, *m)
    _refused("of a's dtype", f, out, a, _b(dtype=torch.uint8), sa, sb, *m)
    _refused("k must be a multiple of 16", f, out, torch.zeros(5, 56, dtype=I8), _b(k=56, dtype=I8), sa, sb, *m)
    _refused("k must be a multiple of 16 up to 65536", f, out, torch.zeros(5, 65552, dtype=I8), _b(k=65552, dtype=I8), sa, sb, *m)
    _refused("output must be", f, out.float(), a, _b(dtype=I8), sa, sb, *m)
    _refused("scales_a must be", f, out, a, _b(dtype=I8), sa[:4], sb, *m)
    _refused("scales_a must be", f, out, a, _b(dtype=I8), sa.half(), sb, *m)
    _refused("scales_b must be", f, out, a, _b(dtype=I8), sa, sb[:1], *m)
    _refused("scales_b must be", f, out, a, _b(dtype=I8), sa, sb.t().contiguous().t(), *m)
    q = esmoe.es_int8_quant
    x = torch.zeros(3, 32, dtype=BF)
    _refused(NO_GPU, q, x)
    _refused(NO_GPU, q, x, torch.zeros(3, 32, dtype=I8))
    _refused("kFloat16 or kBFloat16", q, x.float())
    _refused("k must be a multiple of 16", q, torch.zeros(3, 24, dtype=BF))
    _refused("k must be a multiple of 16", q, torch.zeros(1, 65552, dtype=BF))
    _refused("contiguous", q, torch.zeros(3, 64, dtype=BF)[:, :32])
    _refused("at least 1 dimension", q, torch.zeros((), dtype=BF))
    _refused("quant_output must be", q, x, torch.zeros(3, 16, dtype=I8))
    _refused("scales must be", q, x, None, torch.zeros(2))


def test_clip_refusals(esmoe):
    f, g = esmoe.es_clip_grad_norm, [torch.zeros(3, 4), torch.zeros(5, dtype=BF)]
    _refused(NO_GPU, f, g, 1.0)
    _refused(NO_GPU, f, g, 1.0, norm=torch.zeros(()), outputs=[t.clone() for t in g])
    _refused(NO_GPU, esmoe.es_grad_norm, g)
    for call in (esmoe.es_grad_norm, lambda x: f(x, 1.0)):
        _refused("no tensor arguments|no gradients given", call, [])
        _refused("float32, bfloat16 or half", call, g + [torch.zeros(3, dtype=torch.float64)])
        _refused("dense in memory", call, [torch.zeros(4, 6)[:, :3]])
        _refused("dense in memory", call, [torch.zeros(3, 1).expand(3, 4)])
        _refused("dense tensors|backend", call, [torch.zeros(3, 4).to_sparse()])
    _refused("max_norm", f, g, -1.0)
    _refused("max_norm", f, g, float("nan"))
    _refused("eps must be", f, g, 1.0, eps=-1e-9)
    _refused("eps must be", f, g, 1.0, eps=float("inf"))
    _refused("norm must be", f, g, 1.0, norm=torch.zeros(2))
    _refused("norm must be", f, g, 1.0, norm=torch.zeros((), dtype=torch.float64))
    _refused("a tensor per gradient", f, g, 1.0, outputs=g[:1])
    _refused("shapes, strides and dtypes", f, g, 1.0, outputs=[g[0].t().contiguous().t(), g[1]])
    _refused("shapes, strides and dtypes", f, g, 1.0, outputs=[g[0], g[1].float()])


def _autograd_calls(esmoe):
    """name -> (call, tensors that carry derivatives, buffers that are written)."""
    z, m = torch.zeros, _meta()
    a, d, h = z(5, 48, dtype=BF), z(5, 32, dtype=BF), z(5, 16, dtype=BF)
    b = lambda: _b()
    return {
        "mm": (lambda a, b, out: esmoe.es_grouped_mm(out, a, b, *m), dict(a=a, b=b()), dict(out=d)),
        "swiglu": (lambda a, b, out, gu: esmoe.es_grouped_mm_swiglu(out, a, b, *m, gate_up=gu), dict(a=a, b=b()), dict(out=h, gu=d)),
        "mm_backward": (lambda d, a, b, ga, gb: esmoe.es_grouped_mm_backward(d, a, b, *m, grad_a=ga, grad_b=gb), dict(d=d, a=a, b=b()),
                        dict(ga=z(5, 48, dtype=BF), gb=b())),
        "swiglu_backward": (lambda d, a, b, gu, ga, gb: esmoe.es_grouped_mm_swiglu_backward(d, a, b, gu, *m, grad_a=ga, grad_b=gb),
                            dict(d=h, a=a, b=b(), gu=d), dict(ga=z(5, 48, dtype=BF), gb=b())),
        "int8": (lambda sa, sb, out: esmoe.es_int8_scaled_grouped_mm(out, z(5, 48, dtype=I8), _b(dtype=I8), sa, sb, *m),
                 dict(sa=z(5), sb=z(2, 32)), dict(out=d)),
        "quant": (lambda x, s: esmoe.es_int8_quant(x, None, s), dict(x=a), dict(s=z(5))),
        "quant_new": (lambda x: esmoe.es_int8_quant(x), dict(x=a), {}),
        "norm": (lambda g: esmoe.es_grad_norm([z(3), g]), dict(g=z(4)), {}),
        "clip": (lambda g, n, o: esmoe.es_clip_grad_norm([g], 1.0, norm=n, outputs=[o]), dict(g=z(4), n=z(())), dict(o=z(4))),
        "clip_in_place": (lambda g: esmoe.es_clip_grad_norm([g], 1.0), dict(g=z(4)), {}),
    }


@pytest.mark.parametrize("name", ["mm", "swiglu", "mm_backward", "swiglu_backward", "int8", "quant", "quant_new", "norm", "clip", "clip_in_place"])
def test_derivatives_are_refused(esmoe, name):
    """A result that would silently lack a gradient or a tangent, or a buffer that is part of a graph."""
    call, inputs, outputs = _autograd_calls(esmoe)[name]
    with torch.no_grad(), pytest.raises(RuntimeError, match=NO_GPU):
        call(**inputs, **outputs)
    for which in {**inputs, **outputs}:
        args = {**inputs, **outputs}
        args[which] = args[which].detach().requires_grad_()   # (of the same strides)
        with pytest.raises(RuntimeError, match="not differentiable by autograd" if which in inputs else "output that requires a gradient"):
            call(**args)
        with torch.no_grad(), pytest.raises(RuntimeError, match=NO_GPU):
            call(**args)
        with fwd.dual_level():
            args[which] = fwd.make_dual({**inputs, **outputs}[which], torch.ones_like({**inputs, **outputs}[which]))
            with torch.no_grad(), pytest.raises(RuntimeError, match="tangent"):
                call(**args)


# ---------------------------------------------------------------------------- C ABI
def _memory():
    buf = (ctypes.c_char * 4096)()
    base = ctypes.addressof(buf)
    base += -base % 16
    return buf, ctypes.c_void_p(base), ctypes.c_void_p(base + 8)


def test_c_abi(esmoe):
    from expert_specialization_moe_amd import _native

    lib = _native.lib
    buf, p, odd = _memory()
    none = None

    def bad(rc, what, code=-1):
        assert rc == code and what in _native.last_error(), (rc, _native.last_error())

    mm = lambda out=p, dtype=0, a=p, b=p, ps=p, eo=p, e=2, rows=5, n=32, k=48, swiglu=0, gu=none: lib.esmoe_grouped_mm(
        out, dtype, a, b, ps, eo, e, rows, n, k, swiglu, gu, none)
    bad(mm(dtype=2), "dtype")
    bad(mm(e=0), "num_experts")
    bad(mm(e=1025), "num_experts")
    bad(mm(rows=-1), "total_rows")
    bad(mm(n=36), "n must be")
    bad(mm(n=24, swiglu=1), "n must be")
    bad(mm(k=0), "k must be")
    bad(mm(k=(1 << 20) + 8), "k must be")
    bad(mm(gu=p), "gate_up goes with swiglu")
    for name in ("out", "a", "b", "ps", "eo"):
        bad(mm(**{name: none}), "null")
    for name in ("out", "a", "b"):
        bad(mm(**{name: odd}), "16-byte")
    bad(mm(gu=odd, swiglu=1), "16-byte")
    assert mm(rows=0) == 0
    back = lambda d=p, dtype=0, a=p, b=p, ps=p, eo=p, e=2, rows=5, n=32, k=48, ga=p, gb=p: lib.esmoe_grouped_mm_backward(
        d, dtype, a, b, ps, eo, e, rows, n, k, ga, gb, none)
    bad(back(n=4), "n must be")
    for name in ("d", "a", "b", "ps", "eo"):
        bad(back(**{name: none}), "null")
    for name in ("d", "a", "b", "ga", "gb"):
        bad(back(**{name: odd}), "16-byte")
    assert back(ga=none, gb=none) == 0 and back(ga=p, gb=none, rows=0) == 0
    sw = lambda d=p, gu=p, dtype=0, rows=5, inter=16, out=p: lib.esmoe_swiglu_backward(d, gu, dtype, rows, inter, out, none)
    bad(sw(dtype=3), "dtype")
    bad(sw(inter=12), "inter")
    bad(sw(rows=-1), "total_rows")
    bad(sw(gu=none), "null")
    bad(sw(out=odd), "16-byte")
    assert sw(rows=0) == 0
    i8 = lambda out=p, dtype=0, a=p, b=p, sa=p, sb=p, rows=5, n=32, k=48: lib.esmoe_int8_grouped_mm(out, dtype, a, b, sa, sb, p, p, 2, rows, n, k, 0, none)
    bad(i8(k=56), "k must be")
    bad(i8(k=65552), "k must be")
    bad(i8(sa=none), "null")
    bad(i8(a=odd), "16-byte")
    assert i8(rows=0) == 0
    q = lambda x=p, dtype=0, o=p, s=p, rows=2, k=32: lib.esmoe_int8_quant(x, dtype, o, s, rows, k, none)
    bad(q(dtype=2), "in_dtype")
    bad(q(k=24), "k must be")
    bad(q(rows=-1), "total_rows")
    bad(q(s=none), "null")
    bad(q(o=odd), "16-byte")
    assert q(rows=0) == 0


def test_c_abi_of_the_norm(esmoe):
    from expert_specialization_moe_amd import _native

    lib = _native.lib
    buf, p, odd = _memory()
    assert lib.esmoe_grad_norm_workspace_bytes(1) >= 8 * 2048
    big = lib.esmoe_grad_norm_workspace_bytes(2)

    def clip(ptrs=(p.value, p.value + 64), outs=(p.value, p.value + 64), types=(0, 2), sizes=(5, 6), count=2, max_norm=1.0, eps=0.0, ws=p, nbytes=big,
             which="clip"):
        arr = lambda t, v: (t * max(len(v), 1))(*v)
        ins, o, ty, sz = arr(ctypes.c_void_p, ptrs), arr(ctypes.c_void_p, outs), arr(ctypes.c_int, types), arr(ctypes.c_long, sizes)
        if which == "norm":
            return lib.esmoe_grad_norm(ins, ty, sz, count, p, ws, nbytes, None)
        return lib.esmoe_clip_grad_norm(ins, o, ty, sz, count, max_norm, eps, None, p, ws, nbytes, None)

    def bad(rc, what, code=-1):
        assert rc == code and what in _native.last_error(), (rc, _native.last_error())

    for which in ("clip", "norm"):
        bad(clip(types=(0, 3), which=which), "ESMOE_GRAD")
        bad(clip(sizes=(5, -1), which=which), "2^40")
        bad(clip(sizes=(1 << 40, 1), which=which), "2^40")
        bad(clip(ptrs=(p.value, None), which=which), "null")
        bad(clip(ptrs=(p.value, p.value + 66), which=which), "aligned")
        bad(clip(nbytes=big - 1, which=which), "workspace", -2)
        bad(clip(ws=None, which=which), "workspace", -2)
        bad(clip(count=-1, which=which), "count")
    bad(clip(outs=(p.value, None)), "null")
    bad(clip(outs=(p.value + 1, p.value)), "aligned")
    bad(clip(max_norm=-1.0), "max_norm")
    bad(clip(max_norm=float("nan")), "max_norm")
    bad(clip(eps=float("inf")), "eps")
