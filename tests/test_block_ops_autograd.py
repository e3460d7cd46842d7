"""The operators around the grouped GEMMs are not part of autograd: a call whose result would silently lack a gradient or a tangent, or
whose output buffer is part of a graph, is refused before anything else happens."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

BF = torch.bfloat16


def _calls(esmoe):
    """name -> (call, tensors that carry derivatives, buffers that are written)."""
    g = torch.zeros
    ids, dst = g(3, 4, dtype=torch.int32), g(8, dtype=torch.int32)
    e, n, k, rows = 2, 64, 256, 5
    b, sfb = g(e, n, k // 2, dtype=torch.uint8).transpose(1, 2), g(e, n, k // 32, dtype=torch.uint8).transpose(1, 2)
    ps, eo = torch.tensor([[3, n, k], [2, n, k]], dtype=torch.int32), torch.tensor([0, 3], dtype=torch.int32)
    norm = lambda x, w, r, **out: esmoe.es_add_rms_norm_quant_1x128(x, w, 1e-6, r, **out)
    norm_in = dict(x=g(3, 256, dtype=BF), w=g(256, dtype=BF), r=g(3, 256, dtype=BF))
    back_in = dict(grad=g(4, 16, dtype=BF), y=g(6, 16, dtype=BF), w=g(4, 2))
    return {
        "gating": (lambda x, b: esmoe.es_topk_gating(x, 4, b), dict(x=g(3, 16), b=g(16)), {}),
        "gating_backward": (lambda gw, x: esmoe.es_topk_gating_backward(gw, x, ids), dict(gw=g(3, 4), x=g(3, 16)), {}),
        "combine_new": (lambda y, w: esmoe.es_combine_rows(y, dst, 2, w), dict(y=g(6, 16, dtype=BF), w=g(4, 2)), {}),
        "combine": (lambda y, w, output: esmoe.es_combine_rows(y, dst, 2, w, output), dict(y=g(6, 16, dtype=BF), w=g(4, 2)),
                    dict(output=g(4, 16, dtype=BF))),
        "combine_backward": (lambda grad, y, w, gi, gw: esmoe.es_combine_rows_backward(grad, y, dst, 2, w, gi, gw), back_in,
                             dict(gi=g(6, 16, dtype=BF), gw=g(4, 2))),
        "norm_new": (lambda x, w, r: norm(x, w, r, return_normed=True), norm_in, {}),
        "norm": (norm, norm_in, dict(residual_out=g(3, 256, dtype=BF), normed=g(3, 256, dtype=BF), scales=g(3, 2))),
        "mxfp4": (lambda a, output: esmoe.es_mxfp4_grouped_mm(output, a, b, sfb, ps, eo), dict(a=g(rows, k, dtype=BF)),
                  dict(output=g(rows, n, dtype=BF))),
        "mxfp4_swiglu": (lambda a, output: esmoe.es_mxfp4_grouped_mm_swiglu(output, a, b, sfb, ps, eo), dict(a=g(rows, k, dtype=BF)),
                         dict(output=g(rows, n // 2, dtype=BF))),
    }


NAMES = ["gating", "gating_backward", "combine_new", "combine", "combine_backward", "norm_new", "norm", "mxfp4", "mxfp4_swiglu"]


@pytest.mark.parametrize("name", NAMES)
def test_tangents_are_refused(esmoe, name):
    """With gradients recorded and without: no_grad leaves the forward mode on."""
    call, inputs, outputs = _calls(esmoe)[name]
    with torch.no_grad(), pytest.raises(RuntimeError, match="no CPU implementation"):
        call(**inputs, **outputs)
    for which in {**inputs, **outputs}:
        with fwd.dual_level():
            args = {**inputs, **outputs}
            args[which] = fwd.make_dual(args[which], torch.ones_like(args[which]))
            with pytest.raises(RuntimeError, match="tangent"):
                call(**args)
            with torch.no_grad(), pytest.raises(RuntimeError, match="tangent"):
                call(**args)


@pytest.mark.parametrize("name", ["combine", "combine_backward", "norm", "mxfp4", "mxfp4_swiglu"])
def test_outputs_that_require_a_gradient_are_refused(esmoe, name):
    """A buffer of a graph that is overwritten would give that graph's backward pass other values, or none."""
    call, inputs, outputs = _calls(esmoe)[name]
    for which in outputs:
        leaf = outputs[which].clone().requires_grad_()
        for buffer in (leaf, leaf * 2):
            args = dict(inputs, **outputs)
            args[which] = buffer
            with pytest.raises(RuntimeError, match="output that requires a gradient"):
                call(**args)
            with torch.no_grad(), pytest.raises(RuntimeError, match="no CPU implementation"):
                call(**args)
