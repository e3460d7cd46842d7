"""A training step of a mixture-of-experts layer out of the library's operators: gating, routing, the experts with SwiGLU, combine, all gradients
back to the tokens, the logits and the weights, and their clipping.

Against the same layer in 64 bits through autograd, the chosen experts held.  Every stage rounds to 16 bits, half a step of the value (fp16
2^-11, bf16 2^-8).  On the longest way, loss to token, there are six: gate_up, then the gradients of y, h, gate_up, the packed rows and the
tokens.  A product of independent terms passes on its factors' errors relative to its norm, and so does SwiGLU's gradient, whose slope in the gate
is at most three times as large relative to its norm: any gradient's norm is off by at most eight halves of a step if all errors agree."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


class Layer:
    def __init__(self, tokens, experts, topk, hidden, inter, dtype, seed, first=0, share=None):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        rand = lambda *s: torch.randn(s, generator=gen, device="cuda")
        self.topk, self.first, self.share = topk, first, share or experts
        self.x, self.d = rand(tokens, hidden).to(dtype), rand(tokens, hidden).to(dtype)
        self.logits = rand(tokens, experts).to(dtype)
        self.w13 = (rand(self.share, 2 * inter, hidden) / hidden ** 0.5).to(dtype)
        self.w2 = (rand(self.share, hidden, inter) / inter ** 0.5).to(dtype)

    def step(self, es, max_norm=1e9):
        """-> the output, then the gradients of the tokens, the logits, w13 and w2, clipped together."""
        (tokens, hidden), inter, e = self.x.shape, self.w2.size(2), self.share
        ids, weights = es.es_topk_gating(self.logits, self.topk)
        ps13, offsets, _, dst = es.es_route_metadata(ids, self.first, e, 2 * inter, hidden)
        ps2 = ps13.clone()
        ps2[:, 1], ps2[:, 2] = hidden, inter
        offsets = offsets[:e]
        # (as many rows as there can be: what no expert of the share has stays zero)
        rows = torch.zeros((tokens * self.topk, hidden), dtype=self.x.dtype, device="cuda")
        es.es_permute_rows(self.x, dst, self.topk, rows)
        h, gate_up, y = rows.new_zeros((rows.size(0), inter)), rows.new_zeros((rows.size(0), 2 * inter)), torch.zeros_like(rows)
        b13, b2 = self.w13.transpose(1, 2), self.w2.transpose(1, 2)
        es.es_grouped_mm_swiglu(h, rows, b13, ps13, offsets, gate_up=gate_up)
        es.es_grouped_mm(y, h, b2, ps2, offsets)
        out = es.es_combine_rows(y, dst, self.topk, weights)

        grad_y, grad_weights = es.es_combine_rows_backward(self.d, y, dst, self.topk, weights)
        grad_h, grad_w2 = es.es_grouped_mm_backward(grad_y, h, b2, ps2, offsets)
        grad_rows, grad_w13 = es.es_grouped_mm_swiglu_backward(grad_h, rows, b13, gate_up, ps13, offsets)
        grad_x = es.es_combine_rows(grad_rows, dst, self.topk)
        grad_logits = es.es_topk_gating_backward(grad_weights, self.logits, ids)
        self.ids = ids
        grads = [grad_x, grad_logits, grad_w13.transpose(1, 2), grad_w2.transpose(1, 2)]
        self.norm = es.es_clip_grad_norm(grads, max_norm)
        return [out] + grads

    def exact(self):
        x, logits, w13, w2 = (t.double().requires_grad_() for t in (self.x, self.logits, self.w13, self.w2))
        scores = torch.softmax(logits, dim=1).gather(1, self.ids.long())
        weights = scores / scores.sum(1, keepdim=True)
        out = torch.zeros_like(x)
        for e in range(self.share):
            at, place = (self.ids == e + self.first).nonzero(as_tuple=True)
            gate, up = (x[at] @ w13[e].t()).chunk(2, dim=1)
            out = out.index_add(0, at, (gate * torch.sigmoid(gate) * up) @ w2[e].t() * weights[at, place, None])
        (out * self.d.double()).sum().backward()
        return [out.detach(), x.grad, logits.grad, w13.grad, w2.grad]


CASES = [(50, 8, 2, 64, 48), (1, 4, 4, 128, 40), (300, 16, 4, 264, 136), (700, 6, 3, 512, 264)]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_a_training_step(esmoe, case, dtype):
    layer = Layer(*case, dtype, 1)
    got = layer.step(esmoe)
    half = torch.finfo(dtype).eps / 2
    for name, g, w in zip(("output", "tokens", "logits", "w13", "w2"), got, layer.exact()):
        assert float((g.double() - w).norm()) <= 8 * half * float(w.norm()), name


def test_a_share_of_the_experts(esmoe):
    """Experts 3 to 7 of 16, as a rank has them."""
    layer = Layer(200, 16, 4, 128, 72, HF, 2, first=3, share=5)
    for name, g, w in zip(("output", "tokens", "logits", "w13", "w2"), layer.step(esmoe), layer.exact()):
        assert float((g.double() - w).norm()) <= 8 * 2.0 ** -11 * float(w.norm()), name


def test_clipped_together(esmoe):
    layer = Layer(50, 8, 2, 64, 48, BF, 3)
    free = layer.step(esmoe)[1:]
    norm = float(layer.norm)
    assert abs(norm - float(sum((g.double() ** 2).sum() for g in free)) ** 0.5) <= 2.0 ** -23 * norm
    clipped = layer.step(esmoe, max_norm=norm / 8)[1:]
    for c, f in zip(clipped, free):   # (eps takes 1e-6 of `norm` at most; an eighth of a number is exact)
        assert ((c.double() - f.double() / 8).abs() <= (2.0 ** -8 + 2.0 ** -22 + 1e-6 / norm) * f.double().abs() / 8).all()


def test_a_step_captured_and_replayed(esmoe):
    """The forward, its gradients and the clipping in one graph: each replay as the eager step on the same values."""
    layer = Layer(120, 8, 2, 128, 72, BF, 4)
    layer.step(esmoe, 1.0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = layer.step(esmoe, 1.0)
    for i in range(4):
        layer.x.copy_(torch.randn(layer.x.shape, device="cuda"))
        layer.d.copy_(torch.randn(layer.d.shape, device="cuda"))
        layer.logits.copy_(torch.randn(layer.logits.shape, device="cuda"))
        want = [t.clone() for t in layer.step(esmoe, 1.0)]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(g, w) for g, w in zip(got, want)), i


def test_two_steps_at_once(esmoe):
    """On two streams, and as two graphs replayed side by side: no call has anything of another's."""
    layers = [Layer(400, 8, 2, 256, 136, BF, 5), Layer(30, 16, 4, 512, 264, HF, 6)]
    want = [[t.clone() for t in l.step(esmoe, 1.0)] for l in layers]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in layers]
    got = [None] * 2
    for _ in range(5):
        for i, (l, s) in enumerate(zip(layers, streams)):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got[i] = l.step(esmoe, 1.0)
        torch.cuda.synchronize()
        assert all(torch.equal(g, w) for a, b in zip(got, want) for g, w in zip(a, b))
    graphs = []
    for i, l in enumerate(layers):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            got[i] = l.step(esmoe, 1.0)
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(g, w) for a, b in zip(got, want) for g, w in zip(a, b))
