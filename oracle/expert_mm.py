"""Plain 64-bit restatement of the experts' products with their gradients, the int8 products and quantiser, and the clipping of gradients.
Test infrastructure: torch in float64, on whatever device the inputs are; one expert at a time.  Sums come with the sum of their terms'
magnitudes, which is what their rounding errors go by."""
import torch

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 1e-40, torch.float16: 2.0 ** -25, torch.float32: 1e-45}   # half the smallest number's step


def spans(rows, offsets, total):
    """(expert, first row, rows) of the experts that have any, cut at the tensor's rows."""
    for e, (m, off) in enumerate(zip(rows, offsets)):
        m = min(m, total - off) if 0 <= off < total else 0
        if m > 0:
            yield e, off, m


def offsets_of(rows):
    out, off = [], 0
    for m in rows:
        out.append(off)
        off += m
    return out


def grouped_mm(a, b, rows, offsets):
    """a [M, K], b [E, N, K] -> (out [M, N], magnitudes); NaN in rows of no expert."""
    a, b = a.double(), b.double()
    out = torch.full((a.size(0), b.size(1)), float("nan"), dtype=torch.float64, device=a.device)
    mag = out.clone()
    for e, off, m in spans(rows, offsets, a.size(0)):
        out[off:off + m] = a[off:off + m] @ b[e].t()
        mag[off:off + m] = a[off:off + m].abs() @ b[e].abs().t()
    return out, mag


def grouped_mm_grads(d, a, b, rows, offsets, d_err=None):
    """-> (grad_a, its magnitudes, its error from d's, grad_b, ...): d [M, N] with an error of at most d_err per element."""
    d, a, b = d.double(), a.double(), b.double()
    err = torch.zeros_like(d) if d_err is None else d_err
    ga = torch.full_like(a, float("nan"))
    ga_mag, ga_err, gb, gb_mag, gb_err = ga.clone(), ga.clone(), torch.zeros_like(b), torch.zeros_like(b), torch.zeros_like(b)
    for e, off, m in spans(rows, offsets, a.size(0)):
        at = slice(off, off + m)
        ga[at], ga_mag[at], ga_err[at] = d[at] @ b[e], d[at].abs() @ b[e].abs(), err[at] @ b[e].abs()
        gb[e], gb_mag[e], gb_err[e] = d[at].t() @ a[at], d[at].abs().t() @ a[at].abs(), err[at].t() @ a[at].abs()
    return ga, ga_mag, ga_err, gb, gb_mag, gb_err


def silu(x):
    return x * torch.sigmoid(x)


def swiglu(g, u):
    return silu(g) * u


def swiglu_grad(d, gate_up):
    """Gradient of silu(gate) * up by the formula: [M, 2 * inter]."""
    d = d.double()
    g, u = gate_up.double().chunk(2, dim=1)
    s = torch.sigmoid(g)
    return torch.cat([d * u * (s + g * s * torch.sigmoid(-g)), d * g * s], dim=1)


def int8_quant(x):
    """-> (q int8, scales float64)."""
    x = x.double()
    amax = x.abs().amax(dim=-1, keepdim=True)
    bad = ~torch.isfinite(amax)
    # torch.round takes ties to even; quotients of such short numbers that are no tie are far from one in 64 bits
    q = torch.round(x * 127.0 / torch.where(bad | (amax == 0), 1.0, amax))
    q = torch.where(bad | (amax == 0), 0.0, q).to(torch.int8)
    return q, torch.where(bad, float("nan"), amax / 127.0).squeeze(-1)


def clip(grads, max_norm, eps):
    """-> (norm, factor), floats."""
    norm = float(torch.sqrt(sum((g.double() ** 2).sum() for g in grads)))
    return norm, min(1.0, max_norm / (norm + eps))


def out_bound(want, err, dtype):
    """Largest distance of a result of `dtype` from `want` whose value before its rounding is off by err."""
    return err + HALF_STEP[dtype] * (want.abs() + err) + TINY[dtype]
