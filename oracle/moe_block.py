"""Plain 64-bit restatement of the operators around the grouped GEMMs: router gating, the weighted way back from the experts, the
residual norm with 1x128 quantisation, products with 4-bit weights.  Test infrastructure; numpy on the host, one token or expert at a time."""
import numpy as np

F32 = np.float32


def scores(x, scoring):
    """softmax or sigmoid of one token's logits, in 64 bits."""
    x = np.asarray(x, np.float64)
    with np.errstate(over="ignore", invalid="ignore"):
        if scoring == "sigmoid":
            return 1.0 / (1.0 + np.exp(-x))
        if np.isneginf(x).all():
            return np.zeros_like(x)
        e = np.exp(x - x.max())   # (max is NaN where there is one)
        return e / e.sum()


def _rank(values):
    """Indexes by falling value: NaN first, ties to the lower index."""
    return sorted(range(len(values)), key=lambda i: (0, 0.0, i) if np.isnan(values[i]) else (1, -float(values[i]), i))


def topk_gating(logits, topk, bias=None, scoring="softmax", renormalize=True, scale=1.0, groups=1, topk_groups=1):
    logits = np.asarray(logits, np.float64)
    t, e = logits.shape
    ids, weights = np.full((t, topk), -1, np.int32), np.zeros((t, topk))
    for i, x in enumerate(logits):
        s = scores(x, scoring)
        with np.errstate(invalid="ignore"):
            if bias is None and groups == 1:
                choice = x
            else:
                choice = (s if bias is None else s + np.asarray(bias, np.float64)).astype(F32)
            out = np.isneginf(x) | np.isneginf(choice)
            if groups > 1:
                width, score = e // groups, []
                for g in range(groups):
                    c = choice[g * width:(g + 1) * width][~out[g * width:(g + 1) * width]]
                    best = c[[j for j in _rank(c)[:2]]]
                    score.append(best.sum(dtype=F32) if best.size else None)
                have = [g for g in range(groups) if score[g] is not None]
                kept = [have[j] for j in _rank([score[g] for g in have])[:topk_groups]]
                out = out | ~np.isin(np.arange(e) // width, kept)
        left = np.flatnonzero(~out)
        chosen = [left[j] for j in _rank(choice[left])[:topk]]
        ids[i, :len(chosen)] = chosen
        weights[i, :len(chosen)] = _weights(x, chosen, s, scoring, renormalize) * scale
    return ids, weights


def _weights(x, chosen, s, scoring, renormalize):
    """The chosen experts' scores; renormalised from their logarithms, so that no sum is 0."""
    if not renormalize or not len(chosen):
        return s[chosen]
    with np.errstate(over="ignore", invalid="ignore"):
        log = x[chosen] if scoring == "softmax" else -np.logaddexp(0.0, -x[chosen])
        v = np.exp(log - log.max())
        return v / v.sum()


def gating_weights(logits, ids, scoring, renormalize, scale):
    """Weights of given ids (what a gradient is the derivative of); 0 for an id outside the experts."""
    logits = np.asarray(logits, np.float64)
    w = np.zeros(ids.shape)
    for i, x in enumerate(logits):
        real = (ids[i] >= 0) & (ids[i] < x.size)
        w[i, real] = _weights(x, ids[i][real], scores(x, scoring), scoring, renormalize) * scale
    return w


def gating_grad(grad, logits, ids, scoring, renormalize, scale):
    """d(sum of grad * weights) / d logits by the chain rule over the scores' logarithms: dw_j = w_j (dlog s_j - sum_i w'_i dlog s_i)."""
    logits = np.asarray(logits, np.float64)
    t, e = logits.shape
    out = np.zeros((t, e))
    for i, x in enumerate(logits):
        real = (ids[i] >= 0) & (ids[i] < e)
        at, g = ids[i][real], np.asarray(grad, np.float64)[i][real]
        if not at.size:
            continue
        s = scores(x, scoring)
        w = _weights(x, at, s, scoring, renormalize) * scale
        gw = g * w
        if renormalize:
            gw = gw - w / scale * gw.sum() if scale else gw
        dlog = np.zeros(e)           # d(loss) / d(log s_e)
        np.add.at(dlog, at, gw)
        with np.errstate(over="ignore"):
            # (renormalised, the softmax's own sum drops out: dlog adds up to 0)
            out[i] = dlog / (1.0 + np.exp(x)) if scoring == "sigmoid" else dlog if renormalize else dlog - s * dlog.sum()
        out[i][np.isneginf(x)] = 0.0
    return out


def combine(rows, dst, topk, weights=None):
    """-> (out, sum of |terms|), both 64 bits."""
    rows = np.asarray(rows, np.float64)
    dst = np.asarray(dst).reshape(-1, topk)
    w = np.ones(dst.shape) if weights is None else np.asarray(weights, np.float64).reshape(dst.shape)
    out, mag = np.zeros((dst.shape[0], rows.shape[1])), np.zeros((dst.shape[0], rows.shape[1]))
    for t in range(dst.shape[0]):
        for j in range(topk):
            if 0 <= dst[t, j] < rows.shape[0]:
                out[t] += w[t, j] * rows[dst[t, j]]
                mag[t] += np.abs(w[t, j] * rows[dst[t, j]])
    return out, mag


def combine_grad(grad_out, rows, dst, topk, weights):
    """-> (grad_rows with NaN where no pair points, grad_weights, sum of |terms| of grad_weights)."""
    rows, grad_out = np.asarray(rows, np.float64), np.asarray(grad_out, np.float64)
    dst = np.asarray(dst).reshape(-1, topk)
    w = np.asarray(weights, np.float64).reshape(dst.shape)
    grad_rows, grad_w, mag = np.full(rows.shape, np.nan), np.zeros(dst.shape), np.zeros(dst.shape)
    for t in range(dst.shape[0]):
        for j in range(topk):
            r = dst[t, j]
            if 0 <= r < rows.shape[0]:
                grad_rows[r] = w[t, j] * grad_out[t]
                grad_w[t, j] = grad_out[t] @ rows[r]
                mag[t, j] = np.abs(grad_out[t]) @ np.abs(rows[r])
    return grad_rows, grad_w, mag


def rms_norm(h, weight, eps):
    h = np.asarray(h, np.float64)
    return h / np.sqrt((h * h).mean(axis=1, keepdims=True) + eps) * np.asarray(weight, np.float64)


def block_scales(y):
    """fp32-representable scale of every 1x128 block of y, from 64 bits: max(|y|, 1e-4) / 448."""
    b = np.abs(y).reshape(y.shape[0], -1, 128).max(axis=2)
    return np.maximum(b, float(F32(1e-4))) / 448.0


E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0])


def dequant_mxfp4(b, sf):
    """codes [..., K/2] and E8M0 bytes [..., K/32] -> float64 [..., K]."""
    b, sf = np.asarray(b, np.uint8), np.asarray(sf, np.int64)
    v = np.stack([E2M1[b & 15], E2M1[b >> 4]], axis=-1).reshape(*b.shape[:-1], -1, 32)
    scale = np.where(sf == 255, np.nan, np.ldexp(1.0, np.where(sf == 255, 0, sf - 127)))
    return (v * scale[..., None]).reshape(*b.shape[:-1], -1)


def mxfp4_mm(a, b, sf, rows, offsets):
    """-> (product [total, N], sum of |terms|); rows of no expert NaN."""
    a = np.asarray(a, np.float64)
    n = b.shape[1]
    out, mag = np.full((a.shape[0], n), np.nan), np.full((a.shape[0], n), np.nan)
    for e, (m, off) in enumerate(zip(rows, offsets)):
        if m > 0:
            w = dequant_mxfp4(b[e], sf[e])
            out[off:off + m] = a[off:off + m] @ w.T
            mag[off:off + m] = np.abs(a[off:off + m]) @ np.abs(w).T
    return out, mag


def swiglu(gate, up):
    with np.errstate(over="ignore"):
        return gate / (1.0 + np.exp(-gate)) * up
