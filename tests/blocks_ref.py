"""The block operators' definitions (include/gpann_blocks.h) in binary64 on the CPU, row by row, with bounds of what the kernels may differ by.

Bounds.  u = half a step of the tensors' type (bf16 2^-8, fp16 2^-11), e = 2^-24.  A logit is a sum of d products in binary32, any order: off by at most
d * e * a with a = |scale| * sum |q_i k_i|, and by two more roundings; a weight p = 2^(x log2 e - max) is then off by p * w with w = 2 (d + 4) e max a + 8 e
(exponential and its argument), and the normalising sum and the log-sum-exp by the same plus n e.  The kernels round every p (and ds) once to the tensors'
type, u p; the second products add n products in binary32, n e; the result is rounded once, u |out|."""
import math

import numpy as np

U = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11}
E = 2.0 ** -24


def visible(n, m, t, causal):
    return 0 if t >= m else (min(max(n - m + t + 1, 0), n) if causal else n)


def rows_of(probes, bs, nblk, vis, pages=None):
    """cache rows a query row looks at: the visible rows of its probed blocks, each once, ascending"""
    out = []
    for p in sorted({int(p) for p in probes}):
        if 0 <= p < nblk and p * bs < vis and (pages is None or pages[p]):
            out.extend(range(p * bs, min((p + 1) * bs, vis)))
    return np.asarray(out, np.int64)


def softmax_rows(q, k, scale):
    """x, lse, p, and the relative bound of p, for q [g][d], k [r][d]"""
    x = scale * (q @ k.T)
    a = abs(scale) * (np.abs(q) @ np.abs(k).T)
    with np.errstate(invalid="ignore"):
        top = x.max(1, keepdims=True)
        lse = np.log(np.exp(x - top).sum(1, keepdims=True)) + top
        p = np.exp(x - lse)
    w = 2 * (q.shape[1] + 4) * E * a.max() + 8 * E + k.shape[0] * E
    return lse[:, 0], p, w


def attend(q, k, v, probes, bs, nblk, vis, scale, dtype, pages=None):
    """one query row's heads of a group: out [g][d], lse [g], their bounds"""
    u = U[dtype]
    rows = rows_of(probes, bs, nblk, vis, pages)
    if len(rows) == 0:
        return np.zeros_like(q), np.full(q.shape[0], -np.inf), np.zeros_like(q), np.zeros(q.shape[0])
    lse, p, w = softmax_rows(q, k[rows], scale)
    out = p @ v[rows]
    bound = (u + 2 * w + len(rows) * E) * (p @ np.abs(v[rows]))
    return out, lse, bound + u * (np.abs(out) + bound), 2 * w + 4 * E * np.abs(lse)


def backward(q, k, v, dout, probes, bs, nblk, vis, scale, dtype):
    """one query row's heads of a group: rows, dq, contributions to dk and dv of those rows, and bounds (without the rounding of the results)"""
    u = U[dtype]
    rows = rows_of(probes, bs, nblk, vis)
    if len(rows) == 0:
        return rows, np.zeros_like(q), None, None, np.zeros_like(q), None, None
    kk, vv = k[rows], v[rows]
    lse, p, w = softmax_rows(q, kk, scale)
    w = 3 * w + 4 * E * np.abs(lse).max()                 # the weights come from the stored log-sum-exp
    out = p @ vv
    out_err = (2 * u + 2 * w + len(rows) * E) * (p @ np.abs(vv)) + u * np.abs(out)       # of the forward's out, as attend()
    dp = dout @ vv.T
    delta = (dout * out).sum(1, keepdims=True)
    ds = p * (dp - delta)
    d = q.shape[1]
    dp_err = (d + 2) * E * (np.abs(dout) @ np.abs(vv).T) + (np.abs(dout) * out_err).sum(1, keepdims=True) + (d + 2) * E * (np.abs(dout) * np.abs(out)).sum(1, keepdims=True)
    ds_err = p * (1 + w) * dp_err + (w + u + 2 * E) * np.abs(ds)
    n = len(rows)
    dq, dq_err = scale * (ds @ kk), abs(scale) * ((ds_err + n * E * np.abs(ds)) @ np.abs(kk))
    dk, dk_err = scale * (ds.T @ q), abs(scale) * (ds_err.T @ np.abs(q))
    dv, dv_err = p.T @ dout, ((w + u) * p).T @ np.abs(dout)
    return rows, dq, dk, dv, dq_err, dk_err, dv_err


def summarize(k, n, bs):
    """[blocks][d] centroids of one head: binary64 sums of 16-bit numbers are exact, one division, one rounding"""
    nb = -(-n // bs)
    return np.stack([k[j * bs:min(n, (j + 1) * bs)].sum(0) / (min(n, (j + 1) * bs) - j * bs) for j in range(nb)]).astype(np.float32) if nb else np.zeros((0, k.shape[1]), np.float32)


def route(q, centroids, bs, vis, nprobe, first, last):
    """probes of one query row: q [g][d] of a group, centroids float32"""
    nb = -(-vis // bs)
    score = centroids[:nb].astype(np.float64) @ q.astype(np.float64).sum(0)
    order = sorted(range(nb), key=lambda j: (0 if j < first or j >= nb - last else 1, math.inf if math.isnan(score[j]) else -score[j], j))
    probes = sorted(order[:nprobe])
    return np.asarray(probes + [-1] * (nprobe - len(probes)), np.int32)


def evict(mass, n, keep, first, last):
    if n <= keep:
        return list(range(n))
    order = sorted(range(n), key=lambda j: (0 if j < first or j >= n - last else 1, math.inf if math.isnan(mass[j]) else -mass[j], j))
    return sorted(order[:keep])
