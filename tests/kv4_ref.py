"""float64 restatements of the 4-bit cache's operators, of the sampler's
distribution and of draft verification, written from their definitions
(include/qora_cuda.h) for the tests: loops over rows and heads."""
import math

import numpy as np

EPS = 1e-6


def quantise(x):
    """(codes, scales) of rows x [..][D] (float32) in groups of 32."""
    x = np.asarray(x, np.float32).astype(np.float64)
    g = x.reshape(*x.shape[:-1], -1, 32)
    amax = np.abs(g).max(-1)
    with np.errstate(over="ignore", invalid="ignore"):
        s = np.minimum((amax / 7).astype(np.float32), np.float32(65504)).astype(np.float16)
    s = np.where(np.isfinite(amax), s, np.float16(np.nan))
    sd = s.astype(np.float64)[..., None]
    with np.errstate(divide="ignore", invalid="ignore"):
        c = np.where(sd > 0, np.clip(np.rint(g / sd), -7, 7), 0.0)
    return c, s


def held(x):
    """What rows x stand for in the cache, float32."""
    c, s = quantise(x)
    return (c * s.astype(np.float64)[..., None]).astype(np.float32).reshape(np.shape(x))


def norm_rope(x, gamma_f16, cos, sin):
    """x [D] float32 -> normed and rotated, float64."""
    x = np.asarray(x, np.float64)
    h = x.size // 2
    x = x / math.sqrt(float((x * x).mean()) + EPS) * np.asarray(gamma_f16, np.float16).astype(np.float64)
    c, s = np.asarray(cos, np.float64), np.asarray(sin, np.float64)
    return np.concatenate([x[:h] * c - x[h:] * s, x[h:] * c + x[:h] * s])


def append(qkv, heads, kvh, hd, qn, kn, cos, sin, positions):
    """Rows [n][(heads + 2 kvh) hd] -> q float64, k and v float32 as held."""
    n = qkv.shape[0]
    x = qkv.reshape(n, heads + 2 * kvh, hd)
    q = np.zeros((n, heads, hd))
    k = np.zeros((n, kvh, hd), np.float32)
    for i in range(n):
        c, s = cos[positions[i]], sin[positions[i]]
        for h in range(heads):
            q[i, h] = norm_rope(x[i, h], qn, c, s)
        for h in range(kvh):
            k[i, h] = norm_rope(x[i, heads + h], kn, c, s)
    return q.reshape(n, -1), held(k).reshape(n, -1), held(x[:, heads + kvh:]).reshape(n, -1)


def attend(q, k, v, length, heads, kvh):
    """New tokens q [n][heads][hd] over k, v [length + n][kvh][hd]: (out, bound)
    in float64.  The bound is the error that the kernel's arithmetic can make:
    a score is off by 2^-20 of its sum of magnitudes at most (queries as f16
    pairs 2^-22, the products' accumulation, four scale groups in f32), which
    moves a probability by twice that, and a probability's own exponential,
    split and sums by 2^-19 with 2^-24 for every 32 positions folded."""
    n, _, hd = q.shape
    q, k, v = (np.asarray(t, np.float64) for t in (q, k, v))
    out = np.zeros((n, heads, hd))
    bound = np.zeros((n, heads, 1))
    with np.errstate(invalid="ignore"):
        for h in range(heads):
            kk, vv = k[:, h * kvh // heads], v[:, h * kvh // heads]
            for i in range(n):
                m = length + i + 1
                s = kk[:m] @ q[i, h] / math.sqrt(hd)
                p = np.exp(s - s.max())
                p /= p.sum()
                out[i, h] = p @ vv[:m]
                size = (np.abs(kk[:m]) @ np.abs(q[i, h]) / math.sqrt(hd)).max()
                bound[i, h] = (2 * 2.0 ** -20 * size + 2.0 ** -19 + m / 32 * 2.0 ** -24) * np.abs(vv[:m]).max()
    return out, bound


def reserve(table, lens, counts, page, pool, max_pos, max_tokens):
    """(table, slots, positions, offsets) or None when refused."""
    table, S = np.array(table), len(lens)
    keep = [-(-int(n) // page) for n in lens]
    used = {int(table[b, j]) for b in range(S) for j in range(keep[b])}
    free = [p for p in range(pool) if p not in used]
    slots, positions = np.full(max_tokens, -1, np.int32), np.zeros(max_tokens, np.int32)
    offsets = np.zeros(S + 1, np.int32)
    if any(lens[b] + counts[b] > max_pos or counts[b] < 0 for b in range(S)) or sum(counts) > max_tokens:
        return None
    if sum(-(-(int(lens[b]) + int(counts[b])) // page) - keep[b] for b in range(S)) > len(free):
        return None
    at = i = 0
    for b in range(S):
        for j in range(keep[b], -(-(int(lens[b]) + int(counts[b])) // page)):
            table[b, j] = free[at]
            at += 1
        for p in range(int(lens[b]), int(lens[b]) + int(counts[b])):
            slots[i], positions[i] = table[b, p // page] * page + p % page, p
            i += 1
        offsets[b + 1] = i
    return table, slots, positions, offsets


def probs(x, prev, temperature, top_k, top_p, penalty):
    """sample_token's distribution of one row, float64."""
    x = np.asarray(x, np.float64).copy()
    temperature, top_p, penalty = (float(np.float32(t)) for t in (temperature, top_p, penalty))
    if prev is not None and penalty != 1.0:
        for t in prev:
            if 0 <= t < x.size:
                x[t] = x[t] / penalty if x[t] > 0 else x[t] * penalty
    z = x / (temperature if temperature > 0 else 1.0)
    order = sorted(range(x.size), key=lambda i: (-x[i], i))
    cut = 0 < top_k < x.size
    kept = order[:top_k] if cut else order
    e = np.exp(z[kept] - z.max())
    p = e / e.sum()
    if cut and 0 < top_p < 1:
        stay = np.cumsum(p) - p < top_p
        p = np.where(stay, p, 0)
        p /= p.sum()
    out = np.zeros(x.size)
    out[kept] = p
    return out


def verify(drafts, q, p, u, count):
    """One stream: tokens of the step (accepted drafts and the drawn one)."""
    K = len(u) - 1
    V = p.shape[1]
    out = []
    for i in range(count):
        d = int(drafts[i])
        ok = 0 <= d < V and float(u[i]) * (float(q[i, d]) if q is not None else 1.0) < float(p[i, d])
        if not ok:
            w = p[i].astype(np.float64)
            if q is not None:
                w = w - q[i].astype(np.float64)
            elif 0 <= d < V:
                w[d] = 0
            w = np.where(w > 0, w, 0)
            if not w.sum() > 0:
                w = p[i].astype(np.float64)
            break
        out.append(d)
    else:
        w = p[count].astype(np.float64)
    w = np.where(w > 0, w, 0)
    goal = max(float(u[K]), 0.0) * w.sum()
    over = np.nonzero(np.cumsum(w) > goal)[0]
    pos = np.nonzero(w > 0)[0]
    out.append(int(over[0]) if over.size else int(pos[-1]) if pos.size else 0)
    return out
