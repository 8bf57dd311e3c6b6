"""The quantised registry's definition in numpy and 64 bits: what vdb_registry_* is held to.
Cosines are f64; alternatives are ranked by the cosine rounded to f32, equal ones by the
lower slot."""
import numpy as np


def dim_pad(dim):
    return -(-dim // 64) * 64


def quantise(x, bits):
    """(w (n, dim) int64, group scales (n, ceil(dim / 32)) or None, scale f64 (n,) with NaN
    for rows that hold an infinity or a NaN). The quotients of f32 (or shorter) inputs are
    decided exactly: a f64 quotient next to a border is checked against it in integers by
    construction (both sides of 254 x = (2 w + 1) max have at most 24 + 8 bits)."""
    x = np.asarray(x, np.float64)
    bad = ~np.isfinite(x).all(1)
    x = np.where(bad[:, None], 0.0, x)
    n, dim = x.shape
    top = np.abs(x).max(1)
    safe = np.where(top > 0, top, 1.0)[:, None]
    if bits == 8:
        w, group = np.rint(127.0 * x / safe).astype(np.int64), None
    else:
        g = -(-dim // 32)
        p = np.zeros((n, g * 32))
        p[:, :dim] = x
        p = p.reshape(n, g, 32)
        s = np.ceil(127.0 * np.abs(p).max(2) / safe)
        c = np.rint(889.0 * p / (safe * np.where(s > 0, s, 1.0))[:, :, None])
        w = (c * s[:, :, None]).reshape(n, -1)[:, :dim].astype(np.int64)
        group = s.astype(np.uint8)
    sq = (w * w).sum(1)
    scale = np.where(sq > 0, 1.0 / np.sqrt(np.maximum(sq, 1)), 0.0)
    return w, group, np.where(bad, np.nan, scale)


def pack(w, group, bits):
    """The stored code bytes (n, dim_pad * bits / 8) of whole numbers w."""
    n, dim = w.shape
    d = dim_pad(dim)
    if bits == 8:
        out = np.full((n, d), 128, np.uint8)
        out[:, :dim] = w + 128
        return out
    s = np.repeat(group.astype(np.int64), 32, 1)[:, :dim]
    c = np.full((n, d), 8, np.uint32)
    c[:, :dim] = np.where(s > 0, w // np.maximum(s, 1), 0) + 8
    words = np.zeros((n, d // 8), np.uint32)
    for nib in range(8):
        words |= c[:, 2 * (nib % 4) + nib // 4::8] << np.uint32(4 * nib)
    return words.view(np.uint8).reshape(n, d // 2)


def cosines(q, w, scale):
    """f64 (n_q, n_rows): 0 where a side is all zero, -inf for empty rows, NaN for a query
    with an infinity or a NaN."""
    q = np.asarray(q, np.float64)
    bad = ~np.isfinite(q).all(1)
    q = np.where(bad[:, None], 0.0, q)
    den = np.linalg.norm(q, axis=1)[:, None] * np.sqrt((w * w).sum(1).astype(np.float64))[None]
    c = np.where(den > 0, (q @ w.T.astype(np.float64)) / np.where(den > 0, den, 1.0), 0.0)
    c[bad] = np.nan
    c[:, np.isnan(scale)] = -np.inf
    return c


def posterior(cos, labels, k, temperature, bad=None):
    """(log_prob, entropy, lse, index, alt_log_prob) in f64 from cosines(); `bad` marks the
    queries with an infinity or a NaN (all-empty cosines do not show them)."""
    m, n = cos.shape
    log_prob, entropy = np.full(m, -np.inf), np.zeros(m)
    lse = np.full(m, -np.inf)
    index, alt = np.full((m, k), -1, np.int64), np.full((m, k), -np.inf)
    for i in range(m):
        if np.isnan(cos[i]).any() or (bad is not None and bad[i]):
            log_prob[i] = entropy[i] = lse[i] = np.nan
            continue
        live = np.flatnonzero(cos[i] > -np.inf)
        if not len(live):
            continue
        z = float(temperature) * cos[i, live]
        at = int(z.argmax())
        d = z - z[at]
        e = np.exp(d)
        e[at] = 0.0
        rest = np.log1p(e.sum())
        lse[i] = z[at] + rest
        entropy[i] = rest - (e * d).sum() / (1.0 + e.sum())
        lp = d - rest
        where = np.full(n, -np.inf)
        where[live] = lp
        if labels is not None and 0 <= labels[i] < n:
            log_prob[i] = where[labels[i]]
        order = live[np.lexsort((live, -cos[i, live].astype(np.float32).astype(np.float64)))][:k]
        index[i, :len(order)] = order
        alt[i, :len(order)] = where[order]
    return log_prob, entropy, lse, index, alt


def score_tol(dim):
    """Bound of a cosine's error. Unit vectors: |partial sums| <= 1 by Cauchy-Schwarz. The two
    f16 parts leave at most 2^-22 of each query component, 2^-22 of the cosine in all, and the
    unit vector's own f32 roundings 3 * 2^-24; the products of f16 are exact; each of the ceil(dim / 64) * 4 matrix instructions per part
    may truncate its f32 sum of 17 terms by 2^-22 of at most 1, the low part's being 2^-11 of
    that; the row's scale and its product round to 3 * 2^-24."""
    return (dim_pad(dim) // 16 + 4) * 2.0 ** -22
