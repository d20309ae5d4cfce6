"""A 64-bit restatement of the 4-bit KV cache's operators, softmax and draft
verification (include/mri_llama.h), in numpy."""
import numpy as np

NO_TOKEN = 0xffffffff


def stored(x):
    """The values that blocks of 32 along the last axis stand for, in f64."""
    x = np.asarray(x, np.float32)
    blk = x.reshape(-1, 32).astype(np.float64)
    out = np.full(blk.shape, np.nan)
    ok = np.isfinite(blk).all(1)
    b = blk[ok]
    hi, lo = b.max(1), b.min(1)
    a = np.where(hi >= -lo, hi, lo)
    d = np.clip(a / -8, -65504, 65504).astype(np.float16).astype(np.float64)[:, None]
    with np.errstate(divide="ignore", invalid="ignore"):
        q = np.where(d != 0, b / d, 0.0)
    out[ok] = np.clip(np.rint(q), -8, 7) * d
    return out.reshape(x.shape)


def attend(q, k, v, pos, n_heads):
    """q [m, n_heads * hd] at positions pos .. over stored k, v [>= pos + m, n_kv, hd]:
    the output [m, n_heads * hd], the rows' weights summed per KV head [n_kv, keys]
    and, of each output, sum_t p_t |v_t| and the row's largest |score|."""
    m, (keys, n_kv, hd) = q.shape[0], k.shape
    grp = n_heads // n_kv
    out = np.zeros((m, n_heads, hd))
    mag = np.zeros((m, n_heads, hd))
    top = np.zeros((m, n_heads))
    w = np.zeros((n_kv, keys))
    q = q.reshape(m, n_heads, hd).astype(np.float64)
    for h in range(n_heads):
        g = h // grp
        s = q[:, h] @ k[:, g].T / np.sqrt(hd)
        bound = np.abs(q[:, h]) @ np.abs(k[:, g].T) / np.sqrt(hd)
        for i in range(m):
            n = pos + i + 1
            e = np.exp(s[i, :n] - s[i, :n].max())
            p = e / e.sum()
            out[i, h] = p @ v[:n, g]
            mag[i, h] = p @ np.abs(v[:n, g])
            top[i, h] = bound[i, :n].max()
            w[g, :n] += p
    return out.reshape(m, -1), w, mag.reshape(m, -1), np.repeat(top, hd, 1)


def evict(w, n, keep, recent):
    """The kept positions of one head's n weights."""
    if n <= keep:
        return np.arange(n)
    old = n - recent
    key = np.where(np.isnan(w[:old]), -np.inf, w[:old].astype(np.float64))
    # NaN below -inf: among equals of -inf the numbers come first
    order = np.lexsort((np.arange(old), np.isnan(w[:old]), -key))
    return np.concatenate((np.sort(order[:keep - recent]), np.arange(old, n)))


def verify(drafts, p, u, q=None, count=None):
    """One sequence: (accepted, tokens)."""
    k, n = len(drafts), p.shape[1]
    p = np.where(np.isnan(p), 0, p).astype(np.float64)
    u = u.astype(np.float64)
    count = k if count is None else min(count, k)
    i = 0
    while i < count and drafts[i] < n and \
            u[i] * (1.0 if q is None else float(q[i, drafts[i]])) < p[i, drafts[i]]:
        i += 1
    r = p[i].copy()
    if i < count:
        if q is not None:
            r = r - np.where(np.isnan(q[i]), np.inf, q[i]).astype(np.float64)
        elif drafts[i] < n:
            r[drafts[i]] -= 1.0
        r = np.maximum(r, 0)
        if r.sum() == 0:
            r = np.maximum(p[i], 0)
    r = np.maximum(r, 0)
    out = np.full(k + 1, NO_TOKEN, np.uint32)
    out[:i] = drafts[:i]
    if r.sum() > 0:
        c = np.cumsum(r)
        t = int(np.searchsorted(c, u[k] * c[-1], side="right"))
        out[i] = min(t, int(np.flatnonzero(r > 0)[-1]))
    return i, out
