"""The 4-bit KV cache (mri_kv4_*) against a 64-bit restatement (kv4_ref.py).

What is held in 4 bits is exact: the quants, the f16 scales and so the values
read back (a product of 15 bits) equal the definition's.

Attention is compared in f64.  With hd dims, u = 2^-24:
 * a score is a sum of hd products; q is held in two f16 halves (off by 2^-22 of
   an element at most), each product and sum rounds once: its error is below
   (2^-22 + (hd + 8) u) * sum |q k| / sqrt(hd), under 40 u times that bound for
   sums whose roundings do not all point one way; the exponential and its argument
   add 4 u * |score|.  A weight's relative error is twice the score's (itself and
   the sum's).
 * an output sums p v: p * d is held in two halves (2^-22), and each rounding of
   the running sum adds u of what it holds: (2^-22 + 64 u) * sum p |v| covers the
   64 roundings of a page's matrix products, and pages and waves add a few more.
So |out - ref| <= (160 u * max(1, top) + 128 u) * sum p |v| + tiny, top the largest
sum |q k| / sqrt(hd) of the row: 2^-24 * 288 = 1.7e-5 of it at top = 1.
The halves of p d are f16 in units of 2^(e - 8), 2^e <= the largest d (p may reach 2^6
before its reference follows): what both leave is at most half of f16's smallest step,
2^-25, so 2^-33 of the largest d, times a quant of 8 at most and added over the keys (the
sum of p, before its division, is at least the probability of the key that set the
reference, 1): tiny = keys * 2^-33 * max |v|, for the largest |v| is 8 of the largest d."""
import numpy as np
import pytest

import kv4_ref as R
from gpu_util import dev, host

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32 = np.float32


def mods():
    import mri_llama as L
    import mri_qmatmul as Q
    import torch
    return L, Q, torch


def rows(rng, *shape, gain=0.7):
    return (rng.standard_normal(shape) * np.exp(gain * rng.standard_normal(shape[-1]))).astype(F32)


def read(cache, layer, shape, start, **kw):
    L, Q, torch = mods()
    k = torch.full(shape, 7.5, device="cuda")
    v = torch.full(shape, 7.5, device="cuda")
    cache.read(layer, k, v, start, **kw)
    return host(k), host(v)


# ---------------------------------------------------------------- append and read
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("kv,start,m", [(1, 0, 1), (3, 63, 1), (2, 0, 64), (2, 5, 130),
                                        (1, 60, 9), (5, 127, 2), (1, 0, 200)])
def test_append_read_exact(hd, kv, start, m):
    L, Q, torch = mods()
    rng = np.random.default_rng([hd, kv, start, m])
    c = L.Kv4Cache(2, 3, start + m + 3, kv, hd)
    k, v = rows(rng, m, kv * hd), rows(rng, m, kv * hd)
    c.append(1, dev(k), dev(v), start, first_seq=1)
    gk, gv = read(c, 1, (m, kv * hd), start, first_seq=1)
    assert np.array_equal(gk, R.stored(k).astype(F32))
    assert np.array_equal(gv, R.stored(v).astype(F32))
    # nothing else was written
    n = start + m + 3
    for layer in range(2):
        gk, gv = read(c, layer, (3, n, kv * hd), 0)
        for g, x in ((gk, k), (gv, v)):
            if layer == 1:
                assert np.array_equal(g[1, start:start + m], R.stored(x).astype(F32))
                g[1, start:start + m] = 0
            assert not g.any()


def test_append_over_old_values_and_neighbours():
    """Rows written one by one, over each other and beside others of their page."""
    L, Q, torch = mods()
    rng = np.random.default_rng(5)
    c = L.Kv4Cache(1, 1, 150, 2, 64)
    want_k, want_v = np.zeros((150, 128), F32), np.zeros((150, 128), F32)
    for start, m in ((0, 100), (30, 1), (31, 1), (99, 40), (62, 5), (0, 3), (149, 1), (64, 64)):
        k, v = rows(rng, m, 128), rows(rng, m, 128)
        c.append(0, dev(k), dev(v), start)
        want_k[start:start + m], want_v[start:start + m] = R.stored(k), R.stored(v)
    gk, gv = read(c, 0, (150, 128), 0)
    assert np.array_equal(gk, want_k) and np.array_equal(gv, want_v)


def test_quantizer_borders():
    """Values on and one f32 step beside the borders between quants; ties of the
    extremes; zero, tiny, huge and not finite blocks."""
    L, Q, torch = mods()
    rng = np.random.default_rng(9)
    blocks = []
    for d in (0.1, 0.25, 3.7, 6e-5, 2.0 ** -20, 1234.0):
        d16 = np.float64(np.float16(d))
        for sign in (1, -1):
            for off in (-1, 0, 1):
                x = np.array([n + 0.5 for n in range(-8, 8)] * 2) * d16 * sign
                x = np.nextafter(x.astype(F32), F32(np.inf) * off) if off else x.astype(F32)
                x = np.clip(x, -8 * d16, 8 * d16).astype(F32)
                x[0] = -8 * d16 * sign
                blocks.append(x)
    blocks.append(np.zeros(32, F32))
    blocks.append(np.full(32, -0.0, F32))
    t = rng.standard_normal(32).astype(F32)
    t[3], t[20] = 5, -5
    blocks += [t, -t, t[::-1].copy()]
    blocks.append((rng.standard_normal(32) * 1e-7).astype(F32))
    blocks.append((rng.standard_normal(32) * 1e-39).astype(F32))
    blocks.append((rng.standard_normal(32) * 1e6).astype(F32))
    blocks.append((rng.standard_normal(32) * 3e38).clip(-3e38, 3e38).astype(F32))
    for bad in (np.nan, np.inf, -np.inf):
        x = rng.standard_normal(32).astype(F32)
        x[7] = bad
        blocks.append(x)
    while len(blocks) % 4:
        blocks.append(rng.standard_normal(32).astype(F32))
    x = np.stack(blocks).reshape(-1, 128)
    c = L.Kv4Cache(1, 1, len(x), 2, 64)
    c.append(0, dev(x), dev(x[::-1].copy()), 0)
    gk, gv = read(c, 0, x.shape, 0)
    assert np.array_equal(gk, R.stored(x).astype(F32), equal_nan=True)
    assert np.array_equal(gv, R.stored(x[::-1]).astype(F32), equal_nan=True)


@pytest.mark.parametrize("pad,off", [(0, 0), (3, 0), (4, 1), (64, 0)])
def test_append_read_strided(pad, off):
    """Rows further apart than they are long, at addresses of any alignment."""
    L, Q, torch = mods()
    rng = np.random.default_rng(pad)
    b, m, f = 2, 70, 128
    c = L.Kv4Cache(1, b, m, 2, 64)
    buf = torch.zeros(2, b * m * (f + pad) + off, device="cuda")
    k, v = (t[off:].view(b, m, f + pad)[..., :f] for t in buf)
    xk, xv = rows(rng, b, m, f), rows(rng, b, m, f)
    k.copy_(dev(xk))
    v.copy_(dev(xv))
    c.append(0, k, v, 0)
    out = torch.full_like(buf, 9.0)
    ok, ov = (t[off:].view(b, m, f + pad) for t in out)
    c.read(0, ok[..., :f], ov[..., :f], 0)
    for o, x in ((ok, xk), (ov, xv)):
        o = host(o)
        assert np.array_equal(o[..., :f], R.stored(x).astype(F32))
        assert (o[..., f:] == 9).all()


def test_ragged_rows():
    """Counts, positions on the device, rows past the cache: what is not real is
    neither read into the cache nor written."""
    L, Q, torch = mods()
    rng = np.random.default_rng(3)
    b, m, f, n = 6, 40, 128, 100
    pos = np.array([0, 61, 80, 99, 100, 0xffffffff], np.uint32)
    cnt = np.array([40, 0, 33, 5, 4, 40], np.uint32)
    c = L.Kv4Cache(1, b, n, 1, 128)
    k, v = rows(rng, b, m, f), rows(rng, b, m, f)
    dp, dc = dev(pos.view(np.int32)), dev(cnt.view(np.int32))
    c.append(0, dev(k), dev(v), dp, count=dc)
    gk, gv = read(c, 0, (b, n, f), 0)
    want = np.zeros((2, b, n, f), F32)
    back = np.full((2, b, m, f), 7.5, F32)
    for i in range(b):
        real = 0 if pos[i] >= n else min(int(cnt[i]), n - int(pos[i]))
        for j, x in enumerate((k, v)):
            want[j, i, pos[i]:pos[i] + real] = R.stored(x[i, :real])
            back[j, i, :real] = R.stored(x[i, :real])
    assert np.array_equal(gk, want[0]) and np.array_equal(gv, want[1])
    gk, gv = read(c, 0, (b, m, f), dp, count=dc)
    assert np.array_equal(gk, back[0]) and np.array_equal(gv, back[1])


# ---------------------------------------------------------------- attention
def check_attend(hd, kv, grp, b, m, pos, cnt=None, weights=True, seed=0, scale=1.0, max_seq=None):
    L, Q, torch = mods()
    rng = np.random.default_rng([seed, hd, kv, grp, b, m])
    pos = [pos] * b if isinstance(pos, int) else list(pos)
    cnt_l = [m] * b if cnt is None else [min(x, m) for x in cnt]
    t = max_seq or max(p + m for p in pos)
    c = L.Kv4Cache(1, b, t, kv, hd)
    k, v = rows(rng, b, t, kv * hd), rows(rng, b, t, kv * hd)
    # keys that no row sees hold what must not matter: the largest values, NaN
    for i in range(b):
        end = pos[i] + cnt_l[i]
        k[i, end:], v[i, end:] = np.nan, np.where(np.arange(t - end)[:, None] % 2, np.nan, 5e5)
    c.append(0, dev(k), dev(v), 0)
    q = (rng.standard_normal((b, m, kv * grp * hd)) * scale).astype(F32)
    out = torch.full(q.shape, 7.5, device="cuda")
    w0 = rng.uniform(0, 2, (b, kv, t)).astype(F32)
    w = dev(w0)
    start = pos[0] if len(set(pos)) == 1 else dev(np.array(pos, np.int32))
    count = None if cnt is None else dev(np.array(cnt, np.int32))
    c.attend(0, dev(q), out, start, count=count, weights=w if weights else None)
    got, gw = host(out), host(w)
    for i in range(b):
        n, end = cnt_l[i], pos[i] + cnt_l[i]
        assert (got[i, n:] == 7.5).all()
        if not n:
            assert np.array_equal(gw[i], w0[i])
            continue
        sk = R.stored(k[i, :end]).reshape(end, kv, hd)
        sv = R.stored(v[i, :end]).reshape(end, kv, hd)
        ref, rw, mag, top = R.attend(q[i, :n], sk, sv, pos[i], kv * grp)
        tiny = end * 2.0 ** -33 * np.abs(sv).max()
        err, tol = np.abs(got[i, :n] - ref), (160 * np.maximum(1, top) + 128) * U * mag + tiny
        worst = (err / tol).max()
        assert worst <= 1, (i, worst, err.max())
        if weights:
            old = np.where(np.arange(t) < pos[i], w0[i], 0).astype(np.float64)
            want = old[:, :end] + rw
            # each weight is off by twice its score's error, each of the n * grp
            # additions by u of the sum
            wt = (160 * max(1, top.max()) + 2 * n * grp + 4) * U * (want + 1e-30)
            assert (np.abs(gw[i][:, :end] - want) <= wt).all()
            assert np.array_equal(gw[i][:, end:], w0[i][:, end:])
    # the same call again gives the same bits
    out2, w2 = torch.full(q.shape, 7.5, device="cuda"), dev(w0)
    c.attend(0, dev(q), out2, start, count=count, weights=w2 if weights else None)
    assert np.array_equal(host(out2), got)
    if weights:
        assert np.array_equal(host(w2), gw)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("kv,grp,b,m,pos", [
    (1, 1, 1, 1, 0),            # one key
    (2, 1, 1, 1, 63), (2, 1, 1, 1, 64), (1, 4, 1, 1, 300),
    (2, 3, 2, 1, 1000),         # three heads a group
    (1, 7, 1, 5, 190),          # 35 queries: a ragged last tile
    (1, 16, 1, 1, 70), (1, 17, 1, 1, 70),
    (4, 2, 3, 4, 130),
    (2, 2, 1, 33, 0), (1, 1, 1, 200, 0), (1, 1, 1, 65, 447), (3, 1, 2, 100, 37),
])
def test_attend(hd, kv, grp, b, m, pos):
    check_attend(hd, kv, grp, b, m, pos)


@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("m,pos,cnt", [
    (1, (0, 900, 63, 64, 2047), None),
    (5, (3, 700, 64, 59, 0), (5, 1, 0, 9, 4)),
    (80, (0, 30, 64, 1, 7), (80, 0, 17, 64, 1)),
])
def test_attend_ragged(m, pos, cnt, weights):
    check_attend(128, 2, 2, 5, m, pos, cnt, weights)


def test_attend_many_sequences():
    """More sequences than a wave has lanes, with far apart lengths."""
    rng = np.random.default_rng(1)
    pos = [int(x) for x in rng.integers(0, 40, 70)]
    pos[3], pos[69] = 1500, 640
    check_attend(64, 1, 2, 70, 1, pos, [int(x) for x in rng.integers(0, 2, 70)])


@pytest.mark.parametrize("hd", [64, 128])
def test_attend_more_sequences_than_cus(hd):
    """Enough tiles that none splits its keys, one and several columns a tile."""
    rng = np.random.default_rng(hd)
    pos = [int(x) for x in rng.integers(0, 150, 450)]
    check_attend(hd, 2, 2, 450, 1, pos, [int(x) for x in rng.integers(0, 2, 450)])
    check_attend(hd, 1, 6, 400, 2, pos[:400], [int(x) for x in rng.integers(0, 3, 400)])


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("kv,grp,b,m,pos,cnt", [
    (8, 2, 8, 130, 0, None),                    # 64 queries a workgroup, a short last one
    (8, 1, 7, 300, 70, (300, 0, 1, 64, 65, 299, 17)),
    (4, 3, 16, 100, 5, None),                   # tiles that end inside a row's heads
])
def test_attend_prompts(hd, kv, grp, b, m, pos, cnt):
    """Prompts large enough for the form that shares pages between queries."""
    check_attend(hd, kv, grp, b, m, pos, cnt)


def test_attend_prompt_strided_and_nan():
    """The same form with rows of any spacing and alignment, and with NaN among the
    queries, keys and values: only what sees it is spoilt."""
    L, Q, torch = mods()
    rng = np.random.default_rng(61)
    kv, hd, m = 32, 64, 520
    c = L.Kv4Cache(1, 1, m, kv, hd)
    k, v = rows(rng, m, kv * hd), rows(rng, m, kv * hd)
    q = rng.standard_normal((m, kv * hd)).astype(F32)
    k[200, 3] = np.inf                 # head 0
    v[100, hd + 40] = np.nan           # head 1, its second block
    q[70, 2 * hd + 5] = np.nan         # head 2
    c.append(0, dev(k), dev(v), 0)
    a = torch.empty(m, kv * hd, device="cuda")
    c.attend(0, dev(q), a, 0)
    got = host(a).reshape(m, kv, hd)
    bad = np.zeros((m, kv, hd), bool)
    bad[200:, 0] = bad[70, 2] = True
    bad[100:, 1, 32:] = True
    assert np.array_equal(np.isnan(got), bad)
    for pad, off in ((1, 3), (4, 0)):
        buf = torch.zeros(m * (kv * hd + pad) + off, device="cuda")
        qs = buf[off:].view(m, kv * hd + pad)
        qs[:, :kv * hd] = dev(q)
        ob = torch.full_like(buf, 9.0)
        o = ob[off:].view(m, kv * hd + pad)
        c.attend(0, qs[:, :kv * hd], o[:, :kv * hd], 0)
        assert np.array_equal(host(o[:, :kv * hd]).reshape(got.shape), got, equal_nan=True)
        assert bool((o[:, kv * hd:] == 9).all())


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("b,kv,grp,m,pos", [(2, 2, 2, 1, 900), (3, 2, 4, 5, 300), (8, 8, 2, 130, 0),
                                            (300, 2, 2, 1, 20)])
def test_attend_in_place(hd, b, kv, grp, m, pos):
    """The output over the queries, in every form of the call."""
    L, Q, torch = mods()
    rng = np.random.default_rng([hd, b, kv])
    c = L.Kv4Cache(1, b, pos + m, kv, hd)
    k, v = (dev(rows(rng, b, pos + m, kv * hd)) for _ in range(2))
    c.append(0, k, v, 0)
    q = dev(rng.standard_normal((b, m, kv * grp * hd)).astype(F32))
    out = torch.empty_like(q)
    c.attend(0, q, out, pos)
    c.attend(0, q, q, pos)
    assert torch.equal(q, out)


def test_attend_long():
    check_attend(128, 1, 4, 1, 1, 20000)


@pytest.mark.parametrize("scale", [0.0, 1e-20, 12.0])
def test_attend_query_scales(scale):
    """Equal scores, and scores that leave one key all the weight."""
    check_attend(128, 2, 2, 1, 2, 200, scale=scale)


@pytest.mark.parametrize("first,second", [(1e-5, 300.0), (300.0, 1e-5), (0.0, 1.0)])
def test_attend_value_scales(first, second):
    """Value blocks of very different scales along the keys: the running power of
    two has to follow them."""
    L, Q, torch = mods()
    rng = np.random.default_rng(17)
    n, hd = 640, 64
    k, v = rows(rng, n, hd), rows(rng, n, hd, gain=0.1)
    v[:320] *= F32(first)
    v[320:] *= F32(second)
    c = L.Kv4Cache(1, 1, n, 1, hd)
    c.append(0, dev(k), dev(v), 0)
    for m, pos in ((1, n - 1), (300, n - 300)):
        q = rng.standard_normal((m, hd)).astype(F32)
        out = torch.empty(m, hd, device="cuda")
        c.attend(0, dev(q), out, pos)
        sk, sv = (R.stored(x).reshape(n, 1, hd) for x in (k, v))
        ref, _, mag, top = R.attend(q, sk, sv, pos, 1)
        tiny = n * 2.0 ** -33 * np.abs(sv).max()
        assert (np.abs(host(out) - ref) <= (160 * np.maximum(1, top) + 128) * U * mag + tiny).all()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("kv,m,pos", [(1, 1, 600), (2, 5, 600), (8, 520, 0)])
@pytest.mark.parametrize("small", [1e-3, 2e-5])
def test_attend_blocks_of_different_scales(hd, kv, m, pos, small):
    """Value blocks of a head whose sizes lie far apart: each keeps f32 accuracy, the
    small ones too.  Both halves' smallest steps are those of the block's own scales, and
    p may reach 2^3 before its reference follows: tiny = keys * 2^-36 * max |v of the
    block|."""
    L, Q, torch = mods()
    rng = np.random.default_rng([hd, kv, m])
    n, nb = pos + m, hd // 32
    k, v = (rng.standard_normal((n, kv, hd)).astype(F32) for _ in range(2))
    for b in range(nb):         # every second block is small
        if b % 2 == 0:
            v[:, :, 32 * b:32 * b + 32] *= F32(small)
    k, v = k.reshape(n, -1), v.reshape(n, -1)
    c = L.Kv4Cache(1, 1, n, kv, hd)
    c.append(0, dev(k), dev(v), 0)
    q = rng.standard_normal((m, kv * 2 * hd)).astype(F32)
    out = torch.empty(q.shape, device="cuda")
    c.attend(0, dev(q), out, pos)
    sk, sv = (R.stored(x).reshape(n, kv, hd) for x in (k, v))
    ref, _, mag, top = R.attend(q, sk, sv, pos, 2 * kv)
    most = np.abs(sv).reshape(n, kv, nb, 32).max((0, 3))                  # [kv, blocks]
    tiny = n * 2.0 ** -36 * np.repeat(np.repeat(most, 2, 0), 32, 1).reshape(-1)
    tol = (160 * np.maximum(1, top) + 128) * U * mag + tiny
    err = np.abs(host(out) - ref)
    assert (err <= tol).all(), (err / tol).max()
    # and in the mean of a block, where roundings do not all point one way: a score's last
    # roundings, under u * top, and as many steps as the output's own additions take
    part = [x.reshape(m, -1, nb, 32).sum((0, 1, 3)) for x in (err, mag)]
    assert (part[0] <= (np.maximum(1, top.max()) + 8) * U * part[1]).all(), part[0] / part[1] / U


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("m,at", [(1, 3), (1, 640), (300, 3), (300, 555)])
def test_attend_large_value_that_is_not_attended(hd, m, at):
    """A value block 1000 times the others' at a key of next to no weight, before and
    among the rows' own keys: it stays out of the result, and what is lost beside it is
    2^-36 of it a key at most."""
    L, Q, torch = mods()
    rng = np.random.default_rng([hd, m, at])
    n, kv = 700, 8
    k, v = (rng.standard_normal((n, kv, hd)).astype(F32) for _ in range(2))
    q = rng.standard_normal((m, kv, hd)).astype(F32)
    q[..., 0] = 4
    k[at, :, 0] = -30 * np.sqrt(hd) / 4      # a score of -30 or so
    v[at, :, :32] *= 1000
    c = L.Kv4Cache(1, 1, n, kv, hd)
    c.append(0, dev(k.reshape(n, -1)), dev(v.reshape(n, -1)), 0)
    out = torch.empty(m, kv * hd, device="cuda")
    c.attend(0, dev(q.reshape(m, -1)), out, n - m)
    sk, sv = (R.stored(x.reshape(n, -1)).reshape(n, kv, hd) for x in (k, v))
    ref, _, mag, _ = R.attend(q.reshape(m, -1), sk, sv, n - m, kv)
    # (the keys that have weight: their scores are off by their own sizes)
    near = np.delete(np.arange(n), at)
    top = np.abs(q).max() * np.abs(sk[near]).sum(-1).max() / np.sqrt(hd)
    most = np.abs(sv).reshape(n, kv, hd // 32, 32).max((0, 3))
    tiny = n * 2.0 ** -36 * np.repeat(most, 32, 1).reshape(-1)
    assert (np.abs(host(out) - ref) <= (160 * top + 128) * U * mag + tiny).all()


def test_attend_nan_and_inf():
    """A query with NaN spoils its own row only; a NaN key every row that sees it; a
    NaN value its block's dims."""
    L, Q, torch = mods()
    rng = np.random.default_rng(23)
    n, hd = 150, 64
    k, v = rows(rng, n, hd), rows(rng, n, hd)
    q = rng.standard_normal((n, hd)).astype(F32)
    k[100, 3] = np.inf
    v[50, 40] = np.nan
    q[20, 5] = np.nan
    c = L.Kv4Cache(1, 1, n, 1, hd)
    c.append(0, dev(k), dev(v), 0)
    out = torch.empty(n, hd, device="cuda")
    c.attend(0, dev(q), out, 0)
    bad = np.zeros((n, hd), bool)
    bad[20] = True
    bad[50:, 32:] = True
    bad[100:] = True
    assert np.array_equal(np.isnan(host(out)), bad)


def test_attend_strided():
    L, Q, torch = mods()
    rng = np.random.default_rng(29)
    b, m, n, f = 2, 3, 90, 4 * 64
    c = L.Kv4Cache(1, b, n, 2, 64)
    k, v = rows(rng, b, n, 128), rows(rng, b, n, 128)
    c.append(0, dev(k), dev(v), 0)
    q = rng.standard_normal((b, m, f)).astype(F32)
    a = torch.empty(b, m, f, device="cuda")
    c.attend(0, dev(q), a, n - m)
    for pad, off in ((1, 3), (8, 0)):
        buf = torch.zeros(b * m * (f + pad) + off, device="cuda")
        qs = buf[off:].view(b, m, f + pad)
        qs[..., :f] = dev(q)
        ob = torch.full_like(buf, 9.0)
        os_ = ob[off:].view(b, m, f + pad)
        c.attend(0, qs[..., :f], os_[..., :f], n - m)
        assert torch.equal(os_[..., :f], a) and bool((os_[..., f:] == 9).all())


def test_weights_in_chunks():
    """More (row, head) pairs than the workspace's log-sum-exps hold: the call runs
    in parts, with the same sums as calls of those rows one after the other."""
    L, Q, torch = mods()
    rng = np.random.default_rng(31)
    hd, heads, m = 64, 512, 2100          # 1075200 pairs > 2^20
    c = L.Kv4Cache(1, 1, m, 1, hd)
    k, v = rows(rng, m, hd), rows(rng, m, hd)
    c.append(0, dev(k), dev(v), 0)
    q = dev(rng.standard_normal((m, heads * hd)).astype(F32))
    out, w = torch.empty_like(q), torch.full((1, 1, m), 3.0, device="cuda")
    c.attend(0, q, out, 0, weights=w)
    o2, w2 = torch.empty_like(q), torch.zeros((1, 1, m), device="cuda")
    for i in range(0, m, 1050):
        c.attend(0, q[i:i + 1050], o2[i:i + 1050], i, weights=w2)
    assert float((out - o2).abs().max()) <= 1e-5 * float(o2.abs().max())
    # sums of m * heads weights in [0, 1], each addition off by half a step
    assert float(((w - w2).abs() / w2).max()) <= 2 * 1024 * U
    assert abs(float(w.double().sum()) / (m * heads) - 1) < 1e-4


# ---------------------------------------------------------------- eviction
def run_evict(src, dst, w, lens, keep, recent):
    L, Q, torch = mods()
    lead = w.shape[:3]
    dw = dev(w)
    wo = dw if dst is src else torch.full(lead + (dst.max_seq,), -5.0, device="cuda")
    kept = torch.full(lead + (keep,), 77, dtype=torch.int32, device="cuda")
    dl = dev(np.array(lens, np.uint32).view(np.int32))
    lo = dl if dst is src else torch.full((w.shape[1],), 99, dtype=torch.int32, device="cuda")
    src.evict(dst, dw, wo, dl, lo, keep, recent, kept)
    return host(kept).view(np.uint32), host(lo), host(wo)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("hd,kv,n,keep,recent,lens", [
    (64, 1, 1, 1, 0, (1,)), (64, 1, 2, 1, 1, (2,)), (64, 2, 100, 30, 10, (100, 30)),
    (128, 2, 300, 128, 0, (300, 0, 129)), (128, 1, 300, 65, 65, (300, 66)),
    (64, 3, 1500, 700, 100, (1500, 1, 699, 701)), (128, 1, 5000, 64, 3, (5000, 9000)),
])
def test_evict(hd, kv, n, keep, recent, lens, in_place):
    L, Q, torch = mods()
    rng = np.random.default_rng([hd, kv, n, keep])
    a, b = 2, len(lens)
    w = np.exp(2 * rng.standard_normal((a, b, kv, n))).astype(F32)
    w[rng.random(w.shape) < 0.2] = 0.25        # equal weights
    w[rng.random(w.shape) < 0.01] = 0.0
    w[rng.random(w.shape) < 0.01] = -0.0
    src = L.Kv4Cache(a, b, n, kv, hd)
    k, v = rows(rng, a, b, n, kv * hd), rows(rng, a, b, n, kv * hd)
    for i in range(a):
        src.append(i, dev(k[i]), dev(v[i]), 0)
    dst = src if in_place else L.Kv4Cache(a, b, keep + 5, kv, hd)
    old = rows(rng, b, keep + 5, kv * hd)      # what dst holds past the kept stays
    if not in_place:
        for i in range(a):
            dst.append(i, dev(old), dev(old), 0)
    kept, lo, wo = run_evict(src, dst, w, lens, keep, recent)
    lens = [min(x, n) for x in lens]
    assert list(lo) == [min(x, keep) for x in lens]
    sk, sv = R.stored(k).astype(F32), R.stored(v).astype(F32)
    gk, gv = read(dst, 0, (a, b, dst.max_seq, kv * hd), 0)
    for i in range(a):
        for j in range(b):
            for g in range(kv):
                at = R.evict(w[i, j, g], lens[j], keep, recent)
                assert np.array_equal(kept[i, j, g, :len(at)], at)
                assert (kept[i, j, g, len(at):] == R.NO_TOKEN).all()
                lane = slice(g * hd, (g + 1) * hd)
                assert np.array_equal(gk[i, j, :len(at), lane], sk[i, j, at, lane])
                assert np.array_equal(gv[i, j, :len(at), lane], sv[i, j, at, lane])
                assert np.array_equal(wo[i, j, g, :len(at)], w[i, j, g, at])
                rest = slice(len(at), None)
                if in_place:
                    assert np.array_equal(wo[i, j, g, rest], w[i, j, g, rest])
                    assert np.array_equal(gk[i, j, rest, lane], sk[i, j, rest, lane])
                    assert np.array_equal(gv[i, j, rest, lane], sv[i, j, rest, lane])
                else:
                    assert (wo[i, j, g, rest] == -5).all()
                    so = R.stored(old[j]).astype(F32)
                    assert np.array_equal(gk[i, j, rest, lane], so[rest, lane])
                    assert np.array_equal(gv[i, j, rest, lane], so[rest, lane])


def test_evict_many_positions():
    """More weights a head than registers hold."""
    L, Q, torch = mods()
    rng = np.random.default_rng(37)
    n, keep, recent = 40000, 5000, 700
    w = np.exp(3 * rng.standard_normal((1, 2, 1, n))).astype(F32)
    w[rng.random(w.shape) < 0.3] = 0.5
    src, dst = L.Kv4Cache(1, 2, n, 1, 64), L.Kv4Cache(1, 2, keep, 1, 64)
    kept, lo, wo = run_evict(src, dst, w, (n, n - 77), keep, recent)
    for j, m in enumerate((n, n - 77)):
        at = R.evict(w[0, j, 0], m, keep, recent)
        assert np.array_equal(kept[0, j, 0], at) and np.array_equal(wo[0, j, 0], w[0, j, 0, at])


def test_evict_special_weights():
    """Infinities, NaN, negative and equal weights keep their order."""
    L, Q, torch = mods()
    rng = np.random.default_rng(41)
    n = 400
    w = rng.choice(np.array([np.nan, np.inf, -np.inf, 0.0, -0.0, 1.0, -1.0, 1e-45, 3e38], F32),
                   (1, 2, 1, n))
    w[0, 1] = 1.0
    src, dst = L.Kv4Cache(1, 2, n, 1, 64), L.Kv4Cache(1, 2, n, 1, 64)
    for keep in (1, 40, 200, 333, 399):
        kept, _, _ = run_evict(src, dst, w, (n, n), keep, min(keep, 7))
        for j in range(2):
            assert np.array_equal(kept[0, j, 0], R.evict(w[0, j, 0], n, keep, min(keep, 7))), keep


# ---------------------------------------------------------------- captured graphs
def test_graph_replays():
    """A decode step captured once follows positions that move on the device; every
    replay equals the eager call."""
    L, Q, torch = mods()
    rng = np.random.default_rng(43)
    b, kv, grp, hd, n = 2, 2, 2, 64, 300
    kvd, qd = kv * hd, kv * grp * hd
    graph_c, eager_c = (L.Kv4Cache(1, b, n, kv, hd) for _ in range(2))
    k, v, q = (torch.zeros(b, 1, d, device="cuda") for d in (kvd, kvd, qd))
    out = torch.zeros(b, 1, qd, device="cuda")
    pos = torch.zeros(b, dtype=torch.int32, device="cuda")
    w, w_e = (torch.zeros(b, kv, n, device="cuda") for _ in range(2))

    def step():
        graph_c.append(0, k, v, pos)
        graph_c.attend(0, q, out, pos, weights=w)
        pos.add_(1)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            step()
    pos.copy_(torch.tensor([0, 100], dtype=torch.int32))
    at = [0, 100]
    for _ in range(80):
        for t in (k, v, q):
            t.copy_(dev(rows(rng, *t.shape)))
        graph.replay()
        torch.cuda.synchronize()
        e_out = torch.empty_like(out)
        e_pos = torch.tensor(at, dtype=torch.int32, device="cuda")
        eager_c.append(0, k, v, e_pos)
        eager_c.attend(0, q, e_out, e_pos, weights=w_e)
        assert torch.equal(out, e_out) and torch.equal(w, w_e)
        at = [x + 1 for x in at]
    assert pos.tolist() == at


def test_other_streams():
    """Independent caches on two streams at once give what they give alone."""
    L, Q, torch = mods()
    rng = np.random.default_rng(47)
    n, kv, hd = 1200, 4, 128
    caches = [L.Kv4Cache(1, 1, n, kv, hd) for _ in range(2)]
    ks = [dev(rows(rng, n, kv * hd)) for _ in range(2)]
    qs = [dev(rng.standard_normal((1, 8 * hd)).astype(F32)) for _ in range(2)]
    alone = []
    for c, k, q in zip(caches, ks, qs):
        c.append(0, k, k, 0)
        o = torch.empty_like(q)
        c.attend(0, q, o, n - 1)
        alone.append(o)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [torch.zeros_like(q) for q in qs]
    torch.cuda.synchronize()
    for _ in range(20):
        for c, q, o, s in zip(caches, qs, outs, streams):
            with torch.cuda.stream(s):
                c.attend(0, q, o, n - 1)
    torch.cuda.synchronize()
    assert all(torch.equal(a, o) for a, o in zip(alone, outs))
