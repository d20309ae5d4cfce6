"""mri_softmax and mri_verify_drafts against 64-bit restatements.

Softmax: with u = 2^-24, t = (max x - x) / T: the argument of the exponential is
off by 3 u t (difference, constant, product), the exponential by 2 u, the sum of n by
(log2(1024) + n / 1024 + 2) u, the reciprocal and product by 2 u: within
(4 t + n / 1024 + 20) u of the value, and 2^-126 where exponentials vanish.
Verification is whole numbers: equal."""
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


def check_softmax(x, temperature, got):
    x = x.astype(np.float64)
    m = x.max(-1, keepdims=True)
    t = (m - x) / temperature
    e = np.exp(-t)
    ref = e / e.sum(-1, keepdims=True)
    t = np.where(np.isfinite(t), t, 0)
    tol = (4 * t + x.shape[-1] / 1024 + 20) * U * ref + 2.0 ** -126
    assert (np.abs(got - ref) <= tol).all(), np.nanmax(np.abs(got - ref) / tol)


@pytest.mark.parametrize("rows,n", [(1, 1), (3, 2), (2, 63), (5, 64), (1, 1000), (7, 4099),
                                    (2, 32000), (3, 50021), (1, 131072), (300, 33),
                                    (2, 300001), (1100, 5000), (9, 4096), (2, 8193),
                                    (3, 16384), (2, 32768), (2, 32769), (520, 33001)])
@pytest.mark.parametrize("temperature", [0.3, 1.0, 2.5])
def test_softmax(rows, n, temperature):
    L, Q, torch = mods()
    rng = np.random.default_rng([rows, n])
    x = (rng.standard_normal((rows, n)) * 4).astype(F32)
    x[0, rng.random(n) < 0.5] = -np.inf
    x[0, n // 2] = 1.0
    out = torch.empty(rows, n, device="cuda")
    L.softmax(dev(x), out, temperature=temperature)
    got = host(out)
    check_softmax(x, temperature, got)
    d = dev(x)
    L.softmax(d, d, temperature=temperature)       # in place
    assert np.array_equal(host(d), got)


@pytest.mark.parametrize("n", [777, 9001, 30000, 40000])
def test_softmax_special_rows(n):
    L, Q, torch = mods()
    x = np.zeros((8, n), F32)
    x[0] = -np.inf                      # nothing left: zeros
    x[1], x[1, 5] = -np.inf, -3.0       # one left
    x[2, 9] = np.nan
    x[3, 4] = np.inf
    x[4] = np.finfo(F32).min            # the type's lowest value everywhere
    x[5], x[5, 0] = np.finfo(F32).min, 2.0
    x[6] = np.finfo(F32).max
    x[7, 3], x[7, 4] = np.nan, -np.inf
    out = torch.empty(8, n, device="cuda")
    L.softmax(dev(x), out)
    got = host(out)
    assert not got[0].any()
    assert got[1, 5] == 1 and not np.delete(got[1], 5).any()
    assert np.isnan(got[2]).all() and np.isnan(got[3]).all() and np.isnan(got[7]).all()
    for r in (4, 6):
        assert np.allclose(got[r], 1 / n, rtol=(n / 1024 + 20) * U, atol=0)
    assert got[5, 0] == 1 and not got[5, 1:].any()


@pytest.mark.parametrize("rows,n", [(3, 777), (2, 8193), (2, 30000), (3, 40000), (514, 32769)])
@pytest.mark.parametrize("temperature", [1e38, 3e38, 2e37])
def test_softmax_wide_logits(rows, n, temperature):
    """Logits that lie further apart than the type's largest value, under a temperature
    that brings them together."""
    L, Q, torch = mods()
    rng = np.random.default_rng([rows, n])
    x = (rng.uniform(-1, 1, (rows, n)) * 3.4e38).astype(F32)
    x[:, 0], x[:, n - 1] = 3.4e38, -3.4e38
    out = torch.empty(rows, n, device="cuda")
    L.softmax(dev(x), out, temperature=temperature)
    check_softmax(x, float(F32(temperature)), host(out))


@pytest.mark.parametrize("pad,off", [(1, 0), (3, 1), (4, 0)])
def test_softmax_strided(pad, off):
    L, Q, torch = mods()
    rng = np.random.default_rng(pad)
    rows, n = 3, 2000
    x = rng.standard_normal((rows, n)).astype(F32)
    buf = torch.full((rows * (n + pad) + off,), 9.0, device="cuda")
    v = buf[off:].view(rows, n + pad)
    v[:, :n] = dev(x)
    L.softmax(v[:, :n], v[:, :n], temperature=0.7)
    got = host(v)
    check_softmax(x, 0.7, got[:, :n])
    assert (got[:, n:] == 9).all()


def probs(rng, *shape):
    z = 2.5 * rng.standard_normal(shape)
    e = np.exp(z - z.max(-1, keepdims=True))
    return (e / e.sum(-1, keepdims=True)).astype(F32)


def run_verify(drafts, p, u, q=None, counts=None):
    L, Q, torch = mods()
    b, k = drafts.shape
    tokens = torch.full((b, k + 1), 5, dtype=torch.int32, device="cuda")
    acc = torch.full((b,), 5, dtype=torch.int32, device="cuda")
    i32 = lambda a: dev(np.asarray(a, np.uint32).view(np.int32))  # noqa: E731
    L.verify_drafts(i32(drafts), dev(p), dev(u), tokens, acc,
                    draft_probs=None if q is None else dev(q),
                    n_drafts=None if counts is None else i32(counts))
    tokens, acc = host(tokens).view(np.uint32), host(acc)
    for i in range(b):
        a, t = R.verify(drafts[i], p[i], u[i], None if q is None else q[i],
                        None if counts is None else int(counts[i]))
        assert acc[i] == a and np.array_equal(tokens[i], t), (i, acc[i], a, tokens[i], t)
    return acc, tokens


@pytest.mark.parametrize("b,k,n", [(1, 0, 1), (3, 0, 17), (40, 4, 2), (20, 3, 64), (20, 3, 65),
                                   (16, 8, 1000), (8, 4, 16385), (4, 7, 32000), (2, 2, 131072),
                                   (3, 70, 200), (2, 1, 300001)])
@pytest.mark.parametrize("sampled", [True, False])
def test_verify(b, k, n, sampled):
    rng = np.random.default_rng([b, k, n])
    p, q = probs(rng, b, k + 1, n), probs(rng, b, k, n)
    if k:
        q = (0.5 * q + 0.5 * p[:, :k]).astype(F32)
    drafts = (q.argmax(2) if n > 1 and k else np.zeros((b, k))).astype(np.uint32)
    u = rng.random((b, k + 1)).astype(F32)
    counts = rng.integers(0, k + 3, b).astype(np.uint32)
    for c in (None, counts):
        run_verify(drafts, p, u, q if sampled else None, c)


def test_verify_borders():
    """Equal sides are rejected, exact products decide, zero draft probabilities,
    no residual mass, no mass at all, ids out of range, NaN, uniforms at their ends."""
    rng = np.random.default_rng(3)
    b, k, n = 12, 2, 300
    p, q = probs(rng, b, k + 1, n), probs(rng, b, k, n)
    u = rng.random((b, k + 1)).astype(F32)
    drafts = rng.integers(0, n, (b, k)).astype(np.uint32)
    at = np.arange(k)
    p[0, 0, drafts[0, 0]] = q[0, 0, drafts[0, 0]] * F32(0.5)
    u[0, 0] = 0.5                                     # u q == p: rejected
    x = F32(0.3)
    q[1, 0, drafts[1, 0]], u[1, 0] = x, x
    p[1, 0, drafts[1, 0]] = np.nextafter(F32(x * x), F32(1))   # a rounding above
    q[2, at, drafts[2]] = 0                           # accepted wherever p > 0
    p[3, :k], q[3] = q[3], q[3]                       # no residual: the target's own
    u[3] = (1.0, 0.5, 0.4)
    p[4] = 0                                          # no mass
    drafts[5, 0], drafts[6, 1] = n, 0xffffffff        # no such ids
    u[6, 0] = 0
    p[7, :, ::2] = np.nan
    u[8] = 0
    u[9, k] = np.nextafter(F32(1), F32(0))
    u[10, k] = 1.0
    u[11, k] = 0
    p[11, :, :200] = 0
    run_verify(drafts, p, u, q)
    run_verify(drafts, p, u)


@pytest.mark.parametrize("n", [1, 1023, 1025, 2500, 4096, 140000])
def test_verify_rejected_greedy_drafts(n):
    """The rejected token leaves the target's row wherever it lies among its blocks;
    where it held all the mass, or is no token, the target's row stays."""
    rng = np.random.default_rng(n)
    ids = np.unique([i for i in (0, 3, 1020, 1023, 1024, 2047, n // 2, n - 1) if i < n])
    ids = np.concatenate([ids, [n, n + 7, 0xfffffffe]]).astype(np.uint32)
    b = 2 * len(ids)
    p = probs(rng, b, 2, n)
    u = rng.random((b, 2)).astype(F32)
    u[:, 0] = 1.0                                   # rejected unless p > 1
    drafts = np.concatenate([ids, ids])[:, None]
    p[len(ids):, 0] = 0                             # all mass at the draft
    for i, x in enumerate(ids):
        if x < n:
            p[i, 0, x] = 0.75                       # (most of it: the rest is drawn)
            p[len(ids) + i, 0, x] = 0.5
    acc, tok = run_verify(drafts, p, u)
    assert not acc.any()
    for i, x in enumerate(ids):
        assert tok[len(ids) + i, 0] == (x if x < n else R.NO_TOKEN)


def test_verify_draws_the_targets_distribution():
    """Accepted drafts and redraws together follow the target's probabilities: with
    a grid of uniforms each token's share is off by less than the grid's step allows."""
    rng = np.random.default_rng(8)
    n, g = 6, 128
    p, q = probs(rng, 1, 2, n)[0], probs(rng, 1, 1, n)[0]
    grid = ((np.arange(g) + 0.5) / g).astype(F32)
    share = np.zeros(n)
    for x in range(n):
        u = np.stack(np.meshgrid(grid, grid), -1).reshape(-1, 2).astype(F32)
        b = len(u)
        acc, tok = run_verify(np.full((b, 1), x, np.uint32), np.tile(p, (b, 1, 1)), u,
                              np.tile(q, (b, 1, 1)))
        share += q[0, x] * np.bincount(tok[:, 0], minlength=n)[:n] / b
    # each acceptance rate is off by a grid step at most, and each redraw's share
    assert np.abs(share - p[0]).max() <= 4.0 / g


@pytest.mark.parametrize("n", [5000, 40000])
def test_sampling_graph_replays(n):
    """softmax and verification captured, replayed on new logits and uniforms."""
    L, Q, torch = mods()
    rng = np.random.default_rng(12)
    b, k = 3, 4
    x = torch.zeros(b * (k + 1), n, device="cuda")
    probs_t, u = torch.zeros_like(x), torch.zeros(b, k + 1, device="cuda")
    drafts = torch.zeros(b, k, dtype=torch.int32, device="cuda")
    tok = torch.zeros(b, k + 1, dtype=torch.int32, device="cuda")
    acc = torch.zeros(b, dtype=torch.int32, device="cuda")

    def step():
        L.softmax(x, probs_t, temperature=0.8)
        L.verify_drafts(drafts, probs_t.view(b, k + 1, n), u, tok, acc)

    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            step()
    for _ in range(5):
        z = (rng.standard_normal((b * (k + 1), n)) * 6).astype(F32)
        z[1, ::3] = -np.inf
        x.copy_(dev(z))
        d = z.reshape(b, k + 1, n)[:, :k].argmax(2)
        drafts.copy_(dev(d.astype(np.int32)))
        uu = rng.random((b, k + 1)).astype(F32)
        u.copy_(dev(uu))
        graph.replay()
        torch.cuda.synchronize()
        g_tok, g_acc, g_probs = tok.clone(), acc.clone(), probs_t.clone()
        step()
        # (longer rows' captured softmax takes other launches, to the same bits)
        assert torch.equal(g_probs, probs_t)
        assert torch.equal(g_tok, tok) and torch.equal(g_acc, acc)
        pr = host(probs_t).reshape(b, k + 1, n)
        for i in range(b):
            a, t = R.verify(d[i].astype(np.uint32), pr[i], uu[i])
            assert int(g_acc[i]) == a and np.array_equal(host(g_tok[i]).view(np.uint32), t)
