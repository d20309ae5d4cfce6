"""Calls of the 4-bit cache that take more than one launch (2^22 workgroups), against
64-bit restatements on the device over every sequence: the parts address their own
rows, sequences and heads.  Tolerances as in test_gpu_kv4.py."""
import pytest

pytestmark = pytest.mark.gpu

SEQS, KV, HD = (1 << 19) + 1000, 8, 64     # 2^22 heads and 8000 more
U = 2.0 ** -24


def stored(t, x):
    """What the blocks of 32 along the last axis stand for, f64."""
    b = x.double().view(*x.shape[:-1], -1, 32)
    hi, lo = b.amax(-1), b.amin(-1)
    d = (torch_where(t, hi >= -lo, hi, lo) / -8).to(t.float16).double()[..., None]
    q = torch_where(t, d != 0, b / torch_where(t, d != 0, d, 1.0), 0.0)
    return (q.round().clamp(-8, 7) * d).view(x.shape)


def torch_where(t, c, a, b):
    return t.where(c, a, b if isinstance(b, t.Tensor) else t.full_like(a, b))


def test_parts():
    import torch as t

    import mri_llama as L
    g = t.Generator(device="cuda")
    g.manual_seed(3)
    m, f, chunk = 3, KV * HD, 1 << 15
    c = L.Kv4Cache(1, SEQS, 64, KV, HD)
    k, v, q = (t.randn((SEQS, r, f), generator=g, device="cuda") for r in (m, m, 1))
    c.append(0, k, v, 0)
    bk, bv = t.full_like(k, 7.5), t.full_like(v, 7.5)
    c.read(0, bk, bv, 0)
    pos = (t.arange(SEQS, device="cuda") * 7 % m).to(t.int32)
    out = t.full_like(q, 7.5)
    w = t.rand((SEQS, KV, 64), generator=g, device="cuda")
    w0 = w.clone()
    c.attend(0, q, out, pos, weights=w)
    out2 = t.full_like(q, 7.5)
    c.attend(0, q, out2, pos)
    assert t.equal(out, out2)
    # in place, the lengths over the old ones: each head's heaviest of 3 and the last
    lens, keep = t.full((SEQS,), m, dtype=t.int32, device="cuda"), 2
    kept = t.zeros((1, SEQS, KV, keep), dtype=t.int32, device="cuda")
    we = w.clone()
    c.evict(c, we[None], we[None], lens, lens, keep, 1, kept)
    ek, ev = t.full_like(k, 7.5), t.full_like(v, 7.5)
    c.read(0, ek, ev, 0)
    assert bool((lens == keep).all())
    for i in range(0, SEQS, chunk):
        at = slice(i, min(i + chunk, SEQS))
        n = at.stop - at.start
        sk, sv = stored(t, k[at]), stored(t, v[at])
        assert t.equal(bk[at].double(), sk) and t.equal(bv[at].double(), sv)
        p = pos[at].long()
        sk4, sv4 = sk.view(n, m, KV, HD), sv.view(n, m, KV, HD)
        q4 = q[at].double().view(n, 1, KV, HD)
        s = (q4 * sk4).sum(-1) / 8                                   # [n, m, kv]
        top = ((q4 * sk4).abs().sum(-1) / 8).amax(1)                 # [n, kv]
        seen = (t.arange(m, device="cuda")[None] <= p[:, None])[..., None]
        e = t.exp(s.masked_fill(~seen, -1e300) - s.masked_fill(~seen, -1e300).amax(1, keepdim=True))
        pr = t.where(seen, e, t.zeros_like(e))
        pr = pr / pr.sum(1, keepdim=True)
        ref = (pr[..., None] * sv4).sum(1)
        mag = (pr[..., None] * sv4.abs()).sum(1)
        tiny = m * 2.0 ** -33 * sv4.abs().amax((1, 3))[..., None]
        tol = (160 * top.clamp_min(1) + 128)[..., None] * U * mag + tiny
        assert bool(((out[at].view(n, KV, HD).double() - ref).abs() <= tol).all()), i
        # weights: added before pos, stored at it, untouched past it
        old = w0[at, :, :m].double().permute(0, 2, 1)
        key = t.arange(m, device="cuda")[None, :, None]
        want = t.where(key < p[:, None, None], old, t.zeros_like(old)) + pr
        want = t.where(seen, want, old)
        got = w[at, :, :m].double().permute(0, 2, 1)
        assert bool(((got - want).abs() <= (160 * top.clamp_min(1).amax() + 8) * U
                     * (want + 1e-30)).all()), i
        # eviction: the heavier of keys 0 and 1 (the first if equal), then key 2
        first = (w[at, :, 1] > w[at, :, 0]).to(t.int32)              # [n, kv]
        assert t.equal(kept[0, at, :, 0], first) and bool((kept[0, at, :, 1] == 2).all())
        sel = first.long()[:, None, :, None].expand(-1, 1, -1, HD)
        for e_, s4 in ((ek, sk4), (ev, sv4)):
            e4 = e_[at].double().view(n, m, KV, HD)
            assert t.equal(e4[:, 0], s4.gather(1, sel)[:, 0]) and t.equal(e4[:, 1:], s4[:, [2, 2]])
        wk = w[at, :, :2].gather(2, first.long()[..., None])[..., 0]
        assert t.equal(we[at, :, 0], wk) and t.equal(we[at, :, 1], w[at, :, 2])
        assert t.equal(we[at, :, 2:], w[at, :, 2:])
