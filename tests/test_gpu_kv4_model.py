"""The decoder model on a 4-bit cache (mri_llama_forward_kv4), and a decode loop
of all its operators, against the oracle with its keys and values quantized as the
cache does (kv4_ref.py).

Tolerance: the bound is test_gpu_llama.py's 2e-2 of the largest logit.  With Q4_0
weights (f32 activations) rounding moves next to nothing.  The other formats quantize
activations: a last-bit difference moves one of them by a step of 1 / 127 of its row's
largest, which moves every key of the next layer's row by up to that part of its own
largest, and 1 / 127 is a sixteenth of a 4-bit step (1 / 8 of a block's largest), so that
one key element in sixteen moves by a whole 4-bit step.  The oracle has this spread by
itself: with its attention rows off by 2^-22 of their value, as f32 sums are, its own
logits move by up to 4e-2 (INT8, two layers).  Those formats are held to three times the
spread that the oracle shows under such roundings, where that is more than the bound."""
import numpy as np
import pytest

import kv4_ref as R
import oracle_lib as O
from gpu_util import dev, empty, host
from test_gpu_llama import build, close

pytestmark = pytest.mark.gpu

F32 = np.float32
TOL = 2e-2


class Kv4Oracle(O.LlamaOracle):
    """LlamaOracle whose cache holds what the 4-bit blocks stand for, at positions
    `shift` below the rotary ones."""

    def __init__(self, o):
        self.__dict__.update(o.__dict__)
        self.k_cache, self.v_cache = np.zeros_like(o.k_cache), np.zeros_like(o.v_cache)
        self.shift = 0
        self.noise = None   # random numbers: attention rows off by roundings
        nl, n = len(self.layers), self.cfg["max_seq"]
        self.weights = np.zeros((nl, self.cfg["n_kv_heads"], n))

    def block(self, li, x, start_pos):
        c, L = self.cfg, self.layers[li]
        nh, nkv, hd = c["n_heads"], c["n_kv_heads"], c["head_dim"]
        seq, at = x.shape[0], start_pos - self.shift
        normed = O.rmsnorm(x, L["attn_norm"], c["eps"])
        q = O.rope_apply(L["wq"](normed), nh, hd, self.cos, self.sin, start_pos)
        k = O.rope_apply(L["wk"](normed), nkv, hd, self.cos, self.sin, start_pos)
        self.k_cache[li, at:at + seq] = R.stored(k)
        self.v_cache[li, at:at + seq] = R.stored(L["wv"](normed))
        end = at + seq
        kk, vv = (t[li, :end].reshape(end, nkv, hd).astype(np.float64)
                  for t in (self.k_cache, self.v_cache))
        attn, w, _, _ = R.attend(q, kk, vv, at, nh)
        if self.noise is not None:
            attn = attn * (1 + 2.0 ** -22 * self.noise.standard_normal(attn.shape))
        self.weights[li, :, at:end] = 0
        self.weights[li, :, :end] += w
        x = x + L["wo"](attn.astype(F32))
        normed = O.rmsnorm(x, L["ffn_norm"], c["eps"])
        return x + L["wdown"](O.swiglu(L["wgate"](normed), L["wup"](normed)))

    def evict(self, kept):
        """kept [layers, n_kv, keep] positions."""
        hd = self.cfg["head_dim"]
        for li in range(kept.shape[0]):
            for g in range(kept.shape[1]):
                at, lane = kept[li, g], slice(g * hd, (g + 1) * hd)
                for t in (self.k_cache, self.v_cache):
                    t[li, :len(at), lane] = t[li, at, lane]
                self.weights[li, g, :len(at)] = self.weights[li, g, at]


@pytest.mark.parametrize("fmt,hd", [("q4_0", 64), ("q8_0", 64), ("int8", 128), ("w4a8", 64),
                                    ("mixed", 64)])
def test_forward_kv4(fmt, hd):
    """A prompt, decode steps and a chunk of rows on one sequence of a cache of three;
    the others stay empty."""
    import torch as t
    oracle, gpu, rng = build(fmt, seed=7, d=4 * hd, nh=4, nkv=2, max_seq=100)
    ref = Kv4Oracle(oracle)
    toks = rng.integers(0, 300, 90).tolist()
    off = [Kv4Oracle(oracle) for _ in range(3 if fmt != "q4_0" else 0)]
    for i, o in enumerate(off):
        o.noise = np.random.default_rng(i)
    cache = gpu.kv4_cache(n_seqs=3, max_seq=96)
    w = t.zeros(2, 3, 2, 96, device="cuda")
    at = 0

    def held(got, want, others):
        spread = max([np.abs(o - want).max() / np.abs(want).max() for o in others] + [0])
        close(got, want, max(TOL, 3 * spread))

    for n in (70, 1, 1, 5, 1, 12):
        logits = empty((n, 300), t.float32)
        gpu.forward_kv4(toks[at:at + n], at, cache, logits, seq=1, weights=w)
        want = ref.forward_cached(toks[at:at + n], at)
        held(host(logits), want, [o.forward_cached(toks[at:at + n], at) for o in off])
        at += n
    held(host(w)[:, 1], ref.weights[:, :, :96], [o.weights[:, :, :96] for o in off])
    assert not host(w)[:, [0, 2]].any()
    k, v = (t.zeros(2, 3, 96, 2 * hd, device="cuda") for _ in range(2))
    cache.read(0, k, v, 0)
    assert not host(k)[:, [0, 2]].any() and not host(v)[:, [0, 2]].any()
    assert not host(k)[:, 1, at:].any()


def test_forward_kv4_equals_its_operators():
    """The one-layer model's logits through forward_kv4 do not change when the same rows
    come in other chunks, beyond f32 rounding carried through the layer."""
    import torch as t
    _, gpu, rng = build("q4_0", seed=11, max_seq=64, n_layers=1)
    toks = rng.integers(0, 300, 40).tolist()
    whole, parts = empty((40, 300), t.float32), empty((40, 300), t.float32)
    gpu.forward_kv4(toks, 0, gpu.kv4_cache(), whole)
    cache = gpu.kv4_cache()
    for i in range(0, 40, 8):
        gpu.forward_kv4(toks[i:i + 8], i, cache, parts[i:i + 8])
    close(host(parts), host(whole), TOL)


def test_forward_kv4_refusals():
    import mri_qmatmul as Q
    import torch as t
    _, gpu, rng = build("q4_0", max_seq=48)
    import mri_llama as L
    logits = empty((48, 300), t.float32)
    cache = gpu.kv4_cache(max_seq=40)

    def refused(kind, *a, **kw):
        with pytest.raises(Q.MriError) as e:
            gpu.forward_kv4(*a, **kw)
        assert e.value.kind == kind, e.value

    refused("InvalidShape", [], 0, cache, logits)
    refused("InvalidShape", [1] * 41, 0, cache, logits)                 # the cache's length
    refused("InvalidShape", [1] * 9, 40, cache, logits, cache_pos=0)    # the rotary table's
    refused("InvalidShape", [300], 0, cache, logits)                    # a token id
    refused("InvalidShape", [1], 0, cache, logits, seq=1)
    refused("ShapeMismatch", [1], 0, L.Kv4Cache(1, 1, 40, 2, 64), logits)
    refused("ShapeMismatch", [1], 0, L.Kv4Cache(2, 1, 40, 1, 128), logits)
    refused("InvalidShape", [1], 0, cache, logits, weights=t.zeros(2, 1, 2, 41, device="cuda"))
    c = L.Kv4Cache(1, 2, 40, 2, 64)
    x = t.zeros(2, 4, 128, device="cuda")
    q = t.zeros(2, 4, 192, device="cuda")

    def bad(kind, f, *a, **kw):
        with pytest.raises(Q.MriError) as e:
            f(*a, **kw)
        assert e.value.kind == kind, e.value

    bad("InvalidArgument", c.append, 1, x, x, 0)                        # no such layer
    bad("InvalidShape", c.append, 0, x, x, 37)                          # past the end
    bad("InvalidShape", c.append, 0, x, x, 0, first_seq=1)
    bad("InvalidShape", c.append, 0, x[..., :64], x[..., :64], 0)
    bad("InvalidArgument", c.append, 0, x.half(), x.half(), 0)
    bad("InvalidArgument", c.append, 0, x.cpu(), x.cpu(), 0)
    bad("InvalidShape", c.append, 0, x, x, t.zeros(3, dtype=t.int32, device="cuda"))
    bad("InvalidShape", c.attend, 0, q, q.clone(), 0)                   # 3 heads over 2
    bad("InvalidShape", c.attend, 0, x, x.clone(), -1)
    w = t.zeros(1, 2, 2, 40, device="cuda")
    n = t.zeros(2, dtype=t.int32, device="cuda")
    kept = t.zeros(1, 2, 2, 8, dtype=t.int32, device="cuda")
    small = L.Kv4Cache(1, 2, 8, 2, 64)
    bad("InvalidArgument", c.evict, c, w, w, n, n, 8, 9, kept)          # recent > keep
    bad("InvalidArgument", c.evict, c, w, w.clone(), n, n, 8, 2, kept)
    bad("InvalidShape", c.evict, small, w, w[..., :8].contiguous(), n, n, 9, 2,
        t.zeros(1, 2, 2, 9, dtype=t.int32, device="cuda"))
    bad("InvalidShape", c.evict, L.Kv4Cache(1, 2, 40, 1, 128), w, w[:, :, :1].contiguous(), n, n,
        8, 2, kept)


class CacheOracle(Kv4Oracle):
    """Kv4Oracle whose blocks attend to given keys and values: what a call does with
    its cache, apart from how rounding moves what it writes there."""

    def block(self, li, x, start_pos):
        own = R.stored
        try:
            at = start_pos - self.shift
            rows = iter((self.given_k[li, at:at + len(x)], self.given_v[li, at:at + len(x)]))
            R.stored = lambda _: next(rows)
            return super().block(li, x, start_pos)
        finally:
            R.stored = own


@pytest.mark.parametrize("fmt,hd", [("q4_0", 64), ("q4_0", 128), ("q8_0", 64), ("int8", 128),
                                    ("w4a8", 64), ("mixed", 64)])
def test_forward_kv4_cache_and_logits(fmt, hd):
    """What the call caches in the first layer, and its logits from what it cached.

    The first layer's keys and values come from the embedding rows: their activations
    differ from the oracle's by f32 rounding, which moves about one in 10^4 over a step of
    its int8 rounding.  Such a step is 1 / 127 of the row's largest activation, of 4 * hd
    that a key sums: under a hundredth of a key's usual size, where a 4-bit step is a third
    of it.  So nearly all quants equal the oracle's, and the others are a step off; a
    scale is at most an f16 rounding off, 2^-10 of the value.
    From the cache on, both compute the same attention and the same projections of it:
    the logits are as close as with an f32 cache, for every format (test_gpu_llama.py)."""
    import torch as t
    oracle, gpu, rng = build(fmt, seed=17, d=4 * hd, nh=4, nkv=2, max_seq=100)
    toks = rng.integers(0, 300, 83).tolist()
    cache = gpu.kv4_cache(n_seqs=2, max_seq=96)
    w = t.zeros(2, 2, 2, 96, device="cuda")
    got, at = [], 0
    for n in (64, 1, 5, 1, 12):
        logits = empty((n, 300), t.float32)
        gpu.forward_kv4(toks[at:at + n], at, cache, logits, seq=1, weights=w)
        got.append(host(logits))
        at += n
    k, v = (t.zeros(2, 2, 96, 2 * hd, device="cuda") for _ in range(2))
    cache.read(0, k, v, 0)
    ref = CacheOracle(oracle)
    ref.given_k, ref.given_v = host(k)[:, 1], host(v)[:, 1]
    free, done = Kv4Oracle(oracle), 0
    for part in got:
        n = len(part)
        close(part, ref.forward_cached(toks[done:done + n], done), TOL)
        free.forward_cached(toks[done:done + n], done)
        done += n
    close(host(w)[:, 1], ref.weights[:, :, :96], TOL)
    for mine, want in ((ref.given_k, free.k_cache), (ref.given_v, free.v_cache)):
        mine, want = mine[0, :at].reshape(-1, 32), want[0, :at].reshape(-1, 32)
        top = np.abs(want).max(1, keepdims=True)
        off = np.abs(mine - want)
        assert (off <= top * (1 / 8 + 2.0 ** -9)).all()
        assert (off > top * 2.0 ** -9).mean() <= 0.01


def test_forward_kv4_refuses_logits():
    """Logits that the call would write past, or of another type, place or layout."""
    import mri_qmatmul as Q
    import torch as t
    _, gpu, rng = build("q4_0", max_seq=48)
    cache = gpu.kv4_cache(max_seq=40)
    toks = [1, 2, 3]
    for kind, logits in (("InvalidShape", empty((2, 300), t.float32)),
                         ("InvalidShape", empty((3, 299), t.float32)),
                         ("InvalidArgument", empty((3, 300), t.float16)),
                         ("InvalidArgument", t.zeros(3, 300)),
                         ("InvalidArgument", empty((3, 600), t.float32)[:, ::2])):
        with pytest.raises(Q.MriError) as e:
            gpu.forward_kv4(toks, 0, cache, logits)
        assert e.value.kind == kind, e.value
    gpu.forward_kv4(toks, 0, cache, empty((4, 300), t.float32))


def test_speculative_decode_with_eviction():
    """The loop that the operators are for: a prompt with its keys' weights, steps
    of a token and three drafts, their softmax and verification, positions that
    advance by what was accepted, and evictions to a budget when the cache is full.
    The oracle follows the GPU's tokens and kept positions; each step's logits and
    weights are compared, the verification is recomputed from the probabilities
    and the kept positions from the weights."""
    import mri_llama as L
    import torch as t
    oracle, gpu, rng = build("q4_0", seed=13, max_seq=160, n_layers=2)
    ref = Kv4Oracle(oracle)
    keep, recent, k, full = 32, 8, 3, 64
    cache = gpu.kv4_cache(max_seq=full)
    w = t.zeros(2, 1, 2, full, device="cuda")
    lens = t.zeros(1, dtype=t.int32, device="cuda")
    kept = t.zeros(2, 1, 2, keep, dtype=t.int32, device="cuda")
    probs = empty((k + 1, 300), t.float32)
    tokens = t.zeros(1, k + 1, dtype=t.int32, device="cuda")
    acc = t.zeros(1, dtype=t.int32, device="cuda")
    logits = empty((40, 300), t.float32)
    prompt = rng.integers(0, 300, 40).tolist()
    gpu.forward_kv4(prompt, 0, cache, logits, weights=w)
    close(host(logits), ref.forward_cached(prompt, 0), TOL)
    token, pos, at, evictions, accepted = int(host(logits)[-1].argmax()), 40, 40, 0, 0
    for step in range(20):
        if at + k + 1 > full:
            lens.fill_(at)
            before = host(w)
            cache.evict(cache, w, w, lens, lens, keep, recent, kept)
            got = host(kept)[:, 0]
            for li in range(2):
                for g in range(2):
                    assert np.array_equal(got[li, g], R.evict(before[li, 0, g], at, keep, recent))
            assert lens.tolist() == [keep]
            ref.evict(got)
            at = keep
            evictions += 1
        ref.shift = pos - at
        # drafts: the first is likely, so that some are accepted
        drafts = rng.integers(0, 300, (1, k))
        part = logits[:k + 1]
        was = ref.weights.copy()
        peek = ref.forward_cached([token], pos)[0]
        drafts[0, 0] = int(peek.argmax())
        rows = [token] + drafts[0].tolist()
        gpu.forward_kv4(rows, pos, cache, part, cache_pos=at, weights=w)
        # the look ahead wrote the row's key and gave weights: taken back
        ref.weights[:] = was
        want = ref.forward_cached(rows, pos)
        close(host(part), want, TOL)
        end = at + k + 1
        close(host(w)[:, 0, :, :end], ref.weights[:, :, :end], TOL)
        L.softmax(part, probs, temperature=0.25)
        u = rng.random((1, k + 1)).astype(F32)
        L.verify_drafts(dev(drafts.astype(np.int32)), probs.view(1, k + 1, 300), dev(u), tokens,
                        acc)
        a, want_t = R.verify(drafts[0].astype(np.uint32), host(probs), u[0])
        got_t = host(tokens)[0].view(np.uint32)
        assert int(host(acc)[0]) == a and np.array_equal(got_t, want_t)
        token = int(got_t[a])
        pos += a + 1
        at += a + 1
        accepted += a
        assert np.isfinite(host(w)).all()
    assert evictions >= 1 and accepted >= 1
