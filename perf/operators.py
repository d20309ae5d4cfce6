"""The decode loop's operators on a 4-bit KV cache: what they are timed on.

One loop uses them together.  The rows of a step (a prompt, one token, or a token
and the drafts after it) are appended to the cache in 4-bit blocks; their queries
attend to it and add up how much weight each cached key got; the logits become
probabilities; drafted tokens are verified against them; and when a cache is full the
keys of least weight are evicted.

A cache block is 32 consecutive values of one head's key or value vector: an f16
scale d and 32 quants in [-8, 7].  With mx and mn the block's extremes and
a = mx if mx >= -mn else mn, d = f16(a / -8) and quant = clamp(rint(x / d), -8, 7).
"""
import math
import os
import sys

import numpy as np
import torch

own = False

QK = 32
NO_TOKEN = -1   # 0xffffffff as int32


# ---------------------------------------------------------------- cases
def append(seqs, rows, kv_heads, head_dim, pos, ragged, name=None):
    c = {"op": "append", "seqs": seqs, "rows": rows, "kv_heads": kv_heads, "head_dim": head_dim,
         "pos": pos, "ragged": ragged}
    return dict(c, name=name) if name else c


def attend(seqs, rows, heads, kv_heads, head_dim, pos, ragged, weights, name=None):
    c = {"op": "attend", "seqs": seqs, "rows": rows, "heads": heads, "kv_heads": kv_heads,
         "head_dim": head_dim, "pos": pos, "ragged": ragged, "weights": weights}
    return dict(c, name=name) if name else c


def evict(layers, seqs, kv_heads, head_dim, length, keep, recent, ragged, name=None):
    c = {"op": "evict", "layers": layers, "seqs": seqs, "kv_heads": kv_heads,
         "head_dim": head_dim, "length": length, "keep": keep, "recent": recent, "ragged": ragged}
    return dict(c, name=name) if name else c


def softmax(rows, n, temperature, name=None):
    c = {"op": "softmax", "rows": rows, "n": n, "temperature": temperature}
    return dict(c, name=name) if name else c


def verify(seqs, drafts, n, greedy_drafts, ragged, name=None):
    c = {"op": "verify", "seqs": seqs, "drafts": drafts, "n": n, "greedy_drafts": greedy_drafts,
         "ragged": ragged}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one decode step of one sequence: its 32 heads' key and value rows, written
        # and read back; launches and latency
        append(1, 1, 32, 128, 600, False, "append_token"),
        # two prompts at once, padded to the longer
        append(2, 2048, 32, 128, 0, True, "append_prompts"),
        # one decode step of a 4096-wide model at 600 positions: the smallest attention
        attend(1, 1, 32, 32, 128, 600, False, False, "attend_token"),
        # a speculative step of a batch: a token and four drafts a sequence, positions
        # that differ, grouped heads of 64, the keys' weights kept for eviction
        attend(16, 5, 32, 4, 64, 4000, True, True, "attend_drafts"),
        # single tokens over long caches, grouped heads
        attend(8, 1, 32, 8, 128, 32768, True, False, "attend_long"),
        # a prompt of odd length with its weights, as before an eviction
        attend(1, 1999, 32, 32, 128, 0, False, True, "attend_prompt"),
        # the whole model's cache a little over its budget, between two decode steps
        evict(32, 1, 8, 128, 2304, 2048, 512, False, "evict_step"),
        # long prompts cut to a small budget after their prefill
        evict(4, 4, 8, 128, 32768, 1024, 256, True, "evict_long"),
        # the probabilities of one speculative step's rows, and of a large batch's
        softmax(5, 32000, 0.8, "softmax_step"),
        softmax(320, 100003, 1.0, "softmax_batch"),
        # verification of four drafts of one sequence, and of a batch's
        verify(1, 4, 32000, False, False, "verify_step"),
        verify(64, 7, 100003, False, True, "verify_batch"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """The same operators over the same ranges: 1 to 32 sequences of 1 to 32768
    positions, 1 to 2048 rows, 1 to 32 key heads of 64 or 128 with 1 to 8 query heads
    each, vocabularies up to 131072, budgets from a handful of keys on."""
    most = {c["op"]: max(work(x)["bytes"] for x in listed() if x["op"] == c["op"])
            for c in listed()}
    most_flops = max(work(c)["flops"] for c in listed())
    op = rng.choice(("append", "attend", "attend", "attend", "evict", "softmax", "verify"))
    while True:
        hd, kv = rng.choice((64, 128)), rng.choice((1, 2, 4, 5, 8, 32))
        ragged = rng.random() < 0.5
        if op == "append":
            c = append(_log(rng, 1, 32), _log(rng, 1, 2048), kv, hd, _log(rng, 1, 4000) - 1,
                       ragged)
        elif op == "attend":
            rows = rng.choice((1, 1, rng.randint(2, 8), _log(rng, 9, 2048)))
            c = attend(_log(rng, 1, 32), rows, kv * rng.choice((1, 2, 3, 4, 7, 8)), kv, hd,
                       _log(rng, 1, 32768) - 1, ragged, rng.random() < 0.4)
        elif op == "evict":
            length = _log(rng, 2, 32768)
            keep = rng.randint(1, max(1, min(length, 4096)))
            c = evict(rng.randint(1, 32), _log(rng, 1, 8), kv, hd, length, keep,
                      rng.randint(0, keep), ragged)
        elif op == "softmax":
            c = softmax(_log(rng, 1, 512), _log(rng, 1, 131072), rng.choice((0.5, 0.8, 1.0, 1.7)))
        else:
            c = verify(_log(rng, 1, 128), rng.randint(0, 8), _log(rng, 2, 131072),
                       rng.random() < 0.3, ragged)
        w = work(c)
        if w["bytes"] <= most[op] and w["flops"] <= most_flops and (
                op != "attend" or c["seqs"] * c["rows"] * c["heads"] * (c["pos"] + c["rows"])
                <= 1.5e8):
            return c


# ---------------------------------------------------------------- inputs
def _gen(seed, salt):
    g = torch.Generator(device="cuda")
    g.manual_seed((seed * 1000003 + salt) % (1 << 62))
    return g


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _lengths(case, seed, most, salt):
    """A length a sequence: `most`, or spread over [most / 4, most]."""
    if not case["ragged"]:
        return [most] * case["seqs"]
    r = np.random.default_rng([seed, salt])
    low = max(1, most // 4) if most else 0
    got = [int(v) for v in r.integers(low, most + 1, case["seqs"])]
    got[0] = most
    return got


def _counts(case, seed):
    return _lengths(case, seed, case["rows"], 3) if case["ragged"] else None


def _positions(case, seed):
    return _lengths(case, seed, case["pos"], 4)


def _int(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _max_seq(case):
    return case["pos"] + case["rows"] if case["op"] in ("append", "attend") else case["length"]


def _values(g, seqs, rows, heads, hd):
    """Keys or values as projections give them: a gain a channel, a few outliers."""
    x = _randn(g, seqs, rows, heads * hd)
    return x * (_randn(g, heads * hd) * 0.7).exp()


def _cache(layers, seqs, max_seq, kv_heads, head_dim):
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                    "mini-rust-inference_amd"))
    import mri_llama
    return mri_llama.Kv4Cache(layers, seqs, max_seq, kv_heads, head_dim)


def _raw(case, seed):
    """The f32 inputs of a case and its lengths, from the seed alone."""
    g, op = _gen(seed, 11), case["op"]
    if op == "append":
        b, m, kv, hd = (case[k] for k in ("seqs", "rows", "kv_heads", "head_dim"))
        return {"k": _values(g, b, m, kv, hd), "v": _values(g, b, m, kv, hd),
                "pos": _positions(case, seed), "count": _counts(case, seed)}
    if op == "attend":
        b, m, kv, hd = (case[k] for k in ("seqs", "rows", "kv_heads", "head_dim"))
        t, pos = _max_seq(case), _positions(case, seed)
        s = {"k": _values(g, b, t, kv, hd), "v": _values(g, b, t, kv, hd),
             "q": _randn(g, b, m, case["heads"] * hd), "pos": pos, "count": _counts(case, seed)}
        if case["weights"]:
            s["weights"] = torch.rand((b, kv, t), generator=g, device="cuda") * 3
        return s
    if op == "evict":
        a, b, kv, hd, t = (case[k] for k in ("layers", "seqs", "kv_heads", "head_dim", "length"))
        # accumulated weights: heavy for few keys, near nothing for most; some equal
        w = (_randn(g, a, b, kv, t) * 2.0 - 3).exp()
        w = torch.where(torch.rand(w.shape, generator=g, device="cuda") < 0.05,
                        torch.full_like(w, 0.0625), w)
        return {"k": _values(g, a * b, t, kv, hd).view(a, b, t, kv * hd),
                "v": _values(g, a * b, t, kv, hd).view(a, b, t, kv * hd),
                "weights": w, "lens": _lengths(case, seed, t, 5)}
    if op == "softmax":
        x = _randn(g, case["rows"], case["n"]) * 3
        # every third row comes filtered: all but its larger logits at -inf
        x[::3] = torch.where(x[::3] < x[::3].mean(1, keepdim=True), -math.inf, x[::3])
        return {"x": x}
    b, k, n = case["seqs"], case["drafts"], case["n"]
    lt = _randn(g, b, k + 1, n) * 2.5
    ld = lt[:, :k] + _randn(g, b, k, n) * 0.7
    target = torch.softmax(lt, 2)
    draft = torch.softmax(ld, 2)
    if case["greedy_drafts"]:
        drafts = draft.argmax(2)
    else:
        drafts = (draft.double().clamp_min(1e-30).log() - torch.empty_like(
            draft, dtype=torch.float64).exponential_(generator=g).log()).argmax(2)
    r = np.random.default_rng([seed, 6])
    return {"target": target, "draft": None if case["greedy_drafts"] else draft,
            "drafts": drafts.to(torch.int32),
            "u": torch.rand((b, k + 1), generator=g, device="cuda"),
            "n_drafts": [int(v) for v in r.integers(0, k + 1, b)] if case["ragged"] else None}


def _pack(x, kv, hd):
    """[..., rows, kv * hd] f32 in the plain cache's form: quants two a byte (of values
    i and i + 16 of a block), f16 scales."""
    q, d = _quantize(x.view(*x.shape[:-1], kv * hd // QK, QK))
    q = q + 8
    return (q[..., :16] + q[..., 16:] * 16).to(torch.uint8), d


def prepare(case, seed):
    s = _raw(case, seed)
    op = case["op"]
    s["case"] = case
    for name in ("pos", "count", "lens", "n_drafts"):
        if s.get(name) is not None:
            s[name] = _int(s[name])
    if op in ("append", "attend"):
        kv, hd, t = case["kv_heads"], case["head_dim"], _max_seq(case)
        shape = s["k"].shape if op == "append" else s["q"].shape
        s["out"] = torch.zeros(shape, device="cuda")
        if op == "append":
            s["out_v"] = torch.zeros(shape, device="cuda")
        if own:
            s["cache"] = _cache(1, case["seqs"], t, kv, hd)
        if op == "attend":
            if own:
                s["cache"].append(0, s["k"], s["v"], 0)
            else:
                s["k4"], s["v4"] = _pack(s["k"], kv, hd), _pack(s["v"], kv, hd)
            del s["k"], s["v"]
    if op == "evict":
        a, b, kv, hd, t = (case[k] for k in ("layers", "seqs", "kv_heads", "head_dim", "length"))
        if own:
            s["cache"], s["dst"] = _cache(a, b, t, kv, hd), _cache(a, b, case["keep"], kv, hd)
            for i in range(a):
                s["cache"].append(i, s["k"][i], s["v"][i], 0)
        else:
            s["k4"], s["v4"] = _pack(s["k"], kv, hd), _pack(s["v"], kv, hd)
        del s["k"], s["v"]
        s["out"] = torch.zeros((a, b, case["keep"], kv * hd), device="cuda")
        s["out_v"] = torch.zeros_like(s["out"])
        s["out_w"] = torch.zeros((a, b, kv, case["keep"]), device="cuda")
        s["kept"] = torch.zeros((a, b, kv, case["keep"]), dtype=torch.int32, device="cuda")
        s["new_lens"] = torch.zeros(b, dtype=torch.int32, device="cuda")
    if op == "softmax":
        s["out"] = torch.empty_like(s["x"])
    if op == "verify":
        s["tokens"] = torch.empty((case["seqs"], case["drafts"] + 1), dtype=torch.int32,
                                  device="cuda")
        s["accepted"] = torch.empty(case["seqs"], dtype=torch.int32, device="cuda")
    return s


# ---------------------------------------------------------------- plain forms
def _quantize(x):
    """Quants (as int16) and f16 scales of blocks [..., 32]."""
    mx, mn = x.amax(-1), x.amin(-1)
    d = (torch.where(mx >= -mn, mx, mn) * -0.125).clamp(-65504.0, 65504.0).to(torch.float16)
    # the division in 64 bits: a quotient of 32 can round onto a border between quants
    df = d.double()[..., None]
    q = torch.where(df == 0, torch.zeros_like(df), torch.round(x.double() / df))
    return q.clamp(-8, 7).to(torch.int16), d


def _unpack(packed):
    """[..., rows, kv * hd] f32 of what _pack made."""
    q, d = packed
    low, high = (q & 15).float() - 8, (q >> 4).float() - 8
    return (torch.cat((low, high), -1) * d.float()[..., None]).flatten(-2)


def _live(s):
    """Which rows are real, [seqs, rows]."""
    m = s["case"]["rows"]
    i = torch.arange(m, device="cuda")
    if s["count"] is None:
        return torch.ones((s["case"]["seqs"], m), dtype=torch.bool, device="cuda")
    return i[None] < s["count"][:, None]


def _plain_append(s):
    kv, hd = s["case"]["kv_heads"], s["case"]["head_dim"]
    live = _live(s)[..., None]
    back = []
    for x in (s["k"], s["v"]):
        q, d = _quantize(x.view(*x.shape[:-1], kv * hd // QK, QK))
        y = (q.float() * d.float()[..., None]).flatten(-2)
        back.append(torch.where(live, y, torch.zeros_like(y)))
    return back


def _plain_attend(s):
    c = s["case"]
    b, m, h, kv, hd = (c[k] for k in ("seqs", "rows", "heads", "kv_heads", "head_dim"))
    grp, t = h // kv, _max_seq(c)
    k = _unpack(s["k4"]).view(b, t, kv, hd).permute(0, 2, 3, 1).contiguous()
    v = _unpack(s["v4"]).view(b, t, kv, hd).permute(0, 2, 1, 3).contiguous()
    q = s["q"].view(b, m, kv, grp, hd).permute(0, 2, 1, 3, 4).reshape(b, kv, m * grp, hd)
    x = torch.matmul(q, k) * (1.0 / math.sqrt(hd))
    at = s["pos"][:, None].long() + torch.arange(m, device="cuda")[None]     # [b, m]
    seen = torch.arange(t, device="cuda")[None, None] <= at[..., None]       # [b, m, t]
    x = x.view(b, kv, m, grp, t).masked_fill_(~seen[:, None, :, None], -math.inf)
    x = (x - x.amax(-1, keepdim=True)).exp_()
    p = x / x.sum(-1, keepdim=True)
    live = _live(s)
    o = torch.matmul(p.view(b, kv, m * grp, t), v).view(b, kv, m, grp, hd)
    o = o.permute(0, 2, 1, 3, 4).reshape(b, m, h * hd)
    o = torch.where(live[..., None], o, torch.zeros_like(o))
    if not c["weights"]:
        return o
    p = torch.where(live[:, None, :, None, None], p, torch.zeros_like(p))
    old = torch.arange(t, device="cuda")[None, None] < s["pos"][:, None, None]
    w = torch.where(old, s["weights"], torch.zeros_like(s["weights"]))
    new = w + p.sum((2, 3))
    # keys that no row sees keep what they had
    end = s["pos"].long() + (m if s["count"] is None else s["count"].long())
    past = torch.arange(t, device="cuda")[None] >= end[:, None]
    return o, torch.where(past[:, None], s["weights"], new)


def _plain_evict(s):
    c = s["case"]
    a, b, kv, hd, t, keep = (c[k] for k in ("layers", "seqs", "kv_heads", "head_dim", "length",
                                            "keep"))
    at = torch.arange(t, device="cuda")
    n = s["lens"].long()[None, :, None, None]
    over = n > keep
    # in order of weight; the recent ones (and all of a short cache) before any other,
    # what lies past the end behind them
    w = s["weights"]
    w = torch.where((at >= n - c["recent"]) | ~over, torch.full_like(w, math.inf), w)
    w = torch.where(at >= n, torch.full_like(w, -math.inf), w)
    order = torch.sort(w, dim=-1, descending=True, stable=True)[1][..., :keep]
    kept = torch.where(order < n, order, t).sort(-1)[0]                      # [a, b, kv, keep]
    live = kept < t
    i = kept.clamp(max=t - 1)
    new_w = torch.where(live, s["weights"].gather(3, i), torch.zeros_like(i, dtype=torch.float32))
    back = []
    for q, d in (s["k4"], s["v4"]):
        nb = hd // QK
        j = i.permute(0, 1, 3, 2)                                            # [a, b, keep, kv]
        q = q.view(a, b, t, kv, nb * 16).gather(2, j[..., None].expand(-1, -1, -1, -1, nb * 16))
        d = d.view(a, b, t, kv, nb).gather(2, j[..., None].expand(-1, -1, -1, -1, nb))
        y = _unpack((q.reshape(a, b, keep, kv * nb, 16), d.reshape(a, b, keep, kv * nb)))
        on = live.permute(0, 1, 3, 2)[..., None].expand(-1, -1, -1, -1, hd).reshape(y.shape)
        back.append(torch.where(on, y, torch.zeros_like(y)))
    kept = torch.where(live, kept, torch.full_like(kept, NO_TOKEN)).to(torch.int32)
    return kept, s["lens"].clamp(max=keep), new_w, back[0], back[1]


def _plain_softmax(s):
    x = s["x"]
    e = ((x - x.amax(1, keepdim=True)) / s["case"]["temperature"]).exp()
    return e / e.sum(1, keepdim=True)


def _plain_verify(s):
    c = s["case"]
    b, k, n = c["seqs"], c["drafts"], c["n"]
    # in 64 bits: products of two floats are exact, and a long sum decides between tokens
    u = s["u"].double()
    x = s["drafts"].long()
    px = s["target"][:, :k].gather(2, x[..., None])[..., 0].double()
    qx = torch.ones_like(px) if s["draft"] is None else \
        s["draft"].gather(2, x[..., None])[..., 0].double()
    count = torch.full((b,), k, device="cuda") if s["n_drafts"] is None else s["n_drafts"].long()
    i = torch.arange(k, device="cuda")[None]
    ok = (u[:, :k] * qx < px) & (i < count[:, None])
    got = ok.long().cumprod(1).sum(1)
    p = s["target"].gather(1, got[:, None, None].expand(-1, -1, n))[:, 0].double()
    r = p
    if k:
        at = got.clamp(max=k - 1)
        if s["draft"] is None:
            q = torch.zeros_like(p).scatter_(1, x.gather(1, at[:, None]), 1.0)
        else:
            q = s["draft"].gather(1, at[:, None, None].expand(-1, -1, n))[:, 0].double()
        r = torch.where((got < count)[:, None], (p - q).clamp_min(0), p)
        r = torch.where(r.sum(1, keepdim=True) > 0, r, p)
    sums = r.cumsum(1)
    t = torch.searchsorted(sums, u[:, k:] * sums[:, -1:], right=True)
    last = n - 1 - (r > 0).flip(1).to(torch.int8).argmax(1, keepdim=True)
    t = torch.minimum(t, last)
    j = torch.arange(k + 1, device="cuda")[None]
    row = torch.cat((x, x.new_zeros((b, 1))), 1)
    row = torch.where(j < got[:, None], row, torch.where(j == got[:, None], t, NO_TOKEN))
    return row.to(torch.int32), got.to(torch.int32)


# ---------------------------------------------------------------- one pass
def run(s):
    c = s["case"]
    op = c["op"]
    if not own:
        return {"append": _plain_append, "attend": _plain_attend, "evict": _plain_evict,
                "softmax": _plain_softmax, "verify": _plain_verify}[op](s)
    if op == "append":
        s["cache"].append(0, s["k"], s["v"], s["pos"], count=s["count"])
        s["cache"].read(0, s["out"], s["out_v"], s["pos"], count=s["count"])
        return [s["out"], s["out_v"]]
    if op == "attend":
        if not c["weights"]:
            s["cache"].attend(0, s["q"], s["out"], s["pos"], count=s["count"])
            return s["out"]
        w = s["weights"].clone()   # a pass starts from the same weights
        s["cache"].attend(0, s["q"], s["out"], s["pos"], count=s["count"], weights=w)
        return s["out"], w
    if op == "evict":
        s["cache"].evict(s["dst"], s["weights"], s["out_w"], s["lens"], s["new_lens"],
                         c["keep"], c["recent"], s["kept"])
        s["dst"].read(0, s["out"], s["out_v"], 0, count=s["new_lens"])
        return s["kept"], s["new_lens"], s["out_w"], s["out"], s["out_v"]
    import mri_llama
    if op == "softmax":
        mri_llama.softmax(s["x"], s["out"], temperature=c["temperature"])
        return s["out"]
    mri_llama.verify_drafts(s["drafts"], s["target"], s["u"], s["tokens"], s["accepted"],
                            draft_probs=s["draft"], n_drafts=s["n_drafts"])
    return s["tokens"], s["accepted"]


# ---------------------------------------------------------------- work
def work(case):
    op = case["op"]
    f4 = 18 / 32
    if op == "append":
        n = 2 * case["seqs"] * case["rows"] * case["kv_heads"] * case["head_dim"]
        if case["ragged"]:
            n *= 0.7    # rows that are real, at the mean
        return {"bytes": n * (4 + f4 + f4 + 4), "flops": 4.0 * n}
    if op == "attend":
        b, m, h, kv, hd, p = (case[k] for k in ("seqs", "rows", "heads", "kv_heads", "head_dim",
                                                "pos"))
        if case["ragged"]:
            p, m = 0.65 * p, max(1, 0.65 * m)
        keys = b * (p + m) * kv
        n = 2 * b * m * h * hd * 4 + keys * (2 * hd * f4 + (8 if case["weights"] else 0))
        return {"bytes": n, "flops": 4.0 * b * h * hd * m * (p + (m + 1) / 2)}
    if op == "evict":
        heads = case["layers"] * case["seqs"] * case["kv_heads"]
        n = (0.65 if case["ragged"] else 1) * case["length"]
        kept = min(n, case["keep"])
        hd = case["head_dim"]
        return {"bytes": heads * (4 * n + kept * (8 + 2 * hd * (3 * f4 + 4))),
                "flops": heads * (n + 2.0 * hd * kept)}
    if op == "softmax":
        return {"bytes": 8 * case["rows"] * case["n"], "flops": 5.0 * case["rows"] * case["n"]}
    rows = 1 if case["greedy_drafts"] else 2
    return {"bytes": case["seqs"] * (4 * rows * case["n"] + 16 * (case["drafts"] + 1)),
            "flops": 3.0 * case["seqs"] * case["n"]}


# ---------------------------------------------------------------- 64 bits
def _stored(x):
    """The values that the blocks along x's last axis stand for, in float64."""
    shape = x.shape
    x = x.double().reshape(-1, QK)
    hi, lo = x.max(1)[0], x.min(1)[0]
    a = torch.where(hi + lo >= 0, hi, lo)
    d = (a / -8).to(torch.float16).double()[:, None]
    q = torch.where(d != 0, x / torch.where(d != 0, d, 1.0), 0.0)
    return (q.round().clamp(-8, 7) * d).reshape(shape)


def exact(case, seed):
    s = _raw(case, seed)
    op = case["op"]
    if op == "append":
        got = [_stored(s["k"]), _stored(s["v"])]
        if s["count"] is not None:
            for b, n in enumerate(s["count"]):
                got[0][b, n:] = 0
                got[1][b, n:] = 0
        return got
    if op == "attend":
        h, kv, hd = case["heads"], case["kv_heads"], case["head_dim"]
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        w = s["weights"].double() if case["weights"] else None
        for b, pos in enumerate(s["pos"]):
            m = case["rows"] if s["count"] is None else s["count"][b]
            n = pos + m
            mask = torch.full((m, n), -math.inf, dtype=torch.float64, device="cuda").triu(pos + 1)
            k = _stored(s["k"][b, :n]).view(n, kv, hd)
            v = _stored(s["v"][b, :n]).view(n, kv, hd)
            if w is not None:
                w[b, :, pos:n] = 0
            for j in range(h):
                g = j * kv // h
                q = s["q"][b, :m, j * hd:(j + 1) * hd].double()
                p = torch.softmax(q @ k[:, g].T.contiguous() / math.sqrt(hd) + mask, 1)
                out[b, :m, j * hd:(j + 1) * hd] = p @ v[:, g].contiguous()
                if w is not None:
                    w[b, g, :n] += p.sum(0)
        return out if w is None else (out, w)
    if op == "evict":
        a, b, kv, hd, keep = (case[k] for k in ("layers", "seqs", "kv_heads", "head_dim", "keep"))
        w = s["weights"].double().cpu().numpy()
        kept = np.full((a, b, kv, keep), NO_TOKEN, np.int64)
        out = [torch.zeros((a, b, keep, kv * hd), dtype=torch.float64, device="cuda")
               for _ in range(2)]
        new_w = np.zeros((a, b, kv, keep))
        for i in range(a):
            for j in range(b):
                n = s["lens"][j]
                for g in range(kv):
                    if n <= keep:
                        at = np.arange(n)
                    else:
                        old = n - case["recent"]
                        top = np.argsort(-w[i, j, g, :old], kind="stable")
                        at = np.concatenate((np.sort(top[:keep - case["recent"]]),
                                             np.arange(old, n)))
                    kept[i, j, g, :len(at)] = at
                    new_w[i, j, g, :len(at)] = w[i, j, g, at]
                    at = torch.from_numpy(at).cuda()
                    lane = slice(g * hd, (g + 1) * hd)
                    out[0][i, j, :len(at), lane] = _stored(s["k"][i, j, at, lane])
                    out[1][i, j, :len(at), lane] = _stored(s["v"][i, j, at, lane])
        return (torch.from_numpy(kept).to(torch.int32),
                torch.tensor([min(n, keep) for n in s["lens"]], dtype=torch.int32),
                torch.from_numpy(new_w), out[0], out[1])
    if op == "softmax":
        return torch.softmax(s["x"].double() / case["temperature"], 1)
    k = case["drafts"]
    tokens = np.full((case["seqs"], k + 1), NO_TOKEN, np.int64)
    accepted = np.zeros(case["seqs"], np.int64)
    u, x = s["u"].double().cpu().numpy(), s["drafts"].cpu().numpy()
    for b in range(case["seqs"]):
        p = s["target"][b].double().cpu().numpy()
        q = None if s["draft"] is None else s["draft"][b].double().cpu().numpy()
        count = k if s["n_drafts"] is None else s["n_drafts"][b]
        i = 0
        while i < count and u[b, i] * (1.0 if q is None else q[i, x[b, i]]) < p[i, x[b, i]]:
            tokens[b, i] = x[b, i]
            i += 1
        accepted[b] = i
        r = p[i].copy()
        if i < count:
            if q is None:
                r[x[b, i]] = max(r[x[b, i]] - 1.0, 0.0)
            else:
                r = np.maximum(r - q[i], 0.0)
            if r.sum() == 0:
                r = p[i].copy()
        c = np.cumsum(r)
        t = int(np.searchsorted(c, u[b, k] * c[-1], side="right"))
        tokens[b, i] = min(t, int(np.flatnonzero(r > 0)[-1]))
    return (torch.from_numpy(tokens).to(torch.int32), torch.from_numpy(accepted).to(torch.int32))
