"""Unaligned device arrays are refused by every call of the 4-bit cache and of the
decode loop over it, and nothing is launched (under the stand-in for the HIP runtime,
fake_hip.c).  Each check runs in a process of its own."""
import ctypes as C
import os
import subprocess
import sys

import pytest

from test_host_calls_cpu import OUT, STREAM, X, fake  # noqa: F401
from test_kv4_host_cpu import W, Kv4


def refused(h, call, args, names):
    """`call` of the arguments is accepted, and refused with any one of `names` off by
    1 to 3 bytes."""
    h.m.check(call(*args.values(), STREAM))
    at = h.f.fake_launches()
    for name in names:
        for off in (1, 2, 3):
            a = dict(args)
            a[name] += off
            assert h.status(call(*a.values(), STREAM)) == "InvalidArgument", (name, off)
    assert h.f.fake_launches() == at


def check_evict(h):
    a, b = h.cache(), h.cache(max_seq=20)
    args = dict(src=a, dst=b, w=X, wo=W, lens=X, lo=OUT, keep=10, recent=2, kept=OUT)
    refused(h, h.lib.mri_kv4_evict, args, ("w", "wo", "lens", "lo", "kept"))


def check_verify(h):
    args = dict(drafts=X, q=X, p=X, u=X, counts=X, seqs=2, k=3, n=9, tokens=OUT, accepted=OUT)
    refused(h, h.lib.mri_verify_drafts, args,
            ("drafts", "q", "p", "u", "counts", "tokens", "accepted"))


def check_attend_in_place(h):
    """The weights read q once more after the output is written: not over q."""
    c = h.cache()
    r = h.rows(rows=3)
    args = dict(c=c, layer=0, rows=r, q=X, qs=256, heads=4, out=X, os=256)
    h.m.check(h.lib.mri_kv4_attend(*args.values(), None, STREAM))
    at = h.f.fake_launches()
    assert h.status(h.lib.mri_kv4_attend(*args.values(), W, STREAM)) == "InvalidArgument"
    assert h.status(h.lib.mri_kv4_attend(*dict(args, os=257).values(), None, STREAM)) \
        == "InvalidArgument"
    assert h.f.fake_launches() == at


def check_forward(h):
    L, d, vocab = h.L, 128, 64
    floats = (C.c_float * (vocab * d))()

    def w(n, k):
        return L.WeightRef(L.Q4_0, W, n, k)

    cfg = L.Config(d, 2, 1, 256, vocab, 32, 1e-5, 1e4, 1)
    m = C.c_void_p()
    h.m.check(h.lib.mri_llama_create(C.byref(cfg), floats, floats, w(vocab, d), C.byref(m)))
    refs = (L.WeightRef * 7)(w(d, d), w(64, d), w(64, d), w(d, d), w(256, d), w(256, d), w(d, 256))
    h.m.check(h.lib.mri_llama_set_layer(m, 0, floats, floats, refs))
    toks = (C.c_uint32 * 4)(1, 2, 3, 4)
    for n in (1, 4):
        args = dict(m=m, tokens=toks, n=n, start=0, cache=h.cache(1, 1, 32, 1, 64), seq=0, at=0,
                    weights=X, logits=OUT)
        refused(h, h.lib.mri_llama_forward_kv4, args, ("weights", "logits"))
        h.m.check(h.lib.mri_llama_forward_kv4(*dict(args, weights=None).values(), STREAM))


CHECKS = [n for n in dir() if n.startswith("check_")]


@pytest.mark.parametrize("check", CHECKS)
def test_alignment(fake, check):  # noqa: F811
    r = subprocess.run([sys.executable, os.path.abspath(__file__), fake, check],
                       capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr


if __name__ == "__main__":
    globals()[sys.argv[2]](Kv4(sys.argv[1]))
