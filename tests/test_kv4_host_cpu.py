"""What the 4-bit cache's and the sampling operators' calls do on the host, under the
stand-in for the HIP runtime (fake_hip.c): their refusals on a live cache, the
memory they take and the launches they make.  Each check runs in a process of its
own."""
import ctypes as C
import os
import subprocess
import sys

import pytest

from test_host_calls_cpu import OUT, STREAM, W, X, Host, fake  # noqa: F401


class Kv4(Host):
    def __init__(self, so):
        super().__init__(so)
        import mri_llama
        self.L = mri_llama
        self.lib = mri_llama.lib()

    def cache(self, layers=2, seqs=3, max_seq=100, kv=2, hd=64):
        h = C.c_void_p()
        self.m.check(self.lib.mri_kv4_cache_create(layers, seqs, max_seq, kv, hd, C.byref(h)))
        return h

    def rows(self, first=0, seqs=1, rows=1, start=0, pos=None, count=None):
        return C.byref(self.L.Kv4Rows(first, seqs, rows, start, pos, count))

    def status(self, rc):
        return self.m.STATUS.get(rc, rc)

    def launched(self, rc_of):
        at = self.f.fake_launches()
        self.m.check(rc_of())
        got = self.launches(at)
        for name, v in got:
            assert v[0] * v[3] < 2**32 and v[1] == v[2] == 1, (name, v)
        return got


def check_row_refusals(h):
    """Layers, sequences, positions, strides, pointers: refused, and nothing launched."""
    c = h.cache()

    def calls(layer, r, stride=128, p=X, heads=4):
        yield h.lib.mri_kv4_append(c, layer, r, p, p, stride, STREAM)
        yield h.lib.mri_kv4_read(c, layer, 1, r, p, p, stride, STREAM)
        yield h.lib.mri_kv4_attend(c, layer, r, p, 2 * stride, heads, p, 2 * stride, None, STREAM)

    def refused(kind, *a, **kw):
        at = h.f.fake_launches()
        assert [h.status(rc) for rc in calls(*a, **kw)] == [kind] * 3, (kind, a, kw)
        assert h.f.fake_launches() == at

    refused("InvalidArgument", 2, h.rows())                       # no such layer
    refused("InvalidArgument", 0, None)
    refused("InvalidShape", 0, h.rows(first=3))
    refused("InvalidShape", 0, h.rows(first=2, seqs=2))
    refused("InvalidShape", 0, h.rows(first=2**64 - 1, seqs=1))
    refused("InvalidShape", 0, h.rows(rows=101))
    refused("InvalidShape", 0, h.rows(start=100))
    refused("InvalidShape", 0, h.rows(rows=1, start=2**64 - 1))
    refused("InvalidShape", 0, h.rows(rows=2**30 + 1, pos=X))
    refused("InvalidArgument", 0, h.rows(pos=X + 2))
    refused("InvalidArgument", 0, h.rows(count=X + 1))
    refused("InvalidShape", 0, h.rows(rows=2), stride=127)
    refused("InvalidArgument", 0, h.rows(), p=None)
    refused("InvalidArgument", 0, h.rows(), p=X + 2)
    attend = h.lib.mri_kv4_attend
    for heads, want in ((0, "InvalidShape"), (3, "InvalidShape"), (2**21, "Unsupported")):
        assert h.status(attend(c, 0, h.rows(), X, 2**28, heads, OUT, 2**28, None, STREAM)) == want
    assert h.status(attend(c, 0, h.rows(rows=2**29, pos=X), X, 2**20, 2**13, OUT, 2**20, None,
                           STREAM)) == "Unsupported"
    assert h.status(attend(c, 0, h.rows(), X, 256, 4, OUT, 256, X + 2, STREAM)) \
        == "InvalidArgument"
    assert h.status(h.lib.mri_kv4_read(c, 1, 2, h.rows(), X, X, 128, STREAM)) == "InvalidArgument"
    # nothing to do: accepted, nothing launched
    at = h.f.fake_launches()
    for r in (h.rows(rows=0), h.rows(seqs=0), h.rows(rows=0, start=100)):
        assert list(calls(0, r, p=None)) == [0, 0, 0]
    assert h.f.fake_launches() == at


def check_evict_refusals(h):
    a, small = h.cache(), h.cache(max_seq=20)
    evict = h.lib.mri_kv4_evict

    def st(src, dst, w=X, wo=W, lens=X, lo=OUT, keep=10, recent=2, kept=OUT):
        return h.status(evict(src, dst, w, wo, lens, lo, keep, recent, kept, STREAM))

    at = h.f.fake_launches()
    assert st(a, small, recent=11) == "InvalidArgument"
    assert st(a, small, wo=X) == "InvalidArgument"          # only in place
    assert st(a, a, wo=W) == "InvalidArgument"
    assert st(a, small, keep=0) == st(a, small, keep=21, recent=0) == "InvalidShape"
    for other in (h.cache(layers=1), h.cache(seqs=2), h.cache(kv=1), h.cache(hd=128)):
        assert st(a, other) == "InvalidShape"
    for name in ("w", "wo", "lens", "lo", "kept"):
        assert st(a, small, **{name: None}) == "InvalidArgument"
    assert h.f.fake_launches() == at
    assert st(a, small) == 0 and st(a, a, wo=X, keep=100) == 0


def check_memory(h):
    """A cache holds four allocations, its bytes as reported; calls take none; a
    creation whose memory is refused gives back what it took; destruction all."""
    before = h.live()
    c = h.cache()
    held = h.live() - before
    assert len(held) == 4
    got = sum(h.f.fake_alloc_bytes(i) for i in held)
    assert got == h.lib.mri_kv4_cache_device_bytes(c)
    big = h.cache(max_seq=100)
    n = len(h.live())
    for rows in (1, 5, 90):
        r = h.rows(seqs=3, rows=rows)
        h.m.check(h.lib.mri_kv4_append(c, 0, r, X, X, 128, STREAM))
        h.m.check(h.lib.mri_kv4_attend(c, 0, r, X, 256, 4, OUT, 256, W, STREAM))
        h.m.check(h.lib.mri_kv4_read(c, 0, 2, r, OUT, OUT, 128, STREAM))
    h.m.check(h.lib.mri_kv4_evict(c, big, X, W, X, OUT, 9, 1, OUT, STREAM))
    assert len(h.live()) == n
    h.set("fake_refuse_malloc", 1)
    p = C.c_void_p(7)
    assert h.status(h.lib.mri_kv4_cache_create(1, 1, 8, 1, 64, C.byref(p))) == "HipError"
    assert not p.value and len(h.live()) == n
    h.set("fake_refuse_malloc", 0)
    h.lib.mri_kv4_cache_destroy(c)
    h.lib.mri_kv4_cache_destroy(big)
    assert h.live() == before


def check_attend_forms(h):
    """One launch a call, two with weights; few queries split their keys over a
    workgroup a CU at most, large prompts do not."""
    c = h.cache(layers=1, seqs=64, max_seq=4096, kv=8, hd=128)

    def go(seqs, rows, heads, weights=None, pos=None):
        return h.launched(lambda: h.lib.mri_kv4_attend(
            c, 0, h.rows(seqs=seqs, rows=rows, pos=pos), X, heads * 128, heads, OUT, heads * 128,
            weights, STREAM))

    (name, v), = go(1, 1, 32)
    assert "k_kv4_attend" in name and 8 < v[0] <= 256
    (name, _), = go(1, 2048, 32)
    assert "k_kv4_prompt" in name
    names = [name for name, _ in go(8, 5, 32, weights=W, pos=X)]
    assert len(names) == 2 and "attend" in names[0] and "weights" in names[1]
    # more (row, head) pairs than log-sum-exps are kept: calls of rows, in order
    names = [name for name, _ in go(64, 1024, 32, weights=W)]
    assert len(names) == 4 and all("weights" in n for n in names[1::2])


def check_large_batches(h):
    """Caches that take most of a card: grids within what a launch takes."""
    c = h.cache(layers=80, seqs=256, max_seq=4608, kv=8, hd=64)
    d = h.cache(layers=80, seqs=256, max_seq=4096, kv=8, hd=64)
    for dst, wo in ((d, W), (c, X)):
        names = h.launched(lambda: h.lib.mri_kv4_evict(c, dst, X, wo, X, OUT, 4096, 512, OUT,
                                                       STREAM))
        assert ["select" in names[0][0], "move" in names[1][0]] == [True, True]
    long = h.cache(layers=1, seqs=512, max_seq=2**21, kv=8, hd=64)
    got = h.launched(lambda: h.lib.mri_kv4_attend(
        long, 0, h.rows(seqs=512, rows=1, pos=X), X, 512, 8, OUT, 512, W, STREAM))
    groups = sum(v[0] for n, v in got if "weights" in n)
    assert len(got) > 2 and groups >= 512 * 8 * (2**21 // 256)


def check_softmax_forms(h):
    """Rows of up to 32768 logits in one launch without memory; few longer ones in
    parts, through 256 KiB of the stream's; a captured call and one whose memory is
    refused do the rows whole and take none; beside another stream's capture the memory
    comes without breaking it."""
    def go(rows, n):
        return [name for name, _ in h.launched(lambda: h.lib.mri_softmax(
            X, rows, n, n, C.c_float(1.0), OUT, n, STREAM))]

    h.set("fake_refuse_malloc", 1)
    assert ["k_softmax_row" in n for n in go(3, 40000)] == [True]
    h.set("fake_refuse_malloc", 0)
    h.set("fake_capturing", 1)
    assert ["k_softmax_row" in n for n in go(3, 40000)] == [True] and not h.live()
    h.set("fake_capturing", 0)
    h.set("fake_other_capture", 1)
    names = go(3, 40000)
    assert ["stats" in n for n in names] == [True, False] and "write" in names[1]
    assert C.c_int.in_dll(h.f, "fake_broken_captures").value == 0
    h.set("fake_other_capture", 0)
    assert [h.f.fake_alloc_bytes(i) for i in h.live()] == [1 << 18]
    assert len(go(511, 1 << 22)) == 2 and len(go(511, 200000)) == 2
    assert len(h.live()) == 1
    assert ["k_softmax_row" in n for n in go(512, 40000)] == [True]     # rows enough
    for n in (1, 4096, 4097, 8192, 8193, 16384, 16385, 32768):
        assert ["k_softmax_held" in name for name in go(3, n)] == [True]
    assert len(h.live()) == 1


CHECKS = [n for n in dir() if n.startswith("check_")]


@pytest.mark.parametrize("check", CHECKS)
def test_kv4_host(fake, check):  # noqa: F811
    r = subprocess.run([sys.executable, os.path.abspath(__file__), fake, check],
                       capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr


if __name__ == "__main__":
    globals()[sys.argv[2]](Kv4(sys.argv[1]))
