"""Calls of the 4-bit cache larger than one launch, under the stand-in for the HIP
runtime (fake_hip.c): they run in parts that cover all of their pages.  Each check
runs in a process of its own."""
import os
import subprocess
import sys

import pytest

from test_host_calls_cpu import OUT, STREAM, X, fake  # noqa: F401
from test_kv4_host_cpu import W, Kv4


def workgroups(got, name):
    return sum(v[0] for n, v in got if name in n)


def check_read(h):
    """A whole cache read back in one call, as it is evicted in one call; and layers
    and sequences that one launch does not hold."""
    for layers, seqs, max_seq, kv in ((80, 256, 4608, 8), (3, 1 << 16, 640, 8), (1, 3, 1 << 24, 31)):
        c = h.cache(layers=layers, seqs=seqs, max_seq=max_seq, kv=kv, hd=64)
        got = h.launched(lambda: h.lib.mri_kv4_read(
            c, 0, layers, h.rows(seqs=seqs, rows=max_seq), OUT, OUT, kv * 64, STREAM))
        need = layers * seqs * kv * (max_seq // 64)
        assert len(got) > 1 and need <= workgroups(got, "k_kv4_read") <= 1.01 * need


def check_append(h):
    for seqs, max_seq, kv in ((1 << 16, 640, 8), (3, 1 << 24, 31)):
        c = h.cache(layers=1, seqs=seqs, max_seq=max_seq, kv=kv, hd=64)
        for pos in (None, X):
            got = h.launched(lambda: h.lib.mri_kv4_append(
                c, 0, h.rows(seqs=seqs, rows=max_seq, pos=pos), X, X, kv * 64, STREAM))
            need = seqs * kv * (max_seq // 64)
            assert len(got) > 1 and need <= workgroups(got, "k_kv4_append") <= 1.2 * need


def check_attend(h):
    """Prompts of more queries than a launch's workgroups take, few rows of more
    sequences, with weights and without."""
    c = h.cache(layers=1, seqs=512, max_seq=32768, kv=8, hd=64)
    for pos in (None, X):
        got = h.launched(lambda: h.lib.mri_kv4_attend(
            c, 0, h.rows(seqs=512, rows=32768, pos=pos), X, 40 * 64, 40, OUT, 40 * 64, None,
            STREAM))
        assert len(got) > 1 and workgroups(got, "k_kv4_prompt") >= 512 * 8 * 32768 * 5 // 64
    c = h.cache(layers=1, seqs=1 << 20, max_seq=64, kv=8, hd=64)
    for weights in (None, W):
        got = h.launched(lambda: h.lib.mri_kv4_attend(
            c, 0, h.rows(seqs=1 << 20, rows=1, pos=X), X, 8 * 64, 8, OUT, 8 * 64, weights,
            STREAM))
        assert workgroups(got, "k_kv4_attend") == 8 << 20
    # the pages of one sequence that its weights go over
    c = h.cache(layers=1, seqs=1, max_seq=1 << 28, kv=13, hd=64)
    got = h.launched(lambda: h.lib.mri_kv4_attend(
        c, 0, h.rows(rows=1, pos=X), X, 13 * 64, 13, OUT, 13 * 64, W, STREAM))
    assert workgroups(got, "k_kv4_weights") == 13 << 20


def check_evict(h):
    """More heads of layers and sequences than a launch takes: all are chosen before
    the first is moved (in place, moving stores the new lengths over the old)."""
    c = h.cache(layers=80, seqs=8192, max_seq=128, kv=8, hd=64)
    d = h.cache(layers=80, seqs=8192, max_seq=64, kv=8, hd=64)
    for dst, wo, lens in ((d, W, OUT), (c, X, X)):
        got = h.launched(lambda: h.lib.mri_kv4_evict(c, dst, X, wo, X, lens, 64, 8, OUT, STREAM))
        names = [n for n, _ in got]
        first = min(i for i, n in enumerate(names) if "move" in n)
        assert all("select" in n for n in names[:first])
        assert all("move" in n for n in names[first:])
        assert workgroups(got, "select") == workgroups(got, "move") == 80 * 8192 * 8


CHECKS = [n for n in dir() if n.startswith("check_")]


@pytest.mark.parametrize("check", CHECKS)
def test_kv4_parts(fake, check):  # noqa: F811
    r = subprocess.run([sys.executable, os.path.abspath(__file__), fake, check],
                       capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr


if __name__ == "__main__":
    globals()[sys.argv[2]](Kv4(sys.argv[1]))
