"""Calls of two host threads, under a stand-in for the HIP runtime
(fake_hip_threads.c): the launches of a call that passes data from one kernel to the
next through the stream's memory follow each other on the stream.  Each check runs in
a process of its own."""
import ctypes as C
import os
import subprocess
import sys
import threading

import pytest

from test_host_calls_cpu import HERE, OUT, STREAM, W, X, Host

CALLS = 12


class Threads(Host):
    def __init__(self, so):
        super().__init__(so)
        self.f.fake_launch_thread.restype = C.c_long
        import mri_llama
        self.llama = mri_llama.lib()

    def together(self, call):
        """The launches of CALLS calls a thread of two threads at once, each with its
        thread."""
        at, errors = self.f.fake_launches(), []
        start = threading.Barrier(2)

        def run():
            try:
                start.wait()
                for _ in range(CALLS):
                    self.m.check(call())
            except Exception as e:
                errors.append(e)

        threads = [threading.Thread(target=run) for _ in range(2)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        assert not errors, errors
        return [(name, self.f.fake_launch_thread(at + i))
                for i, (name, _) in enumerate(self.launches(at))]

    def ordered(self, call):
        """Both threads' calls make the launches that one call makes, each call's
        without others between them."""
        at = self.f.fake_launches()
        self.m.check(call())
        one = [name for name, _ in self.launches(at)]
        assert len(one) > 1, one
        got = self.together(call)
        assert len(got) == 2 * CALLS * len(one)
        assert len({t for _, t in got}) == 2
        for i in range(0, len(got), len(one)):
            part = got[i:i + len(one)]
            assert [n for n, _ in part] == one and len({t for _, t in part}) == 1, part


def check_softmax(h):
    """Rows in parts: their statistics, then the probabilities."""
    for stream in (None, STREAM):
        h.ordered(lambda: h.llama.mri_softmax(X, 3, 40000, 40000, C.c_float(1.0), OUT, 40000,
                                              stream))


def check_projections(h):
    """Activations quantized into the stream's scratch, then the product."""
    def dims(m, k):
        return (C.c_size_t * 2)(m, k)

    def int8(m, k, n):
        w = C.c_void_p()
        h.m.check(h.lib.mri_qmatrix_create_device(W, OUT, n, k, STREAM, C.byref(w)))
        return w

    h.ordered(h.q8_0(200, 4096, 6000))
    w = int8(200, 4096, 6000)
    h.ordered(lambda: h.lib.mri_matmul_int8_from_f32(X, dims(200, 4096), 2, w, OUT, None, None,
                                                     None, STREAM))
    odd = int8(3, 1000, 777)
    h.ordered(lambda: h.lib.mri_matmul_int8(X + 1, 3 * 1000, C.c_float(1.0), odd, 3, OUT, None,
                                            STREAM))
    h.ordered(lambda: h.lib.mri_matmul_int8(X + 1, 200 * 4096, C.c_float(1.0), w, 200, OUT, None,
                                            STREAM))
    h.ordered(lambda: h.lib.mri_quantize_symmetric(X, 1 << 22, OUT, W, STREAM))


def check_softmax_per_thread_stream(h):
    """The per-thread stream has one handle and a stream a thread: each thread has
    memory of its own, which its next call finds again."""
    stream, done = 2, threading.Barrier(2)   # hipStreamPerThread
    held = {}

    def run(i):
        for n in (40000, 50000):
            h.m.check(h.llama.mri_softmax(X, 3, n, n, C.c_float(1.0), OUT, n, stream))
        held[i] = True
        done.wait()     # both threads live until both have called

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(held) == 2
    assert [h.f.fake_alloc_bytes(i) for i in h.live()] == [1 << 18] * 2


CHECKS = [n for n in dir() if n.startswith("check_")]


@pytest.fixture(scope="module")
def fake(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("fake_hip") / "libfake_hip_threads.so")
    subprocess.run(["cc", "-O1", "-shared", "-fPIC", "-w", "-pthread", "-I/opt/rocm/include",
                    os.path.join(HERE, "fake_hip_threads.c"), "-o", so], check=True)
    return so


@pytest.mark.parametrize("check", CHECKS)
def test_threads(fake, check):
    r = subprocess.run([sys.executable, os.path.abspath(__file__), fake, check],
                       capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr


if __name__ == "__main__":
    globals()[sys.argv[2]](Threads(sys.argv[1]))
