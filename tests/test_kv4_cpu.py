"""Refusals of the 4-bit cache's and the sampling operators' entry points, which come
before any device work, and the binding's struct (no GPU needed)."""
import ctypes as C
import os

import pytest

import test_rust_sys_cpu as rust

X = 0x100000   # an address that nothing reads


def mods():
    import mri_llama as L
    import mri_qmatmul as M
    return L, M, L.lib()


def status(rc):
    import mri_qmatmul
    return mri_qmatmul.STATUS.get(rc, rc)


@pytest.mark.parametrize("sizes,want", [
    ((0, 1, 8, 1, 64), "InvalidShape"), ((1, 0, 8, 1, 64), "InvalidShape"),
    ((1, 1, 0, 1, 64), "InvalidShape"), ((1, 1, 8, 0, 64), "InvalidShape"),
    ((1, 1, 8, 1, 0), "InvalidShape"), ((1, 1, 8, 1, 96), "Unsupported"),
    ((1, 1, (1 << 30) + 1, 1, 64), "Unsupported"),
    ((1 << 40, 1 << 40, 1 << 30, 1, 64), "Unsupported"),
])
def test_cache_create_refusals(sizes, want):
    L, M, lib = mods()
    h = C.c_void_p(5)
    assert status(lib.mri_kv4_cache_create(*sizes, C.byref(h))) == want
    assert not h.value
    assert status(lib.mri_kv4_cache_create(1, 1, 8, 1, 64, None)) == "InvalidArgument"


def test_null_arguments():
    L, M, lib = mods()
    r = L.Kv4Rows(0, 1, 1, 0, None, None)
    assert status(lib.mri_kv4_append(None, 0, C.byref(r), X, X, 64, None)) == "InvalidArgument"
    assert status(lib.mri_kv4_read(None, 0, 1, C.byref(r), X, X, 64, None)) == "InvalidArgument"
    assert status(lib.mri_kv4_attend(None, 0, C.byref(r), X, 64, 1, X, 64, None, None)) \
        == "InvalidArgument"
    assert status(lib.mri_kv4_evict(None, None, X, X, X, X, 1, 0, X, None)) == "InvalidArgument"
    assert status(lib.mri_llama_forward_kv4(None, X, 1, 0, None, 0, 0, None, X, None)) \
        == "InvalidArgument"
    assert lib.mri_kv4_cache_device_bytes(None) == 0
    lib.mri_kv4_cache_destroy(None)


@pytest.mark.parametrize("args,want", [
    ((X, 1, 8, 8, 0.0, X, 8), "InvalidArgument"), ((X, 1, 8, 8, -1.0, X, 8), "InvalidArgument"),
    ((X, 1, 8, 8, float("nan"), X, 8), "InvalidArgument"),
    ((X, 1, 8, 8, float("inf"), X, 8), "InvalidArgument"),
    ((X, 1, 0, 8, 1.0, X, 8), "InvalidShape"), ((X, 1, 8, 7, 1.0, X, 8), "InvalidShape"),
    ((X, 1, 8, 8, 1.0, X, 7), "InvalidShape"), ((None, 1, 8, 8, 1.0, X, 8), "InvalidArgument"),
    ((X, 1, 8, 8, 1.0, None, 8), "InvalidArgument"), ((X + 2, 1, 8, 8, 1.0, X, 8), "InvalidArgument"),
    ((X, 2, 8, 8, 1.0, X, 9), "InvalidArgument"), ((X, 1 << 22, 8, 8, 1.0, X, 8), "Unsupported"),
    ((None, 0, 0, 0, 1.0, None, 0), 0),
])
def test_softmax_refusals(args, want):
    L, M, lib = mods()
    assert status(lib.mri_softmax(*args, None)) == want


@pytest.mark.parametrize("kw,want", [
    (dict(n=0), "InvalidShape"), (dict(n=0xffffffff), "Unsupported"),
    (dict(k=1 << 21), "Unsupported"), (dict(seqs=1 << 22), "Unsupported"),
    (dict(drafts=None), "InvalidArgument"), (dict(target=None), "InvalidArgument"),
    (dict(u=None), "InvalidArgument"), (dict(tokens=None), "InvalidArgument"),
    (dict(accepted=None), "InvalidArgument"), (dict(seqs=0, n=0), 0),
])
def test_verify_refusals(kw, want):
    L, M, lib = mods()
    a = dict(drafts=X, draft=X, target=X, u=X, counts=None, seqs=1, k=2, n=8, tokens=X, accepted=X)
    a.update(kw)
    assert status(lib.mri_verify_drafts(*a.values(), None)) == want


def test_row_strides():
    import torch
    L, M, _ = mods()
    t = torch.zeros(4, 6, 10)
    assert L._row_stride(t, "t") == 10
    assert L._row_stride(t[:, :, :8], "t") == 10
    assert L._row_stride(t[1:2, 3:4], "t") == 10
    assert L._row_stride(t[1, :, :3], "t") == 10
    assert L._row_stride(t[:, :1], "t") == 60
    for bad in (t[:, :3], t[:, :, ::2], t.transpose(0, 1)):
        with pytest.raises(M.MriError):
            L._row_stride(bad, "t")


def test_struct_matches_rust():
    src = rust.rust_source()
    body = src.split("pub struct mri_kv4_rows {")[1].split("}")[0]
    got = [(f.split(":")[0].replace("pub", "").strip(), rust.rust_norm(f.split(":", 1)[1]))
           for f in body.split(",") if f.strip()]
    want = [(n, rust.rust_norm(t)) for n, t in rust.c_structs()["mri_kv4_rows"]]
    assert got == want
    import mri_llama
    assert [n for n, _ in mri_llama.Kv4Rows._fields_] == [n for n, _ in want]
    assert "0xffff_ffff" in src and mri_llama.NO_TOKEN == 0xffffffff
    assert os.path.isfile(rust.LIB_RS)
