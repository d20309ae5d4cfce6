"""ctypes binding of the GPU LlamaModelInt8, the 4-bit KV cache and the
sampling operators (include/mri_llama.h).

Host plumbing for tests and benchmarks over libmri_qmatmul.so: weights are
the handles of mri_qmatmul (QMatrix / Q8Matrix) or device Q4_0 byte
tensors, logits are torch CUDA (HIP) tensors.  No CPU fallback: every call
runs the HIP kernels.
"""
from __future__ import annotations

import ctypes as C

import mri_qmatmul as Q

P = C.c_void_p
SZ = C.c_size_t
ST = C.c_int

INT8, Q8_0, Q4_0, Q4_0_W4A8 = 0, 1, 2, 3


class Config(C.Structure):
    _fields_ = [("dim", SZ), ("n_heads", SZ), ("n_kv_heads", SZ), ("ffn_dim", SZ),
                ("vocab", SZ), ("max_seq", SZ), ("eps", C.c_float), ("rope_base", C.c_float),
                ("n_layers", SZ)]


class WeightRef(C.Structure):
    _fields_ = [("format", C.c_int), ("ptr", P), ("n_out", SZ), ("k_in", SZ)]


class Kv4Rows(C.Structure):
    _fields_ = [("first_seq", SZ), ("n_seqs", SZ), ("rows", SZ), ("start", SZ), ("pos", P),
                ("count", P)]


_SIGS = {
    "mri_llama_create": ([C.POINTER(Config), P, P, WeightRef, C.POINTER(P)], ST),
    "mri_llama_set_layer": ([P, SZ, P, P, C.POINTER(WeightRef)], ST),
    "mri_llama_destroy": ([P], None),
    "mri_kv_cache_create": ([SZ, SZ, SZ, SZ, C.POINTER(P)], ST),
    "mri_kv_cache_destroy": ([P], None),
    "mri_llama_forward_cached": ([P, P, SZ, SZ, P, P, P], ST),
    "mri_llama_forward_decode": ([P, C.c_uint32, SZ, P, P, P], ST),
    "mri_llama_generate_greedy": ([P, P, SZ, SZ, P, P, P, P], ST),
    "mri_argmax": ([P, SZ, SZ, P, P], ST),
    "mri_kv4_cache_create": ([SZ, SZ, SZ, SZ, SZ, C.POINTER(P)], ST),
    "mri_kv4_cache_device_bytes": ([P], SZ),
    "mri_kv4_cache_destroy": ([P], None),
    "mri_kv4_append": ([P, SZ, C.POINTER(Kv4Rows), P, P, SZ, P], ST),
    "mri_kv4_read": ([P, SZ, SZ, C.POINTER(Kv4Rows), P, P, SZ, P], ST),
    "mri_kv4_attend": ([P, SZ, C.POINTER(Kv4Rows), P, SZ, SZ, P, SZ, P, P], ST),
    "mri_kv4_evict": ([P, P, P, P, P, P, SZ, SZ, P, P], ST),
    "mri_llama_forward_kv4": ([P, P, SZ, SZ, P, SZ, SZ, P, P, P], ST),
    "mri_softmax": ([P, SZ, SZ, SZ, C.c_float, P, SZ, P], ST),
    "mri_verify_drafts": ([P, P, P, P, P, SZ, SZ, SZ, P, P, P], ST),
}
EXPORTED = tuple(_SIGS)

_done = False


def lib():
    global _done
    lib = Q.lib()
    if not _done:
        for name, (args, res) in _SIGS.items():
            f = getattr(lib, name)
            f.argtypes = args
            f.restype = res
        _done = True
    return lib


def weight_ref(w):
    """QMatrix / Q8Matrix / Q4Matrix (W4A8) handle, or (q4_0 device uint8
    tensor, n_out, k_in) for the W4A32 projection."""
    if isinstance(w, Q.QMatrix):
        return WeightRef(INT8, w.h, w.n_out, w.k_in)
    if isinstance(w, Q.Q8Matrix):
        return WeightRef(Q8_0, w.h, w.n_out, w.k_in)
    if isinstance(w, Q.Q4Matrix):
        return WeightRef(Q4_0_W4A8, w.h, w.n_out, w.k_in)
    t, n_out, k_in = w
    return WeightRef(Q4_0, C.c_void_p(t.data_ptr()), n_out, k_in)


class KvCache:
    def __init__(self, n_layers, max_seq, n_kv_heads, head_dim):
        h = C.c_void_p()
        Q.check(lib().mri_kv_cache_create(n_layers, max_seq, n_kv_heads, head_dim, C.byref(h)))
        self.h = h

    def close(self):
        if self.h:
            lib().mri_kv_cache_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


NO_TOKEN = 0xffffffff   # MRI_NO_TOKEN (-1 in int32 tensors)


def _bad(kind, msg):
    return Q.MriError({"InvalidShape": 1, "InvalidArgument": 3}[kind], msg)


_torch = None


def _device():
    """The current device (and torch, loaded at the first call)."""
    global _torch, _F32, _INTS, _raw_stream
    if _torch is None:
        import torch
        _F32, _INTS = (torch.float32,), (torch.int32, torch.uint32)
        # (3 us a call less than making a Stream object)
        _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream",
                              lambda dev: torch.cuda.current_stream(dev).cuda_stream)
        _torch = torch
    return _torch.cuda.current_device()


def _stream(stream, dev):
    return _raw_stream(dev) if stream is None else stream


def _tensor(t, name, dtypes, dev, shape=None):
    """The address of t after its type, place and (contiguous) shape are checked."""
    if t.dtype not in dtypes:
        raise _bad("InvalidArgument", f"{name}: dtype {t.dtype}")
    if t.get_device() != dev:
        raise _bad("InvalidArgument", f"{name}: on {t.device}, not on the current device")
    if shape is not None:
        if t.shape != shape:
            raise _bad("InvalidShape", f"{name}: shape {tuple(t.shape)}, expected {shape}")
        if not t.is_contiguous():
            raise _bad("InvalidArgument", f"{name}: not contiguous")
    return t.data_ptr()


def _row_stride(t, name):
    """Floats between consecutive rows of t [..., rows, features]: the rows of all
    leading indices follow each other at one distance."""
    if t.is_contiguous():
        return t.shape[-1]
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        raise _bad("InvalidArgument", f"{name}: features are not contiguous")
    stride, n = None, 1
    for d in range(t.dim() - 2, -1, -1):
        if t.shape[d] > 1:
            if stride is None:
                stride = t.stride(d) // n if t.stride(d) % n == 0 else -1
            if t.stride(d) != stride * n:
                raise _bad("InvalidArgument", f"{name}: rows are not evenly spaced")
        n *= t.shape[d]
    return t.shape[-1] if stride is None else stride


class Kv4Cache:
    """The KV cache in 4-bit blocks (mri_kv4_*).  Rows are f32 tensors
    [n_seqs, rows, features] (or [rows, features] of one sequence), evenly
    spaced; `start` is the first row's position, an int or an int32 tensor
    [n_seqs], `count` (int32 [n_seqs]) how many rows of a sequence are real."""

    def __init__(self, n_layers, n_seqs, max_seq, n_kv_heads, head_dim):
        h = C.c_void_p()
        Q.check(lib().mri_kv4_cache_create(n_layers, n_seqs, max_seq, n_kv_heads, head_dim,
                                           C.byref(h)))
        self.h, self.lib = h, lib()
        self.n_layers, self.n_seqs, self.max_seq = n_layers, n_seqs, max_seq
        self.n_kv_heads, self.head_dim = n_kv_heads, head_dim

    @property
    def device_bytes(self):
        return self.lib.mri_kv4_cache_device_bytes(self.h)

    def _rows(self, t, start, count, first_seq, dev):
        n_seqs, rows = (1, t.shape[-2]) if t.dim() == 2 else t.shape[-3:-1]
        pos = None
        if not isinstance(start, int):
            pos, start = _tensor(start, "start", _INTS, dev, (n_seqs,)), 0
        elif start < 0:
            raise _bad("InvalidShape", f"start {start} is negative")
        if count is not None:
            count = _tensor(count, "count", _INTS, dev, (n_seqs,))
        return C.byref(Kv4Rows(first_seq, n_seqs, rows, start, pos, count))

    def _kv(self, k, v, dims, dev):
        if k.dim() not in dims or k.shape != v.shape or \
                k.shape[-1] != self.n_kv_heads * self.head_dim:
            raise _bad("InvalidShape", f"k {tuple(k.shape)}, v {tuple(v.shape)}")
        s = _row_stride(k, "k")
        if _row_stride(v, "v") != s:
            raise _bad("InvalidArgument", "k and v differ in their row stride")
        return _tensor(k, "k", _F32, dev), _tensor(v, "v", _F32, dev), s

    def append(self, layer, k, v, start, count=None, first_seq=0, stream=None):
        dev = _device()
        kp, vp, s = self._kv(k, v, (2, 3), dev)
        Q.check(self.lib.mri_kv4_append(self.h, layer, self._rows(k, start, count, first_seq, dev),
                                        kp, vp, s, _stream(stream, dev)))

    def read(self, layer, k, v, start, count=None, first_seq=0, stream=None):
        """Into k and v; with a fourth leading axis, of that many layers."""
        dev = _device()
        kp, vp, s = self._kv(k, v, (2, 3, 4), dev)
        Q.check(self.lib.mri_kv4_read(self.h, layer, k.shape[0] if k.dim() == 4 else 1,
                                      self._rows(k, start, count, first_seq, dev), kp, vp, s,
                                      _stream(stream, dev)))

    def attend(self, layer, q, out, start, count=None, first_seq=0, weights=None, stream=None):
        """weights: f32 [n_seqs of the cache, n_kv_heads, max_seq] of this layer."""
        if q.dim() not in (2, 3) or q.shape != out.shape or q.shape[-1] % self.head_dim:
            raise _bad("InvalidShape", f"q {tuple(q.shape)}, out {tuple(out.shape)}")
        dev = _device()
        qp, op = _tensor(q, "q", _F32, dev), _tensor(out, "out", _F32, dev)
        if weights is not None:
            weights = _tensor(weights, "weights", _F32, dev,
                              (self.n_seqs, self.n_kv_heads, self.max_seq))
        Q.check(self.lib.mri_kv4_attend(self.h, layer, self._rows(q, start, count, first_seq, dev),
                                        qp, _row_stride(q, "q"), q.shape[-1] // self.head_dim, op,
                                        _row_stride(out, "out"), weights, _stream(stream, dev)))

    def evict(self, dst, weights, weights_out, lens, lens_out, keep, recent, kept, stream=None):
        """Into dst (self: in place, with weights_out = weights)."""
        lead, dev = (self.n_layers, self.n_seqs, self.n_kv_heads), _device()
        Q.check(self.lib.mri_kv4_evict(
            self.h, dst.h, _tensor(weights, "weights", _F32, dev, lead + (self.max_seq,)),
            _tensor(weights_out, "weights_out", _F32, dev, lead + (dst.max_seq,)),
            _tensor(lens, "lens", _INTS, dev, (self.n_seqs,)),
            _tensor(lens_out, "lens_out", _INTS, dev, (self.n_seqs,)), keep, recent,
            _tensor(kept, "kept", _INTS, dev, lead + (keep,)), _stream(stream, dev)))

    def close(self):
        if self.h:
            lib().mri_kv4_cache_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class Llama:
    """LlamaModelInt8 (forward_int8.rs:416-546) on the GPU.  `keep` holds the
    weight objects so that they outlive the model."""

    def __init__(self, cfg: dict, token_embd, output_norm, output, layers):
        import numpy as np
        self.cfg = cfg
        self.keep = [output, layers]
        c = Config(cfg["dim"], cfg["n_heads"], cfg["n_kv_heads"], cfg["ffn"], cfg["vocab"],
                   cfg["max_seq"], cfg["eps"], cfg["rope_base"], len(layers))
        emb = np.ascontiguousarray(token_embd, np.float32)
        on = np.ascontiguousarray(output_norm, np.float32)
        h = C.c_void_p()
        Q.check(lib().mri_llama_create(C.byref(c), emb.ctypes.data_as(P), on.ctypes.data_as(P),
                                       weight_ref(output), C.byref(h)))
        self.h = h
        for i, L in enumerate(layers):
            refs = (WeightRef * 7)(*[weight_ref(L[k]) for k in
                                     ("wq", "wk", "wv", "wo", "wgate", "wup", "wdown")])
            an = np.ascontiguousarray(L["attn_norm"], np.float32)
            fn = np.ascontiguousarray(L["ffn_norm"], np.float32)
            Q.check(lib().mri_llama_set_layer(h, i, an.ctypes.data_as(P), fn.ctypes.data_as(P),
                                              refs))

    def kv_cache(self):
        c = self.cfg
        return KvCache(len(self.keep[1]), c["max_seq"], c["n_kv_heads"],
                       c["dim"] // c["n_heads"])

    def forward_cached(self, tokens, start_pos, cache, logits, stream=None):
        import numpy as np
        t = np.ascontiguousarray(tokens, np.uint32)
        Q.check(lib().mri_llama_forward_cached(self.h, t.ctypes.data_as(P), t.size, start_pos,
                                               cache.h, C.c_void_p(logits.data_ptr()),
                                               Q._stream(stream)))

    def kv4_cache(self, n_seqs=1, max_seq=None):
        c = self.cfg
        return Kv4Cache(len(self.keep[1]), n_seqs, max_seq or c["max_seq"], c["n_kv_heads"],
                        c["dim"] // c["n_heads"])

    def forward_kv4(self, tokens, start_pos, cache, logits, seq=0, cache_pos=None, weights=None,
                    stream=None):
        """cache_pos: start_pos unless keys were evicted.  weights: f32
        [n_layers, n_seqs, n_kv_heads, max_seq] of the cache.  logits: f32, contiguous,
        [len(tokens), vocab] or more rows."""
        import numpy as np
        t = np.ascontiguousarray(tokens, np.uint32)
        dev = _device()
        lp = _tensor(logits, "logits", _F32, dev, logits.shape)
        if logits.numel() < t.size * self.cfg["vocab"]:
            raise _bad("InvalidShape", f"logits: shape {tuple(logits.shape)}, expected "
                                       f"{(t.size, self.cfg['vocab'])}")
        wp = None if weights is None else _tensor(
            weights, "weights", _F32, dev,
            (cache.n_layers, cache.n_seqs, cache.n_kv_heads, cache.max_seq))
        Q.check(lib().mri_llama_forward_kv4(
            self.h, t.ctypes.data_as(P), t.size, start_pos, cache.h, seq,
            start_pos if cache_pos is None else cache_pos, wp, lp, Q._stream(stream)))

    def forward_decode(self, token, pos, cache, logits, stream=None):
        Q.check(lib().mri_llama_forward_decode(self.h, int(token), pos, cache.h,
                                               C.c_void_p(logits.data_ptr()), Q._stream(stream)))

    def generate_greedy(self, prompt, n_steps, cache, logits=None, stream=None):
        import numpy as np
        p = np.ascontiguousarray(prompt, np.uint32)
        out = np.empty(n_steps + 1, np.uint32)
        Q.check(lib().mri_llama_generate_greedy(
            self.h, p.ctypes.data_as(P), p.size, n_steps, cache.h, out.ctypes.data_as(P),
            None if logits is None else C.c_void_p(logits.data_ptr()), Q._stream(stream)))
        return out

    def close(self):
        if self.h:
            lib().mri_llama_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def argmax(v, idx, stream=None):
    rows, n = (1, v.numel()) if v.dim() == 1 else tuple(v.shape)
    Q.check(lib().mri_argmax(C.c_void_p(v.data_ptr()), rows, n, C.c_void_p(idx.data_ptr()),
                             Q._stream(stream)))


def softmax(x, out, temperature=1.0, stream=None):
    """Probabilities of rows of logits x [rows, n] (or [n]) into out; may be x."""
    if x.shape != out.shape or x.dim() not in (1, 2):
        raise _bad("InvalidShape", f"x {tuple(x.shape)}, out {tuple(out.shape)}")
    dev = _device()
    rows, n = (1, x.numel()) if x.dim() == 1 else x.shape
    Q.check(lib().mri_softmax(_tensor(x, "x", _F32, dev), rows, n, _row_stride(x, "x"), temperature,
                              _tensor(out, "out", _F32, dev), _row_stride(out, "out"),
                              _stream(stream, dev)))


def verify_drafts(drafts, target_probs, uniforms, tokens, accepted, draft_probs=None,
                  n_drafts=None, stream=None):
    """drafts int32 [n_seqs, k], target_probs f32 [n_seqs, k + 1, n], uniforms f32
    [n_seqs, k + 1], draft_probs f32 [n_seqs, k, n], n_drafts int32 [n_seqs]; into
    tokens int32 [n_seqs, k + 1] and accepted int32 [n_seqs]."""
    if drafts.dim() != 2 or target_probs.dim() != 3:
        raise _bad("InvalidShape",
                   f"drafts {tuple(drafts.shape)}, target_probs {tuple(target_probs.shape)}")
    (b, k), n, dev = drafts.shape, target_probs.shape[2], _device()
    if draft_probs is not None:
        draft_probs = _tensor(draft_probs, "draft_probs", _F32, dev, (b, k, n))
    if n_drafts is not None:
        n_drafts = _tensor(n_drafts, "n_drafts", _INTS, dev, (b,))
    Q.check(lib().mri_verify_drafts(
        _tensor(drafts, "drafts", _INTS, dev, (b, k)), draft_probs,
        _tensor(target_probs, "target_probs", _F32, dev, (b, k + 1, n)),
        _tensor(uniforms, "uniforms", _F32, dev, (b, k + 1)), n_drafts, b, k, n,
        _tensor(tokens, "tokens", _INTS, dev, (b, k + 1)),
        _tensor(accepted, "accepted", _INTS, dev, (b,)), _stream(stream, dev)))
