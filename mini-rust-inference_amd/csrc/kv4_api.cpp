// kv4_api.cpp — the extern "C" entry points of the 4-bit KV cache, softmax and
// draft verification (include/mri_llama.h): checks of the arguments, then the
// launchers of kv4.hip and sample.hip.
#include <hip/hip_runtime.h>

#include <cmath>
#include <new>
#include <string>

#include "kv4_cache.hpp"

namespace mri {
mri_status current_device(int *dev);

namespace {

mri_status bad_arg(const std::string &m) { return set_error(MRI_ERR_INVALID_ARGUMENT, m); }
mri_status bad_shape(const std::string &m) { return set_error(MRI_ERR_INVALID_SHAPE, m); }

#define TRY(call)                              \
    do {                                       \
        const mri_status _st = (call);         \
        if (_st != MRI_OK) return _st;         \
    } while (0)

template <class... P>
bool float_aligned(const P *...p) {
    return ((... | (uintptr_t)p) & 3) == 0;
}

}  // namespace

mri_status kv4_on_device(const mri_kv4_cache *c) {
    int dev;
    TRY(current_device(&dev));
    if (dev != c->device)
        return bad_arg("kv4: the cache is on device " + std::to_string(c->device) +
                       ", the current device is " + std::to_string(dev));
    return MRI_OK;
}

mri_status kv4_rows(const mri_kv4_cache *c, size_t layer, const mri_kv4_rows *r, Kv4Rows *a) {
    if (!c || !r) return bad_arg("kv4: null cache or rows");
    if (layer >= c->n_layers)
        return bad_arg("kv4: layer " + std::to_string(layer) + " of " +
                       std::to_string(c->n_layers));
    if (r->n_seqs > c->n_seqs || r->first_seq > c->n_seqs - r->n_seqs)
        return bad_shape("kv4: sequences " + std::to_string(r->first_seq) + " + " +
                         std::to_string(r->n_seqs) + " of " + std::to_string(c->n_seqs));
    if (r->rows > kKv4MaxSeq) return bad_shape("kv4: too many rows");
    if (!r->pos && (r->start > c->max_seq || r->rows > c->max_seq - r->start))
        return bad_shape("kv4: positions " + std::to_string(r->start) + " + " +
                         std::to_string(r->rows) + " exceed the cache length " +
                         std::to_string(c->max_seq));
    if (!float_aligned(r->pos, r->count))
        return bad_arg("kv4: positions and counts must be 4-byte aligned");
    a->pages = c->pages + layer * c->layer_bytes();
    a->n_kv = (int)c->n_kv;
    a->n_pages = (int)c->n_pages;
    a->max_seq = (unsigned)c->max_seq;
    a->first_seq = (int)r->first_seq;
    a->n_seqs = (int)r->n_seqs;
    a->rows = a->ld_rows = (unsigned)r->rows;
    a->start = r->pos ? 0 : (unsigned)r->start;
    a->pos = r->pos;
    a->count = r->count;
    return MRI_OK;
}

}  // namespace mri

using namespace mri;

extern "C" {

mri_status mri_kv4_cache_create(size_t n_layers, size_t n_seqs, size_t max_seq, size_t n_kv_heads,
                                size_t head_dim, mri_kv4_cache **out) {
    if (!out) return bad_arg("null argument");
    *out = nullptr;
    if (!n_layers || !n_seqs || !max_seq || !n_kv_heads || !head_dim)
        return bad_shape("kv4_cache: zero size");
    if (!attention_supported(head_dim))
        return set_error(MRI_ERR_UNSUPPORTED, "kv4_cache: head_dim must be 64 or 128");
    const size_t n_pages = (max_seq + kPageKeys - 1) / kPageKeys;
    const size_t page = kv4_page_bytes(head_dim);
    size_t bytes = page;
    if (max_seq > kKv4MaxSeq || __builtin_mul_overflow(bytes, n_pages, &bytes) ||
        __builtin_mul_overflow(bytes, n_kv_heads, &bytes) ||
        __builtin_mul_overflow(bytes, n_seqs, &bytes) ||
        __builtin_mul_overflow(bytes, n_layers, &bytes) || bytes > ((size_t)1 << 62) ||
        n_layers > (1u << 20) || n_seqs > (1u << 20) || n_kv_heads > (1u << 20))
        return set_error(MRI_ERR_UNSUPPORTED, "kv4_cache: too large");
    int dev;
    TRY(current_device(&dev));
    auto *c = new (std::nothrow) mri_kv4_cache();
    if (!c) return set_error(MRI_ERR_HIP, "kv4_cache: out of host memory");
    c->n_layers = n_layers;
    c->n_seqs = n_seqs;
    c->max_seq = max_seq;
    c->n_kv = n_kv_heads;
    c->hd = head_dim;
    c->n_pages = n_pages;
    c->device = dev;
    const size_t part = kv4_part_floats(head_dim) * sizeof(float);
    hipError_t e;
    if ((e = hipMalloc(&c->pages, bytes)) || (e = hipMemset(c->pages, 0, bytes)) ||
        (e = hipMalloc(&c->part, part)) ||
        (e = hipMalloc(&c->lse, kKv4LseFloats * sizeof(float))) ||
        (e = hipMalloc(&c->cnts, kKv4PartTiles * sizeof(int))) ||
        (e = hipMemset(c->cnts, 0, kKv4PartTiles * sizeof(int))) ||
        (e = hipStreamSynchronize(nullptr))) {
        (void)hipGetLastError();  // a refused allocation is no later launch's error
        mri_kv4_cache_destroy(c);
        return hip_error(e, "kv4_cache_create");
    }
    *out = c;
    return MRI_OK;
}

size_t mri_kv4_cache_device_bytes(const mri_kv4_cache *c) {
    if (!c) return 0;
    return c->n_layers * c->layer_bytes() +
           (kv4_part_floats(c->hd) + kKv4LseFloats + kKv4PartTiles) * sizeof(float);
}

void mri_kv4_cache_destroy(mri_kv4_cache *c) {
    if (!c) return;
    if (c->pages) (void)hipFree(c->pages);
    if (c->part) (void)hipFree(c->part);
    if (c->lse) (void)hipFree(c->lse);
    if (c->cnts) (void)hipFree(c->cnts);
    delete c;
}

mri_status mri_kv4_append(mri_kv4_cache *c, size_t layer, const mri_kv4_rows *rows, const float *k,
                          const float *v, size_t stride, void *stream) {
    Kv4Rows a;
    TRY(kv4_rows(c, layer, rows, &a));
    if (stride < c->n_kv * c->hd) return bad_shape("kv4_append: rows overlap");
    if (!a.rows || !a.n_seqs) return MRI_OK;
    if (!k || !v) return bad_arg("kv4_append: null pointer");
    if (!float_aligned(k, v)) return bad_arg("kv4_append: unaligned rows");
    TRY(kv4_on_device(c));
    return launch_kv4_append(a, c->hd, k, v, stride, static_cast<hipStream_t>(stream));
}

mri_status mri_kv4_read(const mri_kv4_cache *c, size_t layer, size_t n_layers,
                        const mri_kv4_rows *rows, float *k, float *v, size_t stride,
                        void *stream) {
    Kv4Rows a;
    TRY(kv4_rows(c, layer, rows, &a));
    if (n_layers > c->n_layers - layer)
        return bad_arg("kv4_read: layers " + std::to_string(layer) + " + " +
                       std::to_string(n_layers) + " of " + std::to_string(c->n_layers));
    if (stride < c->n_kv * c->hd) return bad_shape("kv4_read: rows overlap");
    if (!a.rows || !a.n_seqs || !n_layers) return MRI_OK;
    if (!k || !v) return bad_arg("kv4_read: null pointer");
    if (!float_aligned(k, v)) return bad_arg("kv4_read: unaligned rows");
    TRY(kv4_on_device(c));
    return launch_kv4_read(a, c->hd, n_layers, c->layer_bytes(), k, v, stride,
                           static_cast<hipStream_t>(stream));
}

mri_status mri_kv4_attend(mri_kv4_cache *c, size_t layer, const mri_kv4_rows *rows, const float *q,
                          size_t q_stride, size_t n_heads, float *out, size_t out_stride,
                          float *weights, void *stream) {
    Kv4Rows a;
    TRY(kv4_rows(c, layer, rows, &a));
    if (!n_heads || n_heads % c->n_kv)
        return bad_shape("kv4_attend: " + std::to_string(n_heads) + " heads over " +
                         std::to_string(c->n_kv) + " KV heads");
    if (n_heads > kKv4LseFloats || (n_heads / c->n_kv) * a.rows > (1u << 30))
        return set_error(MRI_ERR_UNSUPPORTED, "kv4_attend: too many queries");
    if (q_stride < n_heads * c->hd || out_stride < n_heads * c->hd)
        return bad_shape("kv4_attend: rows overlap");
    if (!a.rows || !a.n_seqs) return MRI_OK;
    if (!q || !out) return bad_arg("kv4_attend: null pointer");
    if (!float_aligned(q, out, weights))
        return bad_arg("kv4_attend: unaligned rows");
    if (q == out && q_stride != out_stride)
        return bad_arg("kv4_attend: in place the strides must be equal");
    if (weights && q == out)  // the weights are summed from q after out is written
        return bad_arg("kv4_attend: out is q, and weights are asked for");
    TRY(kv4_on_device(c));
    return launch_kv4_attend(a, c->hd, q, q_stride, n_heads, out, out_stride, weights, c->part,
                             c->cnts, c->lse, static_cast<hipStream_t>(stream));
}

mri_status mri_kv4_evict(const mri_kv4_cache *src, mri_kv4_cache *dst, const float *weights,
                         float *weights_out, const uint32_t *lens, uint32_t *lens_out, size_t keep,
                         size_t recent, uint32_t *kept, void *stream) {
    if (!src || !dst || !weights || !weights_out || !lens || !lens_out || !kept)
        return bad_arg("kv4_evict: null argument");
    if (src->n_layers != dst->n_layers || src->n_seqs != dst->n_seqs || src->n_kv != dst->n_kv ||
        src->hd != dst->hd)
        return bad_shape("kv4_evict: the caches differ");
    if (!keep || keep > dst->max_seq)
        return bad_shape("kv4_evict: keep " + std::to_string(keep) + " of a cache of " +
                         std::to_string(dst->max_seq));
    if (recent > keep) return bad_arg("kv4_evict: recent > keep");
    if ((src == dst) != (weights == weights_out))
        return bad_arg("kv4_evict: weights_out is weights in place, and only there");
    if (!float_aligned(weights, weights_out, lens, lens_out, kept))
        return bad_arg("kv4_evict: unaligned arrays");
    TRY(kv4_on_device(src));
    TRY(kv4_on_device(dst));
    Kv4Evict e;
    e.src = src->pages;
    e.dst = dst->pages;
    e.n_layers = (int)src->n_layers;
    e.n_seqs = (int)src->n_seqs;
    e.n_kv = (int)src->n_kv;
    e.src_pages = (int)src->n_pages;
    e.dst_pages = (int)dst->n_pages;
    e.src_max = (unsigned)src->max_seq;
    e.dst_max = (unsigned)dst->max_seq;
    e.w = weights;
    e.w_out = weights_out;
    e.lens = lens;
    e.lens_out = lens_out;
    e.keep = (unsigned)keep;
    e.recent = (unsigned)recent;
    e.kept = kept;
    return launch_kv4_evict(e, src->hd, static_cast<hipStream_t>(stream));
}

mri_status mri_softmax(const float *x, size_t rows, size_t n, size_t x_stride, float temperature,
                       float *out, size_t out_stride, void *stream) {
    if (!(temperature > 0.0f) || !std::isfinite(temperature))
        return bad_arg("softmax: the temperature must be positive and finite");
    if (rows && (!n || x_stride < n || out_stride < n))
        return bad_shape("softmax: empty or overlapping rows");
    if (!rows) return MRI_OK;
    if (!x || !out) return bad_arg("softmax: null pointer");
    if (!float_aligned(x, out)) return bad_arg("softmax: unaligned rows");
    if (x == out && x_stride != out_stride)
        return bad_arg("softmax: in place the strides must be equal");
    if (rows > (1u << 21))
        return set_error(MRI_ERR_UNSUPPORTED, "softmax: more than 2^21 rows");
    int dev;
    TRY(current_device(&dev));
    return launch_softmax(x, rows, n, x_stride, temperature, out, out_stride,
                          static_cast<hipStream_t>(stream));
}

mri_status mri_verify_drafts(const uint32_t *drafts, const float *draft_probs,
                             const float *target_probs, const float *uniforms,
                             const uint32_t *n_drafts, size_t n_seqs, size_t k, size_t n,
                             uint32_t *tokens, uint32_t *accepted, void *stream) {
    if (!n_seqs) return MRI_OK;
    if (!n) return bad_shape("verify_drafts: empty vocabulary");
    if (n >= MRI_NO_TOKEN || k > (1u << 20) || n_seqs > (1u << 21))
        return set_error(MRI_ERR_UNSUPPORTED, "verify_drafts: too many tokens or sequences");
    if (!target_probs || !uniforms || !tokens || !accepted || (k && !drafts))
        return bad_arg("verify_drafts: null pointer");
    if (!float_aligned(drafts, draft_probs, target_probs, uniforms, n_drafts, tokens, accepted))
        return bad_arg("verify_drafts: unaligned arrays");
    int dev;
    TRY(current_device(&dev));
    return launch_verify(drafts, draft_probs, target_probs, uniforms, n_drafts, n_seqs, k, n,
                         tokens, accepted, static_cast<hipStream_t>(stream));
}

}  // extern "C"
