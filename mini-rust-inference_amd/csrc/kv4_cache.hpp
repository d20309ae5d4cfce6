// kv4_cache.hpp — the handle of the 4-bit KV cache and the checks of a call's
// rows, shared by its entry points and the model's.
#pragma once

#include "kv4.hpp"

constexpr size_t kKv4MaxSeq = (size_t)1 << 30;

struct mri_kv4_cache {
    size_t n_layers = 0, n_seqs = 0, max_seq = 0, n_kv = 0, hd = 0, n_pages = 0;
    uint8_t *pages = nullptr;
    float *part = nullptr, *lse = nullptr;
    int *cnts = nullptr;
    int device = 0;
    size_t layer_bytes() const { return n_seqs * n_kv * n_pages * mri::kv4_page_bytes(hd); }
};

namespace mri {
// The kernels' form of a call's rows; checks them against the cache.
mri_status kv4_rows(const mri_kv4_cache *c, size_t layer, const mri_kv4_rows *r, Kv4Rows *a);
// The cache's device is the current one.
mri_status kv4_on_device(const mri_kv4_cache *c);
}  // namespace mri
