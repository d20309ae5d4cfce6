// kv4.hpp — the KV cache held in 4-bit blocks: its layout and launchers.
//
// A block is 32 consecutive dims of one head's key or value: an f16 scale d
// and 32 quants q in [-8, 7] (value q * d), a block of GGUF's Q4_0 in what it holds;
// the quants are nearer (Q4_0 files divide by the scale before its rounding to f16).
// With mx, mn the block's extremes and a = mx if mx >= -mn else mn,
// d = f16(a / -8) (saturated at +-65504) and q = clamp(rint(x / d), -8, 7); a
// block with d = 0 holds zeros, one with a value that is not finite reads as
// NaN.
//
// The cache is pages of 64 keys of one (layer, sequence, KV head), 72 * HD
// bytes each (HD the head dim, NB = HD / 32 blocks), at page index
// ((layer * n_seqs + seq) * n_kv + head) * n_pages + key / 64.  A page is laid
// out so that a lane's loads are the operands of v_mfma_f32_16x16x32_f16
// (lane l = 16 g + r: row r, k = 8 g + j, j = 0..7), one dword of nibbles each:
//  * K quants at 0: tile t (keys 16 t ..), lane l, block b: the dword at
//    t * 8 HD + l * 4 NB + 4 b holds key 16 t + r, dims 32 b + 8 g + j.
//  * V quants at 32 HD: dim tile e (dims 16 e ..), lane l, key half h: the dword
//    at (e / 2) * 1024 + l * 16 + (e % 2) * 8 + 4 h holds dim 16 e + r, keys
//    32 h + 4 g + j (j < 4) and 32 h + 16 + 4 g + j - 4: the keys whose
//    probabilities lane group g holds after the score product of tiles 2 h and
//    2 h + 1, so that they are the other operand without leaving the lane.
//  * scales of K at 64 HD and of V at 68 HD: f16, keys 16 t + 4 g + i of block
//    b at ((t * 4 + g) * NB + b) * 8 + 2 i.
// In a dword, element j is nibble (j >> 1) + 4 * (j & 1), stored as q + 8:
// nibbles p and p + 4 are the halves of one register of two f16.
#pragma once

#include "common.hpp"
#include "mri_llama.h"

namespace mri {

constexpr int kPageKeys = 64;
inline size_t kv4_page_bytes(size_t hd) { return 72 * hd; }

// One layer of the cache and the rows of a call, as the kernels take them.
struct Kv4Rows {
    uint8_t *pages = nullptr;  // of the layer
    int n_kv = 0, n_pages = 0;
    unsigned max_seq = 0;
    int first_seq = 0, n_seqs = 0;
    unsigned rows = 0, start = 0;
    unsigned row0 = 0, ld_rows = 0;  // the rows are row0 .. of ld_rows a sequence
    const uint32_t *pos = nullptr, *count = nullptr;
};

// Workspace of the attention, owned by the cache: partial results of split
// rows, a counter a split tile (zero between calls) and the rows' log-sum-exps.
constexpr size_t kKv4PartTiles = 1024;   // 16-query tiles of partials, and counters
constexpr size_t kKv4LseFloats = 1 << 20;
inline size_t kv4_part_floats(size_t hd) { return kKv4PartTiles * 16 * (hd + 2); }

mri_status launch_kv4_append(const Kv4Rows &a, size_t hd, const float *k, const float *v,
                             size_t stride, hipStream_t s);
// n_layers layers, layer_bytes apart; k and v [n_layers][n_seqs][rows][stride].
mri_status launch_kv4_read(const Kv4Rows &a, size_t hd, size_t n_layers, size_t layer_bytes,
                           float *k, float *v, size_t stride, hipStream_t s);
// weights (nullable): [sequence slots][n_kv][max_seq] of the layer.
mri_status launch_kv4_attend(const Kv4Rows &a, size_t hd, const float *q, size_t q_stride,
                             size_t n_heads, float *out, size_t out_stride, float *weights,
                             float *part, int *cnts, float *lse, hipStream_t s);

struct Kv4Evict {
    const uint8_t *src = nullptr;
    uint8_t *dst = nullptr;
    size_t row0 = 0;  // the first (layer, sequence, KV head) of a launch
    int n_layers = 0, n_seqs = 0, n_kv = 0;
    int src_pages = 0, dst_pages = 0;
    unsigned src_max = 0, dst_max = 0;
    const float *w = nullptr;   // [n_layers][n_seqs][n_kv][src_max]
    float *w_out = nullptr;     // the same with dst_max
    const uint32_t *lens = nullptr;
    uint32_t *lens_out = nullptr;
    unsigned keep = 0, recent = 0;
    uint32_t *kept = nullptr;   // [n_layers][n_seqs][n_kv][keep]
};
mri_status launch_kv4_evict(const Kv4Evict &e, size_t hd, hipStream_t s);

// sample.hip
// The parts' statistics of rows in parts: per (device, stream), of one size, for
// calls that are not being captured.  *ptr is null where the memory cannot be had.
constexpr size_t kSoftmaxWsBytes = 1 << 18;
mri_status softmax_ws_get(hipStream_t stream, void **ptr);
mri_status launch_softmax(const float *x, size_t rows, size_t n, size_t x_stride,
                          float temperature, float *out, size_t out_stride, hipStream_t s);
mri_status launch_verify(const uint32_t *drafts, const float *draft_probs,
                         const float *target_probs, const float *uniforms,
                         const uint32_t *n_drafts, size_t n_seqs, size_t k, size_t n,
                         uint32_t *tokens, uint32_t *accepted, hipStream_t s);

}  // namespace mri
