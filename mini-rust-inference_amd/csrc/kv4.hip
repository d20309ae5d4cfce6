// kv4.hip — the KV cache in 4-bit blocks: append, read, attention, eviction.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "kv4.hpp"

namespace mri {
namespace {

constexpr int kWave = 64;

// What all lanes of a wave agree on, in a scalar register.
template <class T>
__device__ inline T uniform(T v) {
    return (T)__builtin_amdgcn_readfirstlane((int)v);
}
__device__ inline int wave_id() { return uniform((int)threadIdx.x >> 6); }

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef float float4_t __attribute__((ext_vector_type(4)));
typedef unsigned uint4_t __attribute__((ext_vector_type(4)));

template <int HD>
struct Page {
    static constexpr int NB = HD / 32;
    static constexpr size_t kBytes = 72 * HD;
    static constexpr int kV = 32 * HD, kKs = 64 * HD, kVs = 68 * HD;
    // byte of the K dword with dims 32 b + 8 g .. of key `key`
    static __device__ int k_dword(int key, int g, int b) {
        return (key >> 4) * 8 * HD + (g * 16 + (key & 15)) * 4 * NB + 4 * b;
    }
    // byte of the V dword with the eight keys of (g, half h) of dim `dim`
    static __device__ int v_dword(int dim, int g, int h) {
        const int e = dim >> 4;
        return kV + (e >> 1) * 1024 + (g * 16 + (dim & 15)) * 16 + (e & 1) * 8 + 4 * h;
    }
    // byte of a scale inside the K or V scales
    static __device__ int scale(int key, int b) {
        return ((key >> 2) * NB + b) * 8 + 2 * (key & 3);
    }
    // where a key's quant sits in a dim's V dwords: (g, h) and element j
    static __device__ void v_place(int key, int *g, int *h, int *j) {
        *h = key >> 5;
        *g = (key >> 2) & 3;
        *j = (key & 3) + ((key >> 4) & 1) * 4;
    }
    // the key that (g, h, j) stands for
    static __device__ int v_key(int g, int h, int j) {
        return 32 * h + (j >> 2) * 16 + 4 * g + (j & 3);
    }
};

__host__ __device__ inline int nibble_of(int j) { return (j >> 1) + 4 * (j & 1); }

// The real rows of the call's sequence b: positions [*p0, *p0 + count).
__device__ inline unsigned rows_of(const Kv4Rows &a, int b, unsigned *p0) {
    const unsigned p = a.pos ? a.pos[b] : a.start;
    if (p >= a.max_seq || a.row0 >= a.max_seq - p) return *p0 = 0;
    *p0 = p + a.row0;
    unsigned n = a.rows;
    if (a.count) n = min(n, a.count[b] - min(a.row0, a.count[b]));
    return min(n, a.max_seq - *p0);
}
// Row i of sequence b among the call's rows.
__device__ inline size_t row_index(const Kv4Rows &a, int b, size_t i) {
    return (size_t)b * a.ld_rows + a.row0 + i;
}

// ---- append ------------------------------------------------------------------------
// One workgroup a page of the rows' positions and KV head.  Eight lanes hold a
// block of 32 values; its extremes are reduced over them.  The quotient x / d
// is rounded exactly: n = rint(x * (1 / d)) is off by one at most, the rest
// x - n d is exact in f32 (n d has 15 bits and is near x), and comparing it
// with d / 2 settles n.  The quants go through LDS, key by key, and leave as
// the page's dwords, 16 bytes a thread; where keys of a V dword are not the call's,
// their nibbles are kept (a dword has one writer; what it held is loaded with the
// rows).  A thread's loads of eight rows are in flight together (2 x 2048 rows of
// 32 heads of 128, one after the other: 49 us).
__device__ inline int quant_of(float x, float d, float inv) {
    float n = rintf(x * inv);
    n = fminf(fmaxf(n, -9.0f), 9.0f);
    const float r = fmaf(-n, d, x), h = 0.5f * fabsf(d);
    const float up = (r < 0.0f) == (d < 0.0f) ? 1.0f : -1.0f;  // where the rest points
    if (fabsf(r) > h || (fabsf(r) == h && ((int)n & 1))) n = n + up;
    return (int)fminf(fmaxf(n, -8.0f), 7.0f) + 8;
}
// The other lanes' values of a group of eight, step by step: 1 and 2 within the
// four, then the mirrored four.
template <int STEP>
__device__ inline float lane8(float v) {
    constexpr int c = STEP == 0 ? 0xb1 : STEP == 1 ? 0x4e : 0x141;
    return __uint_as_float(
        __builtin_amdgcn_update_dpp(0, __float_as_uint(v), c, 0xf, 0xf, true));
}
// Quantizes a lane's four values with its group's: the quants + 8 as bytes, the
// block's scale bits.
__device__ inline unsigned quantize4(float4_t f, unsigned short *scale) {
    float mx = fmaxf(fmaxf(f[0], f[1]), fmaxf(f[2], f[3]));
    float mn = fminf(fminf(f[0], f[1]), fminf(f[2], f[3]));
    float bad = 0.0f;  // 1: a value that is not finite
#pragma unroll
    for (int i = 0; i < 4; ++i) bad = fabsf(f[i]) < INFINITY ? bad : 1.0f;
    mx = fmaxf(mx, lane8<0>(mx));
    mn = fminf(mn, lane8<0>(mn));
    bad = fmaxf(bad, lane8<0>(bad));
    mx = fmaxf(mx, lane8<1>(mx));
    mn = fminf(mn, lane8<1>(mn));
    bad = fmaxf(bad, lane8<1>(bad));
    mx = fmaxf(mx, lane8<2>(mx));
    mn = fminf(mn, lane8<2>(mn));
    bad = fmaxf(bad, lane8<2>(bad));
    const float am = mx >= -mn ? mx : mn;
    const _Float16 d16 = (_Float16)fminf(fmaxf(am * -0.125f, -65504.0f), 65504.0f);
    const float d = (float)d16, inv = 1.0f / d;
    const bool none = bad != 0.0f || d == 0.0f;
    unsigned w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) w |= (unsigned)(none ? 8 : quant_of(f[i], d, inv)) << (8 * i);
    *scale = bad != 0.0f ? 0x7e00 : __builtin_bit_cast(unsigned short, d16);
    return w;
}

template <int HD, bool V4>
__global__ __launch_bounds__(256) void k_kv4_append(Kv4Rows a, const float *__restrict__ k,
                                                    const float *__restrict__ v, size_t stride,
                                                    int n_pg) {
    using P = Page<HD>;
    constexpr int NB = P::NB, LD = HD + 8, R4 = HD / 4, RP = 256 / R4;  // rows a pass
    constexpr int U = 4;  // passes in flight
    __shared__ __attribute__((aligned(16))) uint8_t s_q[2][kPageKeys][LD];
    __shared__ uint16_t s_d[2][kPageKeys][NB];
    const int t = threadIdx.x, lane = t & 63, wv = wave_id(), g = lane >> 4, r = lane & 15;
    unsigned x = blockIdx.x;
    const int pg = x % n_pg;
    x /= n_pg;
    const int head = x % a.n_kv, b = x / a.n_kv;
    unsigned p0;
    const unsigned cnt = rows_of(a, b, &p0);
    const unsigned page = p0 / kPageKeys + pg, key0 = page * kPageKeys;
    if (cnt == 0 || key0 >= p0 + cnt) return;
    const int lo = (int)(max(p0, key0) - key0);
    const int hi = (int)(min(p0 + cnt, key0 + kPageKeys) - key0);
    uint8_t *pb = a.pages + (((size_t)(a.first_seq + b) * a.n_kv + head) * a.n_pages + page) *
                                P::kBytes;
    uint4_t *vto = reinterpret_cast<uint4_t *>(pb + P::kV + wv * 1024 + lane * 16);
    uint4_t old = {0, 0, 0, 0};
    if (wv < NB && hi - lo < kPageKeys) old = *vto;
    const int e = t % R4, first = lo + t / R4;
    const size_t base = row_index(a, b, 0) * stride + head * HD + 4 * e;
    for (int k0 = first; k0 < hi; k0 += U * RP) {
        float4_t f[2][U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            // (the last row again past the end)
            const size_t at = base + (size_t)(key0 + min(k0 + u * RP, hi - 1) - p0) * stride;
            if constexpr (V4) {
                f[0][u] = *reinterpret_cast<const float4_t *>(k + at);
                f[1][u] = *reinterpret_cast<const float4_t *>(v + at);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) f[0][u][i] = k[at + i], f[1][u][i] = v[at + i];
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int key = k0 + u * RP;
            if (key >= hi) break;
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                unsigned short d;
                *reinterpret_cast<unsigned *>(&s_q[w][key][4 * e]) = quantize4(f[w][u], &d);
                if ((e & 7) == 0) s_d[w][key][e >> 3] = d;
            }
        }
    }
    __syncthreads();
    const int kkey = 16 * wv + r;  // K: key kkey, dims 32 blk + 8 g ..
    if (kkey >= lo && kkey < hi) {
        unsigned *to = reinterpret_cast<unsigned *>(pb + P::k_dword(kkey, g, 0));
        unsigned w[NB];
#pragma unroll
        for (int blk = 0; blk < NB; ++blk) {
            const uint2 q = *reinterpret_cast<const uint2 *>(&s_q[0][kkey][32 * blk + 8 * g]);
            // bytes of even elements are nibbles 0..3, of odd ones nibbles 4..7
            const unsigned e0 = q.x & 0x000f000f, o0 = (q.x >> 8) & 0x000f000f;
            const unsigned e1 = q.y & 0x000f000f, o1 = (q.y >> 8) & 0x000f000f;
            const unsigned ev = (e0 & 0xf) | (e0 >> 12) | (e1 & 0xf) << 8 | (e1 >> 4 & 0xf000);
            const unsigned od = (o0 & 0xf) | (o0 >> 12) | (o1 & 0xf) << 8 | (o1 >> 4 & 0xf000);
            w[blk] = ev | od << 16;
        }
#pragma unroll
        for (int blk = 0; blk < NB; ++blk) to[blk] = w[blk];
    }
    if (wv < NB) {  // V: chunk wv, dims 32 wv + 16 dt + r, both halves
        unsigned val[2][2] = {{0, 0}, {0, 0}}, mask[2] = {0, 0};
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int key = P::v_key(g, h, j), sh = 4 * nibble_of(j);
                if (key >= lo && key < hi) {
                    val[0][h] |= (unsigned)s_q[1][key][32 * wv + r] << sh;
                    val[1][h] |= (unsigned)s_q[1][key][32 * wv + 16 + r] << sh;
                    mask[h] |= 0xfu << sh;
                }
            }
        if (mask[0] | mask[1])
            *vto = uint4_t{(old.x & ~mask[0]) | val[0][0], (old.y & ~mask[1]) | val[0][1],
                           (old.z & ~mask[0]) | val[1][0], (old.w & ~mask[1]) | val[1][1]};
    }
    for (int w = t; w < 2 * 64 * NB; w += 256) {  // scales
        const int which = w >= 64 * NB, rest = which ? w - 64 * NB : w;
        const int key = rest / NB, blk = rest % NB;
        if (key < lo || key >= hi) continue;
        *reinterpret_cast<uint16_t *>(pb + (which ? P::kVs : P::kKs) + P::scale(key, blk)) =
            s_d[which][key][blk];
    }
}

// ---- read ---------------------------------------------------------------------------
// A workgroup a page: a thread takes eight dims of a key from one K dword at a time,
// then eight keys of four dims from four V dwords.  Bound by its stores: 537 MB of
// f32 in 140 us (3.8 TB/s; non-temporal stores 180).
template <int HD, bool V4>
__global__ __launch_bounds__(256) void k_kv4_read(Kv4Rows a, size_t layer_bytes,
                                                  float *__restrict__ k, float *__restrict__ v,
                                                  size_t stride, int n_pg) {
    using P = Page<HD>;
    constexpr int NB = P::NB, R4 = HD / 4;
    unsigned x = blockIdx.x;
    const int pg = x % n_pg;
    x /= n_pg;
    const int head = x % a.n_kv;
    x /= a.n_kv;
    const int b = x % a.n_seqs, layer = x / a.n_seqs;
    unsigned p0;
    const unsigned cnt = rows_of(a, b, &p0);
    const unsigned page = p0 / kPageKeys + pg, key0 = page * kPageKeys;
    if (cnt == 0 || key0 >= p0 + cnt) return;
    const int lo = (int)(max(p0, key0) - key0);
    const int hi = (int)(min(p0 + cnt, key0 + kPageKeys) - key0);
    const uint8_t *pb = a.pages + layer * layer_bytes +
                        (((size_t)(a.first_seq + b) * a.n_kv + head) * a.n_pages + page) *
                            P::kBytes;
    // where row 0 of the call goes, and a key of the page
    const size_t base = ((size_t)layer * a.n_seqs * a.ld_rows + row_index(a, b, 0)) * stride +
                        head * HD;
    auto at = [&](int key) { return base + (size_t)(key0 + key - p0) * stride; };
    auto put = [](float *to, const float *f) __attribute__((always_inline)) {
        if constexpr (V4) {
            *reinterpret_cast<float4_t *>(to) = float4_t{f[0], f[1], f[2], f[3]};
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) to[i] = f[i];
        }
    };
    for (int it = threadIdx.x; it < (hi - lo) * (HD / 8); it += 256) {
        const int key = lo + it / (HD / 8), c = it % (HD / 8), blk = c >> 2, g = c & 3;
        const float d = (float)*reinterpret_cast<const _Float16 *>(pb + P::kKs + P::scale(key, blk));
        const unsigned w = *reinterpret_cast<const unsigned *>(pb + P::k_dword(key, g, blk));
        float f[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = (float)((int)(w >> (4 * nibble_of(j)) & 0xf) - 8) * d;
        float *to = k + at(key) + 32 * blk + 8 * g;
        put(to, f);
        put(to + 4, f + 4);
    }
    for (int it = threadIdx.x; it < R4 * 8; it += 256) {
        const int e = it % R4, g = it / R4 & 3, h = it / R4 >> 2, blk = e >> 3;
        if (32 * h + 4 * g >= hi || 32 * h + 20 + 4 * g <= lo) continue;  // none of its keys
        unsigned w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            w[i] = *reinterpret_cast<const unsigned *>(pb + P::v_dword(4 * e + i, g, h));
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const uint2 d = *reinterpret_cast<const uint2 *>(
                pb + P::kVs + (((2 * h + u) * 4 + g) * NB + blk) * 8);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int key = 32 * h + 16 * u + 4 * g + j, sh = 4 * nibble_of(4 * u + j);
                const unsigned dw = (j & 2 ? d.y : d.x) >> (16 * (j & 1));
                const float dv = f16_bits_to_f32(dw & 0xffff);
                float f[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) f[i] = (float)((int)(w[i] >> sh & 0xf) - 8) * dv;
                if (key >= lo && key < hi) put(v + at(key) + 4 * e, f);
            }
        }
    }
}

// ---- attention ----------------------------------------------------------------------
// Sixteen queries (rows x query heads of one KV head, flattened row-major) are
// the columns of S^T = K Q^T and O^T = V^T P^T, both on f16 matrix instructions
// with f32 accuracy.
//  * A nibble n masked out of a dword is the f16 n 2^-24 (16 n 2^-24 where the
//    mask leaves it four bits up); one packed FMA makes it (n - 8) 2^-9.  (As
//    subnormals the quants would go straight into the products, but the matrix
//    instructions align them as they are: 2.0e-7 of sum |a b| off in the mean
//    against 1.8e-9.)
//  * q is split into two f16 halves (22 bits) after a power-of-two scaling of
//    its row (what is below 2^-39 of its largest element is lost), and so is
//    p * d_v, the probability times the value block's scale, under a power of
//    two of each of the head's blocks, which its largest d_v gives (what is
//    below 2^-36 of that d_v is lost).
//  * The key blocks' scales multiply the 32-dim partial products in f32.
typedef float float2_t __attribute__((ext_vector_type(2)));

__device__ inline half8_t join(half2_t a, half2_t b, half2_t c, half2_t d) {
    return half8_t{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}
constexpr unsigned kNib0 = 0x000f000fu, kNib1 = 0x00f000f0u;
// The eight quants of a dword, times 2^-9.
__device__ inline half8_t quants(unsigned w) {
    const half2_t s0 = {(_Float16)0x1p15f, (_Float16)0x1p15f};
    const half2_t s1 = {(_Float16)0x1p11f, (_Float16)0x1p11f};
    const half2_t m8 = {(_Float16)-0x1p-6f, (_Float16)-0x1p-6f};
    const unsigned w8 = w >> 8;
    return join(__builtin_elementwise_fma(__builtin_bit_cast(half2_t, w & kNib0), s0, m8),
                __builtin_elementwise_fma(__builtin_bit_cast(half2_t, w & kNib1), s1, m8),
                __builtin_elementwise_fma(__builtin_bit_cast(half2_t, w8 & kNib0), s0, m8),
                __builtin_elementwise_fma(__builtin_bit_cast(half2_t, w8 & kNib1), s1, m8));
}

// x in two f16, hi + lo: off by 2^-23 of x where lo is not subnormal.  (The
// -1 is hidden from the compiler, which then takes the mixed-precision FMA
// that rounds to f16 by itself: one instruction a value instead of three.)
__device__ inline float minus_one() {
    float v = -1.0f;
    asm("" : "+s"(v));
    return v;
}
__device__ inline void split2(float x0, float x1, half2_t *hi, half2_t *lo) {
    const half2_t h = __builtin_convertvector((float2_t{x0, x1}), half2_t);
    *hi = h;
    const float m = minus_one();
    *lo = half2_t{(_Float16)fmaf((float)h.x, m, x0), (_Float16)fmaf((float)h.y, m, x1)};
}
__device__ inline void split8(const float *x, half8_t *hi, half8_t *lo) {
    half2_t h[4], l[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) split2(x[2 * u], x[2 * u + 1], &h[u], &l[u]);
    *hi = join(h[0], h[1], h[2], h[3]);
    *lo = join(l[0], l[1], l[2], l[3]);
}

// Sum and maximum over the four lanes of a column (lanes r, r + 16, ..).
__device__ inline float col_max(float v) {
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ inline float col_sum(float v) {
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Sum and maximum over a column's blocks (FEW, below): lanes r + k * 16 / NB.
template <int N>
__device__ inline float ror(float v) {  // of lane r + N of the row of 16
    return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), 0x120 + N, 0xf, 0xf,
                                                       true));
}
template <int NB>
__device__ inline float block_sum(float v) {
    v = v + ror<8>(v);
    if constexpr (NB == 4) v = v + ror<4>(v);
    return v;
}
template <int NB>
__device__ inline float block_max(float v) {
    v = fmaxf(v, ror<8>(v));
    if constexpr (NB == 4) v = fmaxf(v, ror<4>(v));
    return v;
}

// A tile's columns are 16 queries; with FEW they are 16 / NB queries times the NB
// blocks of the head dim, column b * 16 / NB + query.  Such a column holds its own
// block of the query only, so the products with all of K's blocks leave its block's
// dot; one scale a key multiplies it and the blocks' columns are added.  A column's
// probabilities need the scales of its own block only, a quarter of the work at head
// dim 128, and its sums count for that block's dims.
//
// What a lane loads of a tile: dims 8 g .. of a column's blocks (FEW: of block own).
template <int HD, bool FEW>
struct QRaw {
    static constexpr int NB = HD / 32, NQ = FEW ? 16 / NB : 16, N = FEW ? 1 : NB;
    float x[N][8];
    // src null: an empty column; vec: 16-byte loads are aligned
    __device__ void load(const float *src, int g, int own, bool vec) {
#pragma unroll
        for (int b = 0; b < N; ++b) {
            const float *p = src + 32 * (FEW ? own : b) + 8 * g;
            if (!src) {
#pragma unroll
                for (int j = 0; j < 8; ++j) x[b][j] = 0.0f;
            } else if (vec) {
                *reinterpret_cast<float4 *>(x[b]) = *reinterpret_cast<const float4 *>(p);
                *reinterpret_cast<float4 *>(x[b] + 4) = *reinterpret_cast<const float4 *>(p + 4);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) x[b][j] = p[j];
            }
        }
    }
};
// Queries are scaled by 2^e: the row's largest magnitude to [2^14, 2^15).
__device__ inline int up_exponent(float mx) {
    return mx > 0.0f && mx < INFINITY ? min(14 - ilogbf(mx), 120) : 0;
}
// What the raw products are multiplied by (log2 units): 2^(9 - e) log2(e) / sqrt(HD),
// rounded once.
template <int HD>
__device__ inline float score_scale(int e) {
    constexpr float c = HD == 64 ? 0.18033688011112042592f : 0.12751743021347021697f;
    return ldexpf(c, 9 - e);
}
template <int HD, bool FEW>
struct QTile {
    using R = QRaw<HD, FEW>;
    static constexpr int NB = HD / 32, NQ = R::NQ, N = R::N;
    half8_t hi[NB], lo[NB];
    float inv;  // what the raw products are multiplied by (log2 units)
    __device__ void make(const R &raw, int lane) {
        float mx = 0.0f;
#pragma unroll
        for (int b = 0; b < N; ++b)
#pragma unroll
            for (int j = 0; j < 8; ++j) mx = fmaxf(mx, fabsf(raw.x[b][j]));
        mx = col_max(mx);
        if constexpr (FEW) mx = block_max<NB>(mx);
        const int e = up_exponent(mx);
        const float up = ldexpf(1.0f, e);
#pragma unroll
        for (int b = 0; b < N; ++b) {
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = raw.x[b][j] * up;
            split8(x, &hi[b], &lo[b]);
        }
        if constexpr (FEW) {
            const int own = (lane & 15) / NQ;
            const half8_t h = hi[0], l = lo[0], z = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                hi[b] = b == own ? h : z;
                lo[b] = b == own ? l : z;
            }
        }
        inv = score_scale<HD>(e);
    }
};

// A page on its way through a wave: every byte is loaded once, in whole lines,
// while the page before it is computed (a wave that takes the scales where it
// needs them touches its page's lines up to sixteen times, and the waves of a CU
// are more than its caches hold: 138 us for 196 MB of pages).  The scales go on
// through LDS, from where each lane group takes those of its keys.
template <int HD>
struct PageLoad {
    static constexpr int NB = HD / 32;
    unsigned k[4][NB];          // tile, block
    unsigned v[HD / 16][2];     // dim tile, key half
    unsigned ks[NB / 2], vs[NB / 2];  // scales, in order over the lanes
    __device__ void load(const uint8_t *pb, int lane) {
        load_k(pb, lane);
#pragma unroll
        for (int c = 0; c < HD / 32; ++c) {
            const uint4 x =
                *reinterpret_cast<const uint4 *>(pb + Page<HD>::kV + c * 1024 + lane * 16);
            v[2 * c][0] = x.x, v[2 * c][1] = x.y, v[2 * c + 1][0] = x.z, v[2 * c + 1][1] = x.w;
        }
        load_scales(pb + Page<HD>::kVs, lane, vs);
    }
    __device__ void load_k(const uint8_t *pb, int lane) {
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const uint8_t *kp = pb + t * 8 * HD + lane * (HD / 8);
            if constexpr (HD == 128) {
                const uint4 x = *reinterpret_cast<const uint4 *>(kp);
                k[t][0] = x.x, k[t][1] = x.y, k[t][2] = x.z, k[t][3] = x.w;
            } else {
                const uint2 x = *reinterpret_cast<const uint2 *>(kp);
                k[t][0] = x.x, k[t][1] = x.y;
            }
        }
        load_scales(pb + Page<HD>::kKs, lane, ks);
    }
    static __device__ void load_scales(const uint8_t *sp, int lane, unsigned *d) {
        if constexpr (HD == 128) {
            const uint2 x = *reinterpret_cast<const uint2 *>(sp + 8 * lane);
            d[0] = x.x, d[1] = x.y;
        } else {
            d[0] = *reinterpret_cast<const unsigned *>(sp + 4 * lane);
        }
    }
    static __device__ void stage(const unsigned *d, int lane, unsigned *lds) {
#pragma unroll
        for (int u = 0; u < NB / 2; ++u) lds[lane * (NB / 2) + u] = d[u];
    }
    // the operands of a key tile's block and of a dim tile's key half
    __device__ half8_t kop(int t, int b) const { return quants(k[t][b]); }
    __device__ half8_t vop(int e, int h) const { return quants(v[e][h]); }
};
template <int HD>
constexpr int kScaleWords = 64 * HD / 64;  // of the keys or the values of a page

// Raw scores (times q.inv: log2 units) of a page's 16 keys of tile t: keys 4 g + i
// of column r in lane (g, r).  s_ks: the page's staged K scales, two dwords a block
// and four keys.
template <int HD, bool FEW, class Src>
__device__ inline float4_t score_tile(const Src &pl, const unsigned *s_ks, int t, int lane,
                                      const QTile<HD, FEW> &q) {
    constexpr int NB = HD / 32;
    const unsigned *sp = s_ks + (t * 4 + (lane >> 4)) * 2 * NB;
    float4_t s = {0, 0, 0, 0};
    if constexpr (FEW) {
        const uint2 d = reinterpret_cast<const uint2 *>(sp)[(lane & 15) / (16 / NB)];
        const half2_t d01 = __builtin_bit_cast(half2_t, d.x),
                      d23 = __builtin_bit_cast(half2_t, d.y);
        half8_t kq[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            kq[b] = pl.kop(t, b);
            s = __builtin_amdgcn_mfma_f32_16x16x32_f16(kq[b], q.lo[b], s, 0, 0, 0);
        }
#pragma unroll
        for (int b = 0; b < NB; ++b)
            s = __builtin_amdgcn_mfma_f32_16x16x32_f16(kq[b], q.hi[b], s, 0, 0, 0);
        return float4_t{block_sum<NB>(s[0] * (float)d01.x), block_sum<NB>(s[1] * (float)d01.y),
                        block_sum<NB>(s[2] * (float)d23.x), block_sum<NB>(s[3] * (float)d23.y)};
    }
    unsigned d[2 * NB];
#pragma unroll
    for (int u = 0; u < NB / 2; ++u)
        *reinterpret_cast<uint4 *>(d + 4 * u) = reinterpret_cast<const uint4 *>(sp)[u];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const half8_t kq = pl.kop(t, b);
        const half2_t d01 = __builtin_bit_cast(half2_t, d[2 * b]),
                      d23 = __builtin_bit_cast(half2_t, d[2 * b + 1]);
        float4_t c = {0, 0, 0, 0};
        c = __builtin_amdgcn_mfma_f32_16x16x32_f16(kq, q.lo[b], c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_16x16x32_f16(kq, q.hi[b], c, 0, 0, 0);
        s[0] = fmaf(c[0], (float)d01.x, s[0]);
        s[1] = fmaf(c[1], (float)d01.y, s[1]);
        s[2] = fmaf(c[2], (float)d23.x, s[2]);
        s[3] = fmaf(c[3], (float)d23.y, s[3]);
    }
    return s;
}

// The powers of two that a head's value scales are taken in: byte b is 15 + ve of its
// block b, 2^ve <= the largest d_v < 2^(ve + 1), at least 2^-15.  A lane's dwords of a
// page's scales are of one block.
template <int HD>
__device__ inline int scale_block(int lane) {
    return HD == 128 ? lane & 3 : lane >> 1 & 1;
}
__device__ inline int exp_byte(unsigned e, int b) { return e >> 8 * b & 0xff; }
// A lane's value scales of a page; those of keys from n_keys on become 0.
template <int HD>
struct ValueScales {
    static constexpr int NB = HD / 32, N = NB / 2;
    half2_t x[N];
    __device__ ValueScales(const unsigned *d, int lane, int n_keys) {
#pragma unroll
        for (int u = 0; u < N; ++u) x[u] = __builtin_bit_cast(half2_t, d[u]);
        if (n_keys >= kPageKeys) return;
#pragma unroll
        for (int u = 0; u < N; ++u) {
            const int w = lane * N + u, key = w / (2 * NB) * 4 + 2 * (w & 1);
            if (key >= n_keys) x[u].x = (_Float16)0.0f;
            if (key + 1 >= n_keys) x[u].y = (_Float16)0.0f;
        }
    }
    __device__ half2_t most() const {  // (NaN is no maximum)
        half2_t m = __builtin_elementwise_abs(x[0]);
        if constexpr (N == 2) m = __builtin_elementwise_max(m, __builtin_elementwise_abs(x[1]));
        return m;
    }
    // times the two powers of two in up: d 2^(15 - ve), below 2^16, and exact
    __device__ void scale(half2_t up) {
#pragma unroll
        for (int u = 0; u < N; ++u) x[u] = x[u] * half2_t{up.x, up.x} * half2_t{up.y, up.y};
    }
    __device__ void put(unsigned *d) const {
#pragma unroll
        for (int u = 0; u < N; ++u) d[u] = __builtin_bit_cast(unsigned, x[u]);
    }
};
// The powers of two of the lanes' largest scales, at least those of e.
template <int HD>
__device__ inline unsigned exponents(half2_t most, unsigned e, int lane) {
    float f = fmaxf((float)most.x, (float)most.y);
    if constexpr (HD == 64) f = fmaxf(f, lane8<0>(f));  // the lanes of the block
    f = fmaxf(f, ror<4>(f));
    f = fmaxf(f, ror<8>(f));
    f = col_max(f);
    const int own = exp_byte(e, scale_block<HD>(lane));
    const int byte = max(own, f > 0.0f ? 15 + ilogbf(f) : 0);
    unsigned r = 0;
#pragma unroll
    for (int b = 0; b < HD / 32; ++b)
        r |= __builtin_amdgcn_readlane(byte, HD == 128 ? b : 2 * b) << 8 * b;
    return r;
}
// What the lane's scales are multiplied by: 2^(30 - byte), in two steps.
template <int HD>
__device__ inline half2_t scale_up(unsigned e, int lane) {
    const int up = 30 - exp_byte(e, scale_block<HD>(lane)), half = up >> 1;
    return half2_t{__builtin_bit_cast(_Float16, (short)((15 + half) << 10)),
                   __builtin_bit_cast(_Float16, (short)((15 + up - half) << 10))};
}

// The running softmax of a wave's 16 columns.  Its reference m follows the scores
// only when one is 2^kLazy times larger (sixteen columns would otherwise rescale
// at most pages): p < 2^kLazy, taken in units of 2^kUp, so that p d_v is below 2^15
// in its block's units.  (2^6: three bits less of small p d_v, the same time to 1 %.)
constexpr int kLazy = 3, kUp = kLazy + 1;
template <int HD>
struct Softmax {
    float m = -INFINITY;  // per column, log2 units: within kLazy of the largest score
    float l = 0.0f;       // of this lane's keys; in units of 2^kUp
    unsigned e = 0;       // the powers of two that the value scales are taken in
    float4_t o[HD / 16];  // in units of 2^(kUp + ve - 15 + 9)
    __device__ Softmax() {
#pragma unroll
        for (int e = 0; e < HD / 16; ++e) o[e] = float4_t{0, 0, 0, 0};
    }
    __device__ void units(unsigned e_new) {
#pragma unroll
        for (int b = 0; b < HD / 32; ++b) {
            const float f = ldexpf(1.0f, exp_byte(e, b) - exp_byte(e_new, b));
            o[2 * b] = o[2 * b] * f;
            o[2 * b + 1] = o[2 * b + 1] * f;
        }
        e = e_new;
    }
    // what brings o of a dim tile to l's units
    __device__ float down(int tile) const { return ldexpf(1.0f, 9 - 30 + exp_byte(e, tile / 2)); }
};

// Adds one page.  WHOLE: every column sees its 64 keys; else keys [0, lim) of it
// are seen by this lane's column (none if <= 0).  s_ks, s_vs: its staged scales, the
// values' in the units of st.e.
template <int HD, bool FEW, bool WHOLE, class Src>
__device__ inline void attend_page(const Src &pl, const unsigned *s_ks, const unsigned *s_vs,
                                   int lane, const QTile<HD, FEW> &q, int lim, Softmax<HD> &st) {
    constexpr int NB = HD / 32;
    const int g = lane >> 4;
    float s[16];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        const float4_t v = score_tile<HD, FEW>(pl, s_ks, t, lane, q);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            s[4 * t + i] = WHOLE || 16 * t + 4 * g + i < lim ? v[i] : -INFINITY;
    }
    float pm = s[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) pm = fmaxf(pm, s[i]);
    const float m_new = fmaxf(st.m, col_max(pm) * q.inv);
    if (__any(m_new > st.m + (float)kLazy)) {
        const float f = __builtin_amdgcn_exp2f(st.m - (m_new == -INFINITY ? 0.0f : m_new));
        st.l = st.l * f;
#pragma unroll
        for (int e = 0; e < HD / 16; ++e) st.o[e] = st.o[e] * f;
        st.m = m_new;
    }
    // p 2^-kUp
    const float m0 = (st.m == -INFINITY ? 0.0f : st.m) + (float)kUp;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], q.inv, -m0));
        st.l = st.l + s[i];
    }
    // p d_v of the keys of half h under the scales d: two dwords a tile
    auto weigh = [&](int h, const unsigned (*d)[2], half8_t *hi, half8_t *lo)
                     __attribute__((always_inline)) {
        half2_t hh[4], ll[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {  // keys 16 t + 4 g + 2 (u % 2) + {0, 1}
            const int t = 2 * h + (u >> 1), n = 4 * t + 2 * (u & 1);
            half2_t x = __builtin_bit_cast(half2_t, d[u >> 1][u & 1]);
            if (!WHOLE) {  // a key past the end may hold anything, NaN too
                const int key = 16 * t + 4 * g + 2 * (u & 1);
                if (key >= lim) x.x = (_Float16)0.0f;
                if (key + 1 >= lim) x.y = (_Float16)0.0f;
            }
            split2(fmaf(s[n], (float)x.x, 0.0f), fmaf(s[n + 1], (float)x.y, 0.0f), &hh[u], &ll[u]);
        }
        *hi = join(hh[0], hh[1], hh[2], hh[3]);
        *lo = join(ll[0], ll[1], ll[2], ll[3]);
    };
    // the dims of block b (two tiles in turn, so that no product waits for the last)
    auto sum = [&](int b, int h, half8_t hi, half8_t lo) __attribute__((always_inline)) {
        const half8_t v0 = pl.vop(2 * b, h), v1 = pl.vop(2 * b + 1, h);
        float4_t o0 = st.o[2 * b], o1 = st.o[2 * b + 1];
        o0 = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, lo, o0, 0, 0, 0);
        o1 = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, lo, o1, 0, 0, 0);
        st.o[2 * b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, hi, o0, 0, 0, 0);
        st.o[2 * b + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, hi, o1, 0, 0, 0);
    };
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        if constexpr (FEW) {
            unsigned d[2][2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const uint2 x = reinterpret_cast<const uint2 *>(
                    s_vs + ((2 * h + u) * 4 + g) * 2 * NB)[(lane & 15) / (16 / NB)];
                d[u][0] = x.x, d[u][1] = x.y;
            }
            half8_t hi, lo;
            weigh(h, d, &hi, &lo);
#pragma unroll
            for (int b = 0; b < NB; ++b) sum(b, h, hi, lo);
        } else {
            unsigned dv[2][2 * NB];  // the scales of tiles 2 h and 2 h + 1
#pragma unroll
            for (int u = 0; u < NB; ++u)
                *reinterpret_cast<uint4 *>(&dv[u / (NB / 2)][u % (NB / 2) * 4]) =
                    reinterpret_cast<const uint4 *>(
                        s_vs + ((2 * h + u / (NB / 2)) * 4 + g) * 2 * NB)[u % (NB / 2)];
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const unsigned d[2][2] = {{dv[0][2 * b], dv[0][2 * b + 1]},
                                          {dv[1][2 * b], dv[1][2 * b + 1]}};
                half8_t hi, lo;
                weigh(h, d, &hi, &lo);
                sum(b, h, hi, lo);
            }
        }
    }
}

// How the pages of a call's sequences are dealt to at most `slots` runs (slots
// >= 2 n_seqs) of at most `chunk` pages, chunk the least that suffices: sequence b
// takes ceil(pages_b / chunk) runs, in order.  Every wave computes the same, a
// sequence a lane.  A run has at least min_chunk pages.
__device__ inline unsigned seq_pages(const Kv4Rows &a, int b) {
    unsigned p0;
    const unsigned cnt = rows_of(a, b, &p0);
    return cnt ? (p0 + cnt + kPageKeys - 1) / kPageKeys : 0;
}
// Inclusive sums over the lanes.
__device__ inline unsigned wave_scan_u(unsigned v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr 1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row 0's last to row 1, 2's to 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row 1's last to rows 2, 3
    return v;
}
__device__ inline unsigned wave_sum_u(unsigned v) {
    return __builtin_amdgcn_readlane(wave_scan_u(v), kWave - 1);
}
// ceil(n / d) of n, d < 2^24: the f32 quotient is off by less than one.
__device__ inline unsigned ceil_div(unsigned n, unsigned d, float inv) {
    unsigned q = (unsigned)((float)n * inv);
    q -= q * d > n;
    q += (q + 1) * d <= n;
    return q + (q * d < n);
}
struct Run {
    int b;                // the sequence, -1: no such run
    unsigned first, n;    // its runs
    unsigned pg0, pg1;    // the run's pages
};
__device__ inline Run find_run(const Kv4Rows &a, unsigned slots, unsigned slot,
                               unsigned min_chunk) {
    const int lane = threadIdx.x & 63;
    const unsigned n_seqs = a.n_seqs;
    if (n_seqs == 1) {
        const unsigned np = seq_pages(a, 0), chunk = max((np + slots - 1) / slots, min_chunk);
        const unsigned n = (np + chunk - 1) / chunk;
        return Run{slot < n ? 0 : -1, 0, n, slot * chunk, min(slot * chunk + chunk, np)};
    }
    const unsigned mine = lane < (int)n_seqs ? seq_pages(a, lane) : 0;  // of the first 64
    unsigned total = mine;
    for (unsigned b = lane + kWave; b < n_seqs; b += kWave) total += seq_pages(a, b);
    total = wave_sum_u(total);
    // ceil(total / slots) is too few pages, or just enough; ceil(total / (slots -
    // n_seqs)) suffices, for each sequence has one short run at most
    unsigned lo = max((total + slots - 1) / slots, min_chunk);
    unsigned hi = max((total + slots - n_seqs - 1) / (slots - n_seqs), min_chunk);
    while (lo < hi) {
        const unsigned mid = (lo + hi) >> 1;
        const float inv = 1.0f / (float)mid;
        unsigned runs = ceil_div(mine, mid, inv);
        for (unsigned b = lane + kWave; b < n_seqs; b += kWave)
            runs += ceil_div(seq_pages(a, b), mid, inv);
        if (wave_sum_u(runs) <= slots) hi = mid;
        else lo = mid + 1;
    }
    const float inv = 1.0f / (float)lo;
    unsigned before = 0;
    for (unsigned b0 = 0; b0 < n_seqs; b0 += kWave) {
        const unsigned np = b0 == 0 ? mine : b0 + lane < n_seqs ? seq_pages(a, b0 + lane) : 0;
        const unsigned n = ceil_div(np, lo, inv), inc = wave_scan_u(n);
        const unsigned long long over = __ballot(before + inc > slot);
        if (over) {
            const int l = __ffsll((long long)over) - 1;
            Run r;
            r.b = (int)b0 + l;
            r.n = __builtin_amdgcn_readlane(n, l);
            r.first = before + __builtin_amdgcn_readlane(inc, l) - r.n;
            r.pg0 = (slot - r.first) * lo;
            r.pg1 = min(r.pg0 + lo, (unsigned)__builtin_amdgcn_readlane(np, l));
            return r;
        }
        before += __builtin_amdgcn_readlane(inc, kWave - 1);
    }
    return Run{-1, 0, 0, 0, 0};
}

// Partial results go through the memory that all XCDs see, two floats an access.
__device__ inline void part_store(float *p, float a, float b) {
    const unsigned long long v =
        (unsigned long long)__float_as_uint(b) << 32 | __float_as_uint(a);
    __hip_atomic_store(reinterpret_cast<unsigned long long *>(p), v, __ATOMIC_RELAXED,
                       __HIP_MEMORY_SCOPE_AGENT);
}
__device__ inline float2 part_load(const float *p) {
    const unsigned long long v =
        __hip_atomic_load(reinterpret_cast<const unsigned long long *>(p), __ATOMIC_RELAXED,
                          __HIP_MEMORY_SCOPE_AGENT);
    return float2{__uint_as_float((unsigned)v), __uint_as_float((unsigned)(v >> 32))};
}

// Waves of a workgroup, and workgroups of a CU where keys are split (registers
// leave two waves a SIMD at head dim 128, three at 64).
constexpr int waves_of(int hd, bool split) { return split && hd == 128 ? 8 : 4; }
constexpr int wgs_of(int hd) { return hd == 128 ? 1 : 3; }

// Grid: slots x (KV heads x query tiles).  SPLIT: a slot is a run of pages of
// one sequence; else it is a sequence.  The waves take its pages in turn and meet
// in LDS.  Where a sequence has several runs, each publishes its columns'
// (m, l, o) in `part` by device-scope stores that are complete before it counts
// itself on the tile's counter; the one that counts last joins them in the order
// of the runs and leaves the counter zero, so none waits for another.
// A token of 32 heads over 8 of 128, 8 sequences of 32768 keys: 47 us for 196 MB of
// pages (4.1 TB/s, 90 % of a large copy's rate).
template <int HD, bool FEW, bool SPLIT>
__global__ __launch_bounds__(waves_of(HD, SPLIT) * kWave, 2) void k_kv4_attend(
    Kv4Rows a, const float *__restrict__ q, size_t qs, bool vec, int groups, int n_qt,
    unsigned slots, float *__restrict__ out, size_t os, float *__restrict__ part,
    int *__restrict__ cnts, float *__restrict__ lse) {
    using P = Page<HD>;
    constexpr int NQ = QTile<HD, FEW>::NQ;  // queries of a tile
    constexpr int kWaves = waves_of(HD, SPLIT);
    __shared__ float s_m[kWaves][NQ], s_l[kWaves][NQ];
    __shared__ __attribute__((aligned(16))) float s_o[kWaves][NQ][HD + 4];
    __shared__ __attribute__((aligned(16))) unsigned s_d[kWaves][2][kScaleWords<HD>];
    __shared__ int s_last;
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, g = lane >> 4, r = lane & 15;
    const int qt = blockIdx.x % n_qt, head = blockIdx.x / n_qt % a.n_kv;
    const unsigned slot = blockIdx.x / (n_qt * a.n_kv);
    Run run{(int)slot, 0, 1, 0, 0};
    if constexpr (SPLIT) {
        // two pages a wave cost less than another workgroup's partial results
        run = find_run(a, slots, slot, 2 * kWaves);
        run = Run{uniform(run.b), uniform(run.first), uniform(run.n), uniform(run.pg0),
                  uniform(run.pg1)};
        if (run.b < 0) return;
    }
    const int b = run.b;
    unsigned p0;
    const int cnt = (int)rows_of(a, b, &p0);
    const int n_q = cnt * groups;       // real queries of the KV head
    if (qt * NQ >= n_q) return;
    const int last_row = (min(qt * NQ + NQ, n_q) - 1) / groups;
    const unsigned end = p0 + last_row + 1;  // keys that the tile's last row sees
    const unsigned end_pg = (end + kPageKeys - 1) / kPageKeys;
    const unsigned pg1 = SPLIT ? min(run.pg1, end_pg) : end_pg;
    // a page's loads are in flight while the one before it is computed
    const uint8_t *base =
        a.pages + ((size_t)(a.first_seq + b) * a.n_kv + head) * a.n_pages * P::kBytes;
    PageLoad<HD> next;
    unsigned pg = run.pg0 + wv;
    if (pg < pg1) next.load(base + (size_t)pg * P::kBytes, lane);
    const int qi = qt * NQ + r % NQ, row = qi / groups;
    const bool real = qi < n_q;
    QRaw<HD, FEW> raw;
    raw.load(real ? q + row_index(a, b, row) * qs + (head * groups + qi % groups) * HD : nullptr,
             g, r / NQ, vec);
    QTile<HD, FEW> qtile;
    qtile.make(raw, lane);
    const long see = real ? (long)p0 + row + 1 : 0;      // keys this column sees
    const unsigned all = p0 + (qt * NQ) / groups + 1;    // keys every real column sees
    Softmax<HD> st;
    half2_t up = scale_up<HD>(st.e, lane);
    for (; pg < pg1; pg += kWaves) {
        PageLoad<HD> now = next;
        ValueScales<HD> vs(now.vs, lane, (int)min(end - pg * kPageKeys, 64u)), up_vs = vs;
        up_vs.scale(up);
        const half2_t top = up_vs.most();
        constexpr int kInf = 0x200;  // past 2^16: a block's power of two has to grow
        if (__any(__builtin_amdgcn_classh(top.x, kInf) || __builtin_amdgcn_classh(top.y, kInf))) {
            st.units(exponents<HD>(vs.most(), st.e, lane));
            up = scale_up<HD>(st.e, lane);
            up_vs = vs;
            up_vs.scale(up);
        }
        up_vs.put(now.vs);
        __builtin_amdgcn_wave_barrier();  // the last page's scales are read (LDS is in order)
        PageLoad<HD>::stage(now.ks, lane, s_d[wv][0]);
        PageLoad<HD>::stage(now.vs, lane, s_d[wv][1]);
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        if (pg + kWaves < pg1) next.load(base + (size_t)(pg + kWaves) * P::kBytes, lane);
        const int lim = (int)min(see - (long)pg * kPageKeys, 64l);
        if ((pg + 1) * kPageKeys <= all)
            attend_page<HD, FEW, true>(now, s_d[wv][0], s_d[wv][1], lane, qtile, lim, st);
        else
            attend_page<HD, FEW, false>(now, s_d[wv][0], s_d[wv][1], lane, qtile, lim, st);
    }
    // the column's sum over its four lane groups, then the waves
    st.l = col_sum(st.l);
    if (g == 0 && r < NQ) {
        s_m[wv][r] = st.m;
        s_l[wv][r] = st.l;
    }
#pragma unroll
    for (int e = 0; e < HD / 16; ++e)
        if (!FEW || e / 2 == r / NQ)
            *reinterpret_cast<float4_t *>(&s_o[wv][r % NQ][16 * e + 4 * g]) =
                st.o[e] * st.down(e);
    __syncthreads();
    const int cols = min(NQ, n_q - qt * NQ);
    const size_t z0 = ((size_t)b * a.rows) * (a.n_kv * groups);
    // four dims of a column from d on
    auto store = [&](int c, int d, float m, float l, const float *o) {
        const int ci = qt * NQ + c, oh = head * groups + ci % groups;
        float *to = out + row_index(a, b, ci / groups) * os + oh * HD + d;
#pragma unroll
        for (int j = 0; j < 4; ++j) to[j] = o[j] / l;
        if (lse && d == 0)
            lse[z0 + (size_t)(ci / groups) * (a.n_kv * groups) + oh] =
                m + __log2f(l * ldexpf(1.0f, kUp));
    };
    const bool alone = !SPLIT || run.n == 1;
    // partial results of run i, column c
    auto part_of = [&](unsigned i, int c) {
        return part + ((((size_t)(run.first + i) * a.n_kv + head) * n_qt + qt) * NQ + c) * (HD + 2);
    };
    for (int it = threadIdx.x; it < cols * (HD / 4); it += kWaves * kWave) {
        const int c = it / (HD / 4), d = it % (HD / 4) * 4;
        float m = s_m[0][c];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) m = fmaxf(m, s_m[w][c]);
        const float m_use = m == -INFINITY ? 0.0f : m;
        float l = 0.0f, o[4] = {0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float f = __builtin_amdgcn_exp2f(s_m[w][c] - m_use);
            const float4_t x = *reinterpret_cast<const float4_t *>(&s_o[w][c][d]);
            l = l + s_l[w][c] * f;
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] = o[j] + x[j] * f;
        }
        if (alone) {
            store(c, d, m_use, l, o);
        } else {
            float *pc = part_of(slot - run.first, c);
            part_store(pc + 2 + d, o[0], o[1]);
            part_store(pc + 4 + d, o[2], o[3]);
            if (d == 0) part_store(pc, m, l);
        }
    }
    if (alone) return;
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this thread's partials are at the device
    __syncthreads();
    int *cn = cnts + ((size_t)b * a.n_kv + head) * n_qt + qt;
    if (threadIdx.x == 0)
        s_last = __hip_atomic_fetch_add(cn, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
                 (int)run.n - 1;
    __syncthreads();
    if (!s_last) return;
    if (threadIdx.x == 0) __hip_atomic_store(cn, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    for (int it = threadIdx.x; it < cols * (HD / 4); it += kWaves * kWave) {
        const int c = it / (HD / 4), d = it % (HD / 4) * 4;
        constexpr unsigned B = 8;
        float m = -INFINITY, l = 0.0f, o[4] = {0, 0, 0, 0};
        for (unsigned i0 = 0; i0 < run.n; i0 += B) {  // B runs' loads in flight
            float2 ml[B], x[B][2];
#pragma unroll
            for (unsigned u = 0; u < B; ++u) {
                const float *pc = part_of(min(i0 + u, run.n - 1), c);
                ml[u] = part_load(pc);
                x[u][0] = part_load(pc + 2 + d);
                x[u][1] = part_load(pc + 4 + d);
            }
            float mn = m;
#pragma unroll
            for (unsigned u = 0; u < B; ++u) mn = fmaxf(mn, ml[u].x);
            const float m_use = mn == -INFINITY ? 0.0f : mn, f0 = __builtin_amdgcn_exp2f(m - m_use);
            l = l * f0;
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] = o[j] * f0;
            m = mn;
#pragma unroll
            for (unsigned u = 0; u < B; ++u) {
                if (i0 + u < run.n) {
                    const float f = __builtin_amdgcn_exp2f(ml[u].x - m_use);
                    l = l + ml[u].y * f;
                    o[0] = o[0] + x[u][0].x * f;
                    o[1] = o[1] + x[u][0].y * f;
                    o[2] = o[2] + x[u][1].x * f;
                    o[3] = o[3] + x[u][1].y * f;
                }
            }
        }
        store(c, d, m, l, o);
    }
}

// A tile's 16 rows on their way to LDS, as a load takes four of them: sixteen lanes a
// row, four dims of each 64.  (Whole lines a load: with a row's dims over four lanes,
// 16 half lines a load, issuing the loads takes as long as the products: 91 us, not 76.)
template <int HD>
struct QRows {
    static constexpr int N = HD / 64;
    float4_t x[4][N];
    // src null: an empty row
    __device__ void load(int i, const float *src, int l, bool vec) {
#pragma unroll
        for (int h = 0; h < N; ++h) {
            const float *p = src + 64 * h + 4 * l;
            if (!src) {
                x[i][h] = float4_t{0, 0, 0, 0};
            } else if (vec) {
                x[i][h] = *reinterpret_cast<const float4_t *>(p);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) x[i][h][j] = p[j];
            }
        }
    }
    // As the products take them: [block][hi, lo][at].  The groups' and blocks' rows
    // are turned against each other, so that a store's lanes have banks of their own.
    static __device__ int at(int block, int g, int row) {
        return 16 * g + (row ^ 4 * g ^ 2 * (block & 1));
    }
    __device__ void store(half8_t (*to)[2][kWave], float *inv, int lane) const {
        const int l = lane & 15;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = 4 * i + (lane >> 4);
            float mx = 0.0f;
#pragma unroll
            for (int h = 0; h < N; ++h)
#pragma unroll
                for (int j = 0; j < 4; ++j) mx = fmaxf(mx, fabsf(x[i][h][j]));
            mx = fmaxf(mx, ror<8>(mx));
            mx = fmaxf(mx, ror<4>(mx));
            mx = fmaxf(mx, ror<2>(mx));
            mx = fmaxf(mx, ror<1>(mx));
            const int e = up_exponent(mx);
            const float up = ldexpf(1.0f, e);
#pragma unroll
            for (int h = 0; h < N; ++h) {
                half2_t hi[2], lo[2];
#pragma unroll
                for (int u = 0; u < 2; ++u)
                    split2(x[i][h][2 * u] * up, x[i][h][2 * u + 1] * up, &hi[u], &lo[u]);
                half8_t *const p = &to[2 * h + (l >> 3)][0][at(l >> 3, l >> 1 & 3, row)];
                reinterpret_cast<uint2 *>(p)[l & 1] = __builtin_bit_cast(uint2, hi);
                reinterpret_cast<uint2 *>(p + kWave)[l & 1] = __builtin_bit_cast(uint2, lo);
            }
            if (l == 0) inv[row] = score_scale<HD>(e);
        }
    }
};

// Prompts: a workgroup takes 64 queries of a KV head over all the pages they see,
// a tile of 16 a wave.  The waves turn each page's quants into f16 operands once,
// a quarter each, and read them from LDS in the operands' order; the next page
// comes in while this one is computed, into a second buffer (one barrier a page).
// The workgroups with the most pages start first.  1999 rows of 32 heads of 128:
// 123 us, 57 of them the products (both halves) at a large product's rate; the rest
// is VALU work (unpacking, softmax, p d_v) that two waves a SIMD hide in part, and
// each workgroup's first loads (5 us).
// Eight waves a workgroup: 129.  The values' powers of two are found before the pages, from
// their scales alone: following them page by page, as k_kv4_attend does, holds up the
// barrier (131).
constexpr int kPromptWaves = 4;
template <int HD>
struct LdsPage {
    static constexpr int NB = HD / 32;
    half8_t k[4][NB][kWave];
    half8_t v[HD / 16][2][kWave];
    unsigned d[2][kScaleWords<HD>];
};
template <int HD>
struct LdsSrc {
    const LdsPage<HD> &p;
    int lane;
    __device__ half8_t kop(int t, int b) const { return p.k[t][b][lane]; }
    __device__ half8_t vop(int e, int h) const { return p.v[e][h][lane]; }
};
// What a thread holds of a page on its way to LDS: K tile `wave`, V chunk `wave`
// (head dim 64: the first two waves), and K's scales in the first wave, V's in the second.
// (The others hold them too: with a branch around them, the second wave's products come
// last before each barrier: 512 rows behind 32000 keys 1030 us for 1003.)
template <int HD>
struct PagePart {
    using P = Page<HD>;
    static constexpr int NB = HD / 32;
    unsigned k[NB], v[4], d[NB / 2];
    __device__ void load(const uint8_t *pb, int wv, int lane) {
        const uint8_t *kp = pb + wv * 8 * HD + lane * 4 * NB;
        if constexpr (HD == 128) {
            const uint4 x = *reinterpret_cast<const uint4 *>(kp);
            k[0] = x.x, k[1] = x.y, k[2] = x.z, k[3] = x.w;
        } else {
            const uint2 x = *reinterpret_cast<const uint2 *>(kp);
            k[0] = x.x, k[1] = x.y;
        }
        if (wv < NB) {
            const uint4 x = *reinterpret_cast<const uint4 *>(pb + P::kV + wv * 1024 + lane * 16);
            v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
        }
        PageLoad<HD>::load_scales(pb + (wv & 1 ? P::kVs : P::kKs), lane, d);
    }
    // up: what the wave's scales are multiplied by (those past the end may become infinite)
    __device__ void store(LdsPage<HD> &p, int wv, int lane, half2_t up) {
        ValueScales<HD> ds(d, lane, kPageKeys);
        ds.scale(up);
        ds.put(d);
#pragma unroll
        for (int b = 0; b < NB; ++b) p.k[wv][b][lane] = quants(k[b]);
        if (wv < NB) {
#pragma unroll
            for (int i = 0; i < 4; ++i) p.v[2 * wv + (i >> 1)][i & 1][lane] = quants(v[i]);
        }
        if (wv < 2) PageLoad<HD>::stage(d, lane, p.d[wv]);
    }
};

template <int HD>
__global__ __launch_bounds__(kPromptWaves *kWave, 2) void k_kv4_prompt(
    Kv4Rows a, const float *__restrict__ q, size_t qs, bool vec, int groups, int n_qg,
    float *__restrict__ out, size_t os, float *__restrict__ lse) {
    using P = Page<HD>;
    constexpr int QW = kPromptWaves * 16;  // queries of a workgroup
    constexpr int NB = P::NB;
    __shared__ LdsPage<HD> s_p[2];
    __shared__ float s_inv[kPromptWaves][16];
    __shared__ unsigned s_e[kPromptWaves];
    const int lane = threadIdx.x & 63, wv = wave_id(), g = lane >> 4, r = lane & 15;
    unsigned x = blockIdx.x;
    const int head = x % a.n_kv;
    x /= a.n_kv;
    const int b = x % a.n_seqs, qg = n_qg - 1 - (int)(x / a.n_seqs);
    unsigned p0;
    const int cnt = (int)rows_of(a, b, &p0);
    const int n_q = cnt * groups;
    if (qg * QW >= n_q) return;
    const unsigned n_keys = p0 + (min(qg * QW + QW, n_q) - 1) / groups + 1;
    const unsigned n_pg = (n_keys + kPageKeys - 1) / kPageKeys;
    const uint8_t *base =
        a.pages + ((size_t)(a.first_seq + b) * a.n_kv + head) * a.n_pages * P::kBytes;
    PagePart<HD> next;
    next.load(base, wv, lane);
    // the largest value scales of all the pages, a quarter of them a wave
    half2_t most = {(_Float16)0.0f, (_Float16)0.0f};
#pragma unroll 4
    for (unsigned pg = wv; pg < n_pg; pg += kPromptWaves) {
        unsigned d[NB / 2];
        PageLoad<HD>::load_scales(base + (size_t)pg * P::kBytes + P::kVs, lane, d);
        const ValueScales<HD> vs(d, lane, (int)min(n_keys - pg * kPageKeys, 64u));
        most = __builtin_elementwise_max(most, vs.most());
    }
    const int q0 = qg * QW + wv * 16, qi = q0 + r, row = qi / groups;
    const bool real = qi < n_q;
    const int qh = head * groups + qi % groups;
    // the queries pass through the second page's place
    static_assert(sizeof(half8_t) * kPromptWaves * NB * 2 * kWave <= sizeof(LdsPage<HD>));
    half8_t(*const s_q)[2][kWave] = reinterpret_cast<half8_t(*)[2][kWave]>(&s_p[1]) + wv * NB;
    {
        QRows<HD> rows;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int at = q0 + 4 * i + g;
            rows.load(i,
                      at < n_q ? q + row_index(a, b, at / groups) * qs +
                                     (head * groups + at % groups) * HD
                               : nullptr,
                      r, vec);
        }
        rows.store(s_q, s_inv[wv], lane);
    }
    const long see = real ? (long)p0 + row + 1 : 0;  // keys this column sees
    // keys every real column of the wave sees
    const unsigned all = q0 < n_q ? p0 + q0 / groups + 1 : 0;
    // pages that the wave's last row sees
    const unsigned my_pg =
        q0 < n_q ? (p0 + (min(q0 + 16, n_q) - 1) / groups) / kPageKeys + 1 : 0;
    Softmax<HD> st;
    const unsigned most_e = exponents<HD>(most, 0, lane);
    if (lane == 0) s_e[wv] = most_e;
    __syncthreads();
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        int byte = 0;
#pragma unroll
        for (int w = 0; w < kPromptWaves; ++w) byte = max(byte, exp_byte(s_e[w], b));
        st.e |= uniform((unsigned)byte) << 8 * b;
    }
    const half2_t one = {(_Float16)1.0f, (_Float16)1.0f};
    const half2_t up = wv == 1 ? scale_up<HD>(st.e, lane) : one;
    next.store(s_p[0], wv, lane, up);
    QTile<HD, false> qtile;
#pragma unroll
    for (int c = 0; c < NB; ++c) {
        qtile.hi[c] = s_q[c][0][QRows<HD>::at(c, g, r)];
        qtile.lo[c] = s_q[c][1][QRows<HD>::at(c, g, r)];
    }
    qtile.inv = s_inv[wv][r];
    __syncthreads();
    for (unsigned pg = 0; pg < n_pg; ++pg) {
        const LdsSrc<HD> src{s_p[pg & 1], lane};
        if (pg + 1 < n_pg) next.load(base + (size_t)(pg + 1) * P::kBytes, wv, lane);
        const int lim = (int)min(see - (long)pg * kPageKeys, 64l);
        if ((pg + 1) * kPageKeys <= all)
            attend_page<HD, false, true>(src, src.p.d[0], src.p.d[1], lane, qtile, lim, st);
        else if (pg < my_pg)
            attend_page<HD, false, false>(src, src.p.d[0], src.p.d[1], lane, qtile, lim, st);
        if (pg + 1 < n_pg) next.store(s_p[(pg + 1) & 1], wv, lane, up);
        __syncthreads();
    }
    const float l = col_sum(st.l);
    if (!real) return;
    float *to = out + row_index(a, b, row) * os + qh * HD + 4 * g;
    const float inv = 1.0f / l;
#pragma unroll
    for (int e = 0; e < HD / 16; ++e) {
        const float f = st.down(e) * inv;
#pragma unroll
        for (int i = 0; i < 4; ++i) to[16 * e + i] = st.o[e][i] * f;
    }
    if (lse && g == 0)
        lse[((size_t)b * a.rows + row) * (a.n_kv * groups) + qh] =
            st.m + __log2f(l * ldexpf(1.0f, kUp));
}

// The keys' attention weights: a wave a page of a KV head goes over all the
// queries that see it, with the scores of the attention itself and the rows'
// log-sum-exps; the page's quants stay in its registers.  The four waves of a
// workgroup (consecutive pages) prepare a query tile each and share the four
// through LDS.  Where pages alone do not fill the CUs, n_parts workgroups take
// every n_parts-th batch of four tiles, and the one that is done last adds their
// sums in order: each key has one writer and one order of sums.
// 1999 rows of 32 heads of 128: 71 us; scores alone are 29 at the rate of a large
// product.  Two waves a SIMD (registers) wait for their products and the scales'
// turns; eight waves to a tile batch 103, blocks outermost 98 (more chains, 219
// registers), three waves a SIMD without tiles loaded ahead 102.
constexpr int kWtWaves = 4;
template <int HD>
__global__ __launch_bounds__(kWtWaves *kWave, 2) void k_kv4_weights(
    Kv4Rows a, const float *__restrict__ q, size_t qs, bool vec, int groups, int n_grp,
    int n_parts, const float *__restrict__ lse, float *__restrict__ weights,
    float *__restrict__ part, int *__restrict__ cnts) {
    using P = Page<HD>;
    constexpr int NB = P::NB;
    __shared__ half8_t s_q[kWtWaves][NB][2][kWave];
    __shared__ float s_inv[kWtWaves][16], s_z[kWtWaves][16];
    __shared__ unsigned s_see[kWtWaves][16];
    __shared__ __attribute__((aligned(16))) unsigned s_d[kWtWaves][kScaleWords<HD>];
    __shared__ float s_w[kWtWaves][kPageKeys];
    __shared__ int s_last;
    const int lane = threadIdx.x & 63, wv = wave_id(), g = lane >> 4, r = lane & 15;
    unsigned x = blockIdx.x;
    const int mine = x % n_parts;
    x /= n_parts;
    const int head = x % a.n_kv;
    x /= a.n_kv;
    const int b = x % a.n_seqs, grp = x / a.n_seqs;  // (the first keys have the most queries)
    unsigned p0;
    const int cnt = (int)rows_of(a, b, &p0);
    const unsigned end = p0 + cnt, key0 = grp * kWtWaves * kPageKeys;
    if (cnt == 0 || key0 >= end) return;
    const unsigned pg = grp * kWtWaves + wv, pkey = pg * kPageKeys;
    const bool has = pkey < end;
    const int n_q = cnt * groups;
    float w[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) w[i] = 0.0f;
    half8_t kq[4][NB];
    if (has) {
        PageLoad<HD> pl;
        pl.load_k(a.pages + (((size_t)(a.first_seq + b) * a.n_kv + head) * a.n_pages + pg) *
                                P::kBytes,
                  lane);
        PageLoad<HD>::stage(pl.ks, lane, s_d[wv]);
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int c = 0; c < NB; ++c) kq[t][c] = quants(pl.k[t][c]);
    }
    // Batches from the last down to the first whose rows see the group's first key:
    // all groups of a head go over the same tiles at the same time, so that their
    // XCD's cache serves most of them.  A tile's queries are loaded while the batch
    // before it is computed.
    const int qt0 = (key0 > p0 ? (int)(key0 - p0) : 0) * groups / 16 / kWtWaves * kWtWaves;
    const int n_qt = (n_q + 15) / 16, step = n_parts * kWtWaves;
    const int last = ((n_qt - 1) / kWtWaves - mine) / n_parts * n_parts + mine;
    QRows<HD> rows;
    float z_next = 0.0f;
    unsigned see_next = 0;
    auto fetch = [&](int t) {
        unsigned row = (t * 16 + g) / (unsigned)groups, col = (t * 16 + g) % (unsigned)groups;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool real = t * 16 + 4 * i + g < n_q;
            rows.load(i, real ? q + row_index(a, b, row) * qs + (head * groups + col) * HD : nullptr,
                      r, vec);
            row += 4 / groups;  // four queries on
            col += 4 % groups;
            if (col >= (unsigned)groups) ++row, col -= groups;
        }
        const unsigned qi = t * 16 + r;
        row = qi / (unsigned)groups;
        const bool real = qi < (unsigned)n_q;
        see_next = real ? p0 + row + 1 : 0;
        z_next = real ? lse[((size_t)b * a.rows + row) * (a.n_kv * groups) + head * groups +
                            qi % (unsigned)groups]
                      : 0.0f;
    };
    const int q_last = (n_qt - 1) / kWtWaves >= mine ? last * kWtWaves : -1;
    if (q_last >= qt0) fetch(q_last + wv);
    for (int q0 = q_last; q0 >= qt0; q0 -= step) {
        const int nt = min(kWtWaves, n_qt - q0);
        rows.store(s_q[wv], s_inv[wv], lane);
        if (g == 0) {
            s_z[wv][r] = z_next;
            s_see[wv][r] = see_next;
        }
        __syncthreads();
        if (q0 - step >= qt0) fetch(q0 - step + wv);
        // the first of the tiles whose last row sees this wave's page
        for (int u = 0; u < nt && has; ++u) {
            const int c0 = (q0 + u) * 16, c1 = min(c0 + 16, n_q) - 1;
            if (p0 + c1 / groups < pkey) continue;
            const bool whole = c0 + 16 <= n_q && p0 + c0 / groups + 1 >= pkey + kPageKeys;
            const float inv = s_inv[u][r], z = s_z[u][r];
            const int lim = (int)(s_see[u][r] - min(pkey, s_see[u][r]));
            half8_t hi[NB], lo[NB];
#pragma unroll
            for (int c = 0; c < NB; ++c) {
                hi[c] = s_q[u][c][0][rows.at(c, g, r)];
                lo[c] = s_q[u][c][1][rows.at(c, g, r)];
            }
            float s[16];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                unsigned kd[2 * NB];  // the scales of this lane's keys
#pragma unroll
                for (int c = 0; c < NB / 2; ++c)
                    *reinterpret_cast<uint4 *>(kd + 4 * c) =
                        reinterpret_cast<const uint4 *>(s_d[wv] + (t * 4 + g) * 2 * NB)[c];
#pragma unroll
                for (int c = 0; c < NB; ++c) {
                    float4_t y = {0, 0, 0, 0};
                    y = __builtin_amdgcn_mfma_f32_16x16x32_f16(kq[t][c], lo[c], y, 0, 0, 0);
                    y = __builtin_amdgcn_mfma_f32_16x16x32_f16(kq[t][c], hi[c], y, 0, 0, 0);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const half2_t d = __builtin_bit_cast(half2_t, kd[2 * c + (i >> 1)]);
                        const float x = (float)(i & 1 ? d.y : d.x);
                        s[4 * t + i] = c == 0 ? y[i] * x : fmaf(y[i], x, s[4 * t + i]);
                    }
                }
            }
            if (whole) {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    w[i] = w[i] + __builtin_amdgcn_exp2f(fmaf(s[i], inv, -z));
            } else {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (16 * (i >> 2) + 4 * g + (i & 3) < lim)
                        w[i] = w[i] + __builtin_amdgcn_exp2f(fmaf(s[i], inv, -z));
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        float v = w[i];
        v = v + ror<8>(v);
        v = v + ror<4>(v);
        v = v + ror<2>(v);
        v = v + ror<1>(v);
        if (r == 0) s_w[wv][16 * (i >> 2) + 4 * g + (i & 3)] = v;
    }
    __syncthreads();
    float sum = s_w[wv][lane];
    const size_t row = (size_t)b * a.n_kv + head;
    if (n_parts > 1) {
        float *pp = part + (row * n_grp + grp) * n_parts * (kWtWaves * kPageKeys) + threadIdx.x;
        __hip_atomic_store(pp + mine * (kWtWaves * kPageKeys), sum, __ATOMIC_RELAXED,
                           __HIP_MEMORY_SCOPE_AGENT);
        __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): the sums are at the device
        __syncthreads();
        int *cn = cnts + row * n_grp + grp;
        if (threadIdx.x == 0)
            s_last = __hip_atomic_fetch_add(cn, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
                     n_parts - 1;
        __syncthreads();
        if (!s_last) return;
        if (threadIdx.x == 0)
            __hip_atomic_store(cn, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        sum = 0.0f;
        for (int i = 0; i < n_parts; ++i)
            sum = sum + __hip_atomic_load(pp + i * (kWtWaves * kPageKeys), __ATOMIC_RELAXED,
                                          __HIP_MEMORY_SCOPE_AGENT);
    }
    const unsigned key = pkey + lane;
    if (key < end) {
        float *to = weights + ((size_t)(a.first_seq + b) * a.n_kv + head) * a.max_seq + key;
        *to = (key < p0 ? *to : 0.0f) + sum;
    }
}

// ---- eviction ------------------------------------------------------------------------
// Weights as unsigned keys in their order; NaN below all, -0 as 0.
__device__ inline unsigned weight_key(float w) {
    if (w != w) return 0u;
    const unsigned b = __float_as_uint(w == 0.0f ? 0.0f : w);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

// The kept positions of one (layer, sequence, KV head) a workgroup: the k-th
// largest weight by three passes over its bits (11, 11 and 10, counts in LDS: an
// exponent alone would put most weights on a few counters), then the positions
// above it and the first of those equal to it, in order: each wave counts and
// writes contiguous positions.  Weights of a cache of up to 32768 positions are read
// once, into registers (128 heads of 32768 keys to 1024: 58 us a call; 103 in a cache of
// 32832; 256 heads of 2304 keys to 2048: 63, and 57 in a cache of 32832).
// 256 rows of 2304: 13 us, three passes' latency; 128 of 32768: 23 us.
constexpr int kSelThreads = 1024, kSelWaves = kSelThreads / kWave, kSelBins = 2048;
constexpr int kSelRegs = 32;
template <bool REGS>
__global__ __launch_bounds__(kSelThreads) void k_kv4_select(Kv4Evict e) {
    __shared__ unsigned s_hist[kSelBins];
    __shared__ unsigned s_wave[kSelWaves], s_digit, s_left;
    __shared__ unsigned s_gt[kSelWaves], s_eq[kSelWaves];
    const int t = threadIdx.x, lane = t & 63, wv = wave_id();
    const size_t rowi = e.row0 + blockIdx.x;
    const int b = (int)(rowi / e.n_kv % e.n_seqs);
    const unsigned n = min(e.lens[b], e.src_max);
    uint32_t *kept = e.kept + rowi * e.keep;
    if (n <= e.keep) {
        for (unsigned i = t; i < e.keep; i += kSelThreads) kept[i] = i < n ? i : MRI_NO_TOKEN;
        return;
    }
    const float *w = e.w + rowi * e.src_max;
    const unsigned old = n - e.recent, take = e.keep - e.recent;
    for (unsigned i = t; i < e.recent; i += kSelThreads) kept[take + i] = old + i;
    if (take == 0) return;
    // wave wv has positions [wv seg, (wv + 1) seg), 64 at a time
    const unsigned seg = ((old + kSelWaves - 1) / kSelWaves + kWave - 1) / kWave * kWave;
    const unsigned i0 = min(wv * seg, old), i1 = min(i0 + seg, old);
    unsigned reg[REGS ? kSelRegs : 1];
    if constexpr (REGS) {
#pragma unroll
        for (int u = 0; u < kSelRegs; ++u) {
            const unsigned i = i0 + u * kWave + lane;
            reg[u] = i < i1 ? __float_as_uint(w[i]) : 0;
        }
#pragma unroll
        for (int u = 0; u < kSelRegs; ++u) reg[u] = weight_key(__uint_as_float(reg[u]));
    }
    // f(key, position) of each of the wave's positions, 64 at a time; ok: a real one
    auto each = [&](auto &&f) __attribute__((always_inline)) {
        if constexpr (REGS) {
#pragma unroll
            for (int u = 0; u < kSelRegs; ++u) {
                const unsigned i = i0 + u * kWave;
                if (i < i1) f(reg[u], i + lane, i + lane < i1);
            }
        } else {
            for (unsigned i = i0; i < i1; i += kWave)
                f(i + lane < i1 ? weight_key(w[i + lane]) : 0u, i + lane, i + lane < i1);
        }
    };
    unsigned prefix = 0, left = take;  // the bits so far; how many to take below them
#pragma unroll
    for (int pass = 0; pass < 3; ++pass) {
        const int sh = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
        s_hist[t] = 0;
        s_hist[t + kSelThreads] = 0;
        __syncthreads();
        each([&](unsigned key, unsigned, bool ok) {
            if (ok && (pass == 0 || (key >> (sh + bits)) == prefix))
                atomicAdd(&s_hist[key >> sh & ((1u << bits) - 1)], 1u);
        });
        __syncthreads();
        // thread t holds digits 2047 - 2 t and 2046 - 2 t, from the largest down
        const unsigned c0 = s_hist[kSelBins - 1 - 2 * t], c1 = s_hist[kSelBins - 2 - 2 * t];
        const unsigned inc = wave_scan_u(c0 + c1);
        if (lane == kWave - 1) s_wave[wv] = inc;
        __syncthreads();
        const unsigned ends = wave_scan_u(lane < kSelWaves ? s_wave[lane] : 0);
        const unsigned above =
            inc - c0 - c1 + (wv ? __builtin_amdgcn_readlane(ends, wv - 1) : 0);
        if (above < left && left <= above + c0) {
            s_digit = kSelBins - 1 - 2 * t;
            s_left = left - above;
        } else if (above + c0 < left && left <= above + c0 + c1) {
            s_digit = kSelBins - 2 - 2 * t;
            s_left = left - above - c0;
        }
        __syncthreads();
        prefix = prefix << bits | s_digit;
        left = s_left;
        __syncthreads();
    }
    // keys > prefix are taken, and the first `left` of those equal to it
    unsigned gt = 0, eq = 0;
    each([&](unsigned key, unsigned, bool ok) {
        gt += __popcll(__ballot(ok && key > prefix));
        eq += __popcll(__ballot(ok && key == prefix));
    });
    if (lane == 0) {
        s_gt[wv] = gt;
        s_eq[wv] = eq;
    }
    __syncthreads();
    gt = wave_scan_u(lane < kSelWaves ? s_gt[lane] : 0);
    eq = wave_scan_u(lane < kSelWaves ? s_eq[lane] : 0);
    gt = wv ? __builtin_amdgcn_readlane(gt, wv - 1) : 0;
    eq = wv ? __builtin_amdgcn_readlane(eq, wv - 1) : 0;
    const unsigned long long below = (1ull << lane) - 1;
    each([&](unsigned key, unsigned i, bool ok) {
        const unsigned long long bg = __ballot(ok && key > prefix),
                                 be = __ballot(ok && key == prefix);
        const unsigned e_at = eq + __popcll(be & below);
        const unsigned at = gt + __popcll(bg & below) + min(e_at, left);
        if (ok && (key > prefix || (key == prefix && e_at < left))) kept[at] = i;
        gt += __popcll(bg);
        eq += __popcll(be);
    });
}

// Moves the kept keys of one (layer, sequence, KV head) to their new places,
// page by page.  In place one workgroup walks the pages in order: a page's
// sources lie at it or behind it, so only a page's own loads have to end
// before its stores begin.  Into another cache every page has a workgroup.
// A thread makes the 16 bytes of one lane of a K tile (a key's, moved whole) and
// of a V chunk: two dims and both key halves, a nibble each of the sixteen keys of
// its lane group, taken from the sixteen bytes that hold it.  Where a page's keys come
// from a few pages, as they do while little is dropped, those pages' values are
// staged in LDS (2304 keys of 256 heads to 2048: 61 us; 107 with a load a nibble
// from global memory).  In place, one page of a head after the other, a call of it takes
// 97 us for 63, and of 128 heads of 32768 keys to 1024 67 for 58.
constexpr int kMovePages = 3;
template <int HD>
__global__ __launch_bounds__(256) void k_kv4_move(Kv4Evict e, int per_row) {
    using P = Page<HD>;
    constexpr int NB = P::NB, VB = 32 * HD, SD = (128 * NB + 255) / 256;
    __shared__ unsigned s_i[kPageKeys], s_pg[kPageKeys], s_d[kPageKeys];
    __shared__ uint4_t s_v[kMovePages * VB / 16];
    const int t = threadIdx.x, lane = t & 63, wv = wave_id(), g = lane >> 4, r = lane & 15;
    const size_t rowi = e.row0 + blockIdx.x / per_row;
    const int b = (int)(rowi / e.n_kv % e.n_seqs);
    if (rowi < (size_t)e.n_seqs * e.n_kv && rowi % e.n_kv == 0 && blockIdx.x % per_row == 0 &&
        t == 0)
        e.lens_out[b] = min(min(e.lens[b], e.src_max), e.keep);
    const bool in_place = e.src == e.dst;
    const uint8_t *src = e.src + rowi * e.src_pages * P::kBytes;
    uint8_t *dst = e.dst + rowi * e.dst_pages * P::kBytes;
    const float *w = e.w + rowi * e.src_max;
    float *wo = e.w_out + rowi * e.dst_max;
    const uint32_t *kept = e.kept + rowi * e.keep;
    const unsigned n_pg = (e.keep + kPageKeys - 1) / kPageKeys;
    for (unsigned pg = blockIdx.x % per_row; pg < n_pg; pg += per_row) {
        const unsigned key0 = pg * kPageKeys;
        __syncthreads();  // the previous page's indexes are read, its stores issued
        if (t < kPageKeys) {
            const unsigned i = key0 + t < e.keep ? kept[key0 + t] : MRI_NO_TOKEN;
            int sg, sh, sj;
            P::v_place(i % kPageKeys, &sg, &sh, &sj);
            s_i[t] = i;
            s_pg[t] = i / kPageKeys;
            s_d[t] = sg * 256 | sh << 5 | 4 * nibble_of(sj);  // lane group's bytes, half, shift
        }
        __syncthreads();
        if (s_i[0] == MRI_NO_TOKEN) return;  // (the kept ones come first)
        if (in_place && s_i[kPageKeys - 1] == key0 + kPageKeys - 1) continue;  // all in place
        const int n = __popcll(__ballot(s_i[lane] != MRI_NO_TOKEN));  // keys of the page
        const unsigned from = s_pg[0], n_src = s_pg[n - 1] - from + 1;
        const bool staged = n_src <= kMovePages;
        if (staged) {
            for (unsigned x = t; x < n_src * (VB / 16); x += 256)
                s_v[x] = *reinterpret_cast<const uint4_t *>(
                    src + (size_t)(from + x / (VB / 16)) * P::kBytes + P::kV + x % (VB / 16) * 16);
        }
        // K: 16 (or 8) bytes of key 16 wv + r
        unsigned kq[NB];
        const int kkey = 16 * wv + r;
        if (kkey < n) {
            const unsigned *p = reinterpret_cast<const unsigned *>(
                src + (size_t)s_pg[kkey] * P::kBytes +
                P::k_dword(s_i[kkey] % kPageKeys, g, 0));
#pragma unroll
            for (int u = 0; u < NB; ++u) kq[u] = p[u];
        }
        unsigned sc[SD];
#pragma unroll
        for (int u = 0; u < SD; ++u) {
            const int x = t + 256 * u, which = x >= 64 * NB, rest = x % (64 * NB);
            sc[u] = 0;
            if (x < 128 * NB && rest / NB < n)
                sc[u] = *reinterpret_cast<const uint16_t *>(
                    src + (size_t)s_pg[rest / NB] * P::kBytes + (which ? P::kVs : P::kKs) +
                    P::scale(s_i[rest / NB] % kPageKeys, rest % NB));
        }
        float wt = 0.0f;
        if (t < n) wt = w[s_i[t]];
        __syncthreads();  // the staged values
        // V: chunk wv
        unsigned vq[4] = {0, 0, 0, 0}, vm[2] = {0, 0};
        uint8_t *pb = dst + (size_t)pg * P::kBytes;
        uint4_t *vto = reinterpret_cast<uint4_t *>(pb + P::kV + wv * 1024 + lane * 16);
        uint4_t old = {0, 0, 0, 0};
        auto gather = [&](auto st) __attribute__((always_inline)) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint4_t x[8];
                unsigned d[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int key = P::v_key(g, h, j), k0 = min(key, n - 1);
                    d[j] = s_d[k0];
                    const unsigned at = (d[j] & ~63u) + wv * 1024 + r * 16;
                    if constexpr (decltype(st)::value)
                        x[j] = s_v[(s_pg[k0] - from) * (VB / 16) + at / 16];
                    else
                        x[j] = *reinterpret_cast<const uint4_t *>(
                            src + (size_t)s_pg[k0] * P::kBytes + P::kV + at);
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int sh = d[j] & 31, to = 4 * nibble_of(j);
                    const bool hi = d[j] & 32, in = P::v_key(g, h, j) < n;
                    vq[h] |= ((hi ? x[j].y : x[j].x) >> sh & 0xfu) << to;
                    vq[2 + h] |= ((hi ? x[j].w : x[j].z) >> sh & 0xfu) << to;
                    vm[h] |= (in ? 0xfu : 0u) << to;
                }
            }
        };
        if (wv < NB) {
            if (staged) gather(std::true_type{});
            else gather(std::false_type{});
            if (n < kPageKeys) old = *vto;
        }
        __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this thread's loads have ended
        __syncthreads();
        if (kkey < n) {
            unsigned *p = reinterpret_cast<unsigned *>(pb + P::k_dword(kkey, g, 0));
#pragma unroll
            for (int u = 0; u < NB; ++u) p[u] = kq[u];
        }
        if (wv < NB && (vm[0] | vm[1]))
            *vto = uint4_t{(old.x & ~vm[0]) | (vq[0] & vm[0]), (old.y & ~vm[1]) | (vq[1] & vm[1]),
                           (old.z & ~vm[0]) | (vq[2] & vm[0]), (old.w & ~vm[1]) | (vq[3] & vm[1])};
#pragma unroll
        for (int u = 0; u < SD; ++u) {
            const int x = t + 256 * u, which = x >= 64 * NB, rest = x % (64 * NB);
            if (x < 128 * NB && rest / NB < n)
                *reinterpret_cast<uint16_t *>(pb + (which ? P::kVs : P::kKs) +
                                              P::scale(rest / NB, rest % NB)) = (uint16_t)sc[u];
        }
        if (t < n) wo[key0 + t] = wt;
    }
}

inline bool al16(const void *p) { return ((uintptr_t)p & 15) == 0; }

// Workgroups of one launch (512 threads each at most; a launch takes fewer than 2^32).
// Calls of more run in parts.
constexpr size_t kMostWgs = 1u << 22;

template <class F>
void by_head(size_t hd, F &&f) {
    if (hd == 64) f(std::integral_constant<int, 64>{});
    else f(std::integral_constant<int, 128>{});
}

// Pages that the call's rows can touch.
inline size_t pages_touched(const Kv4Rows &a) {
    const size_t p = (size_t)a.start + a.row0;
    if (!a.pos) return (p + a.rows - 1) / kPageKeys - p / kPageKeys + 1;
    return ((size_t)a.rows + kPageKeys - 2) / kPageKeys + 1;
}
// Sequences b .. b + n - 1 of the call's.
inline Kv4Rows some_seqs(const Kv4Rows &a, size_t b, size_t n) {
    Kv4Rows c = a;
    c.first_seq += (int)b;
    c.n_seqs = (int)std::min<size_t>(n, a.n_seqs - b);
    if (c.pos) c.pos += b;
    if (c.count) c.count += b;
    return c;
}
// Append and read, a workgroup a page, in launches of at most kMostWgs: f(rows, pages
// of a sequence, first layer, layers, first sequence) for parts of the rows (where one
// sequence's pages are too many), the sequences, then the layers.
template <class F>
mri_status by_pages(const Kv4Rows &a, size_t n_layers, F &&f) {
    const size_t most = kMostWgs / a.n_kv;  // (n_kv <= 2^20: four pages or more)
    const size_t rows = pages_touched(a) <= most ? a.rows : (most - 2) * kPageKeys;
    for (size_t i = 0; i < a.rows; i += rows) {
        Kv4Rows r = a;
        r.row0 = (unsigned)i;
        r.rows = (unsigned)std::min<size_t>(rows, a.rows - i);
        const size_t n_pg = pages_touched(r);
        const size_t seqs = std::min<size_t>(a.n_seqs, kMostWgs / (n_pg * a.n_kv));
        const size_t layers =
            seqs < (size_t)a.n_seqs ? 1 : kMostWgs / (n_pg * a.n_kv * a.n_seqs);
        for (size_t b = 0; b < (size_t)a.n_seqs; b += seqs)
            for (size_t l = 0; l < n_layers; l += layers)
                if (const mri_status st = f(some_seqs(r, b, seqs), n_pg, l,
                                            std::min(layers, n_layers - l), b))
                    return st;
    }
    return MRI_OK;
}

}  // namespace

mri_status launch_kv4_append(const Kv4Rows &a, size_t hd, const float *k, const float *v,
                             size_t stride, hipStream_t s) {
    if (!a.rows || !a.n_seqs) return MRI_OK;
    const bool v4 = stride % 4 == 0 && al16(k) && al16(v);
    return by_pages(a, 1, [&](const Kv4Rows &c, size_t n_pg, size_t, size_t, size_t b) {
        const dim3 grid((unsigned)(n_pg * c.n_kv * c.n_seqs));
        const size_t at = b * a.ld_rows * stride;
        by_head(hd, [&](auto h) {
            constexpr int HD = decltype(h)::value;
            if (v4)
                hipLaunchKernelGGL((k_kv4_append<HD, true>), grid, dim3(256), 0, s, c, k + at,
                                   v + at, stride, (int)n_pg);
            else
                hipLaunchKernelGGL((k_kv4_append<HD, false>), grid, dim3(256), 0, s, c, k + at,
                                   v + at, stride, (int)n_pg);
        });
        MRI_LAUNCHED("k_kv4_append");
        return MRI_OK;
    });
}

mri_status launch_kv4_read(const Kv4Rows &a, size_t hd, size_t n_layers, size_t layer_bytes,
                           float *k, float *v, size_t stride, hipStream_t s) {
    if (!a.rows || !a.n_seqs || !n_layers) return MRI_OK;
    const bool v4 = stride % 4 == 0 && al16(k) && al16(v);
    return by_pages(a, n_layers, [&](Kv4Rows c, size_t n_pg, size_t layer, size_t layers,
                                     size_t b) {
        const dim3 grid((unsigned)(n_pg * c.n_kv * c.n_seqs * layers));
        c.pages += layer * layer_bytes;
        const size_t at = (layer * a.n_seqs + b) * a.ld_rows * stride;
        by_head(hd, [&](auto h) {
            constexpr int HD = decltype(h)::value;
            if (v4)
                hipLaunchKernelGGL((k_kv4_read<HD, true>), grid, dim3(256), 0, s, c, layer_bytes,
                                   k + at, v + at, stride, (int)n_pg);
            else
                hipLaunchKernelGGL((k_kv4_read<HD, false>), grid, dim3(256), 0, s, c, layer_bytes,
                                   k + at, v + at, stride, (int)n_pg);
        });
        MRI_LAUNCHED("k_kv4_read");
        return MRI_OK;
    });
}

namespace {

// One chunk of rows: at most kKv4LseFloats (row, head) pairs when weights are
// asked for.
template <int HD>
mri_status attend_rows(const Kv4Rows &a, const float *q, size_t qs, size_t n_heads, float *out,
                       size_t os, float *weights, float *part, int *cnts, float *lse,
                       hipStream_t s) {
    const int groups = (int)(n_heads / a.n_kv);
    const size_t n_q = (size_t)a.rows * groups;
    const bool vec = qs % 4 == 0 && al16(q);
    float *z = weights ? lse : nullptr;
    const size_t cus = (size_t)std::max(device_cus(), 1);
    auto go = [&](auto few_) -> mri_status {
        constexpr bool FEW = decltype(few_)::value;
        constexpr int NQ = QTile<HD, FEW>::NQ;
        const size_t n_qt = (n_q + NQ - 1) / NQ, tiles = n_qt * a.n_kv;
        // A call with tiles for half of the CUs or less splits its keys.  A token of 32
        // heads over 8 at 4000 keys: head dim 128, 1 sequence 14 us against 30, 16
        // sequences 24 against 32, 24 sequences 31 against 32; head dim 64, 24 21
        // against 23, 48 31 against 34, 72 49 against 46.  (At 500 keys the join
        // costs a call 0.7 us: the positions may be the device's.  The rule goes by
        // the tiles alone: of 32768 keys 16 sequences take 115 us and 17, not split,
        // 205.)
        const size_t fill = std::min<size_t>(wgs_of(HD) * cus, kKv4PartTiles);
        if (tiles * a.n_seqs * 2 <= fill) {
            const size_t slots = fill / tiles;
            hipLaunchKernelGGL((k_kv4_attend<HD, FEW, true>), dim3((unsigned)(slots * tiles)),
                               dim3(waves_of(HD, true) * kWave), 0, s, a, q, qs, vec, groups,
                               (int)n_qt, (unsigned)slots, out, os, part, cnts, z);
        } else {
            hipLaunchKernelGGL((k_kv4_attend<HD, FEW, false>), dim3((unsigned)(tiles * a.n_seqs)),
                               dim3(waves_of(HD, false) * kWave), 0, s, a, q, qs, vec, groups,
                               (int)n_qt, 0u, out, os, part, cnts, z);
        }
        MRI_LAUNCHED("k_kv4_attend");
        return MRI_OK;
    };
    // Shared pages where they give every CU a workgroup.  32 heads of 128: 256 rows
    // (half of the CUs) 20 us against 17, 512 rows 28 against 35, 1024 47 against 78,
    // 1536 81 against 131; behind 4000 keys 256 rows 137 against 71, 512 145 against
    // 131, 1024 220 against 269.
    const size_t n_qg = (n_q + kPromptWaves * 16 - 1) / (kPromptWaves * 16);
    const size_t prompt_wgs = n_qg * a.n_kv * a.n_seqs;
    if (n_q > 32 && prompt_wgs >= cus) {
        hipLaunchKernelGGL((k_kv4_prompt<HD>), dim3((unsigned)prompt_wgs),
                           dim3(kPromptWaves * kWave), 0, s, a, q, qs, vec, groups, (int)n_qg, out,
                           os, z);
        MRI_LAUNCHED("k_kv4_prompt");
    } else {
        const mri_status st =
            n_q <= QTile<HD, true>::NQ ? go(std::true_type{}) : go(std::false_type{});
        if (st) return st;
    }
    if (weights) {
        const size_t n_pg =
            a.pos ? a.n_pages : (a.start + (size_t)a.row0 + a.rows - 1) / kPageKeys + 1;
        const size_t n_grp = (n_pg + kWtWaves - 1) / kWtWaves;
        const size_t groups_all = n_grp * a.n_kv * a.n_seqs;
        // parts of the queries: three workgroups a CU, four query tiles a part at least
        // (1999 rows of 32 heads of 128: 76 us; two a CU 87, four 78, eight 90).  With
        // positions on the device both go by the cache's length: a call of 500 rows of
        // 32 heads over 8 takes 40 us in a cache of 512 positions, 55 in one of 4096, 165
        // in one of 32768 (41 in each where the host gives the position); 16 x 5 rows at
        // 4000 keys 37 in a cache of 4005, 38 in one of 32768, 72 in one of 262144.
        size_t parts = 3 * cus / groups_all;
        parts = std::min(parts, ((n_q + 15) / 16 + kWtWaves - 1) / kWtWaves);
        parts = std::max<size_t>(1, std::min<size_t>(parts, 16));
        if (groups_all > kKv4PartTiles ||
            groups_all * parts * kWtWaves * kPageKeys > kv4_part_floats(HD))
            parts = 1;
        // (positions on the device: the pages are those of the longest possible
        // sequence, so many sequences of a long cache take more than one launch; one
        // sequence's groups of 256 threads fit one: 288 GB hold fewer than 2^24 groups)
        const size_t seqs = std::min<size_t>(
            a.n_seqs, std::max<size_t>(1, kMostWgs / (n_grp * a.n_kv * parts)));
        for (size_t b = 0; b < (size_t)a.n_seqs; b += seqs) {
            const Kv4Rows c = some_seqs(a, b, seqs);
            hipLaunchKernelGGL((k_kv4_weights<HD>),
                               dim3((unsigned)(n_grp * c.n_kv * c.n_seqs * parts)),
                               dim3(kWtWaves * kWave), 0, s, c, q + b * a.ld_rows * qs, qs, vec,
                               groups, (int)n_grp, (int)parts, lse + b * a.rows * n_heads, weights,
                               part, cnts);
            MRI_LAUNCHED("k_kv4_weights");
        }
    }
    return MRI_OK;
}

}  // namespace

mri_status launch_kv4_attend(const Kv4Rows &a, size_t hd, const float *q, size_t q_stride,
                             size_t n_heads, float *out, size_t out_stride, float *weights,
                             float *part, int *cnts, float *lse, hipStream_t s) {
    if (!a.rows || !a.n_seqs || !n_heads) return MRI_OK;
    mri_status st = MRI_OK;
    auto go = [&](const Kv4Rows &c, const float *cq, float *co) {
        by_head(hd, [&](auto h) {
            constexpr int HD = decltype(h)::value;
            st = attend_rows<HD>(c, cq, q_stride, n_heads, co, out_stride, weights, part, cnts, lse,
                                 s);
        });
    };
    // as many rows of a sequence, and sequences, as a launch takes in tiles of 16
    // queries; with weights, as their log-sum-exps fit
    const size_t groups = n_heads / a.n_kv;
    size_t rows = std::max<size_t>(1, (kMostWgs / a.n_kv - 1) * 16 / groups);
    if (weights) rows = std::min(rows, std::max<size_t>(1, kKv4LseFloats / n_heads));
    rows = std::min<size_t>(rows, a.rows);
    size_t seqs = std::max<size_t>(1, kMostWgs / (a.n_kv * ((rows * groups + 15) / 16)));
    if (weights) seqs = std::min(seqs, std::max<size_t>(1, kKv4LseFloats / (a.rows * n_heads)));
    for (size_t b = 0; b < (size_t)a.n_seqs && !st; b += seqs)
        for (size_t i = 0; i < a.rows && !st; i += rows) {
            Kv4Rows c = some_seqs(a, b, seqs);
            c.row0 = (unsigned)i;
            c.rows = (unsigned)std::min<size_t>(rows, a.rows - i);
            go(c, q + b * a.ld_rows * q_stride, out + b * a.ld_rows * out_stride);
        }
    return st;
}

mri_status launch_kv4_evict(const Kv4Evict &call, size_t hd, hipStream_t s) {
    Kv4Evict e = call;
    const size_t all = (size_t)e.n_layers * e.n_seqs * e.n_kv;
    // every head's keys are chosen before any lengths are stored, maybe over the old
    constexpr size_t kMostSel = kMostWgs / 2;  // (1024 threads each)
    for (e.row0 = 0; e.row0 < all; e.row0 += kMostSel) {
        const dim3 grid((unsigned)std::min(kMostSel, all - e.row0));
        if (e.src_max <= kSelRegs * kSelThreads)
            hipLaunchKernelGGL(k_kv4_select<true>, grid, dim3(kSelThreads), 0, s, e);
        else
            hipLaunchKernelGGL(k_kv4_select<false>, grid, dim3(kSelThreads), 0, s, e);
        MRI_LAUNCHED("k_kv4_select");
    }
    const size_t n_pg = ((size_t)e.keep + kPageKeys - 1) / kPageKeys;
    for (e.row0 = 0; e.row0 < all; e.row0 += kMostWgs) {
        const size_t rows = std::min(kMostWgs, all - e.row0);
        const size_t per_row = e.src == e.dst ? 1 : std::min(n_pg, kMostWgs / rows);
        by_head(hd, [&](auto h) {
            constexpr int HD = decltype(h)::value;
            hipLaunchKernelGGL((k_kv4_move<HD>), dim3((unsigned)(rows * per_row)), dim3(256), 0, s,
                               e, (int)per_row);
        });
        MRI_LAUNCHED("k_kv4_move");
    }
    return MRI_OK;
}

}  // namespace mri
