// sample.hip — probabilities of logit rows and the verification of drafted
// tokens against them.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cfloat>
#include <type_traits>

#include "kv4.hpp"

namespace mri {
namespace {

constexpr int kWave = 64;

// Four floats at any float's address (global loads and stores of four words need
// no more than a word's alignment).
typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));

// ---- softmax with a temperature ----------------------------------------------
// p_i = exp((x_i - max x) / T) / sum.  Bound by its reads and writes, and by the
// launch where they are few.
// A row of up to 32768 logits stays in the registers of one workgroup: read once,
// one exponential a value (HELD).  A longer one is cut into `parts` parts of `len`
// values (a multiple of four); 256 threads take a part's (max, sum of
// exponentials under it), sixteen values a thread at a time.  Few rows: a
// workgroup a part, then a second launch that joins a row's parts and writes; the
// values come from the device's cache then.  Else a workgroup of 1024 a row does
// the same steps, four parts at a time, to the same bits.
struct Temp {
    // exp((x - m) / T) = 2^((h x - h m) c): h is 1 / 2 where the temperature may bring
    // logits together whose difference passes the largest float (T >= 1), else 1
    float h, c;
    __device__ float exp_diff(float x, float m) const {
        return __builtin_amdgcn_exp2f(fmaf(x, h, -h * m) * c);
    }
};
struct MaxSum {
    float m, l;  // l = sum of exp of what is not -inf; NaN stays in it
};
__device__ inline MaxSum join(MaxSum a, MaxSum b, Temp c) {
    const float m = fmaxf(a.m, b.m);
    return MaxSum{m, (a.m == m ? a.l : a.l * c.exp_diff(a.m, m)) +
                         (b.m == m ? b.l : b.l * c.exp_diff(b.m, m))};
}

// HELD: V times four values a thread.
template <int V>
__global__ __launch_bounds__(1024) void k_softmax_held(const float *x, size_t n, size_t xs,
                                                       Temp c, float *out, size_t os) {
    __shared__ float s_m[16], s_l[16];
    const float *row = x + (size_t)blockIdx.x * xs;
    const int t = threadIdx.x, lane = t % kWave, wave = t / kWave;
    float v[4 * V];
#pragma unroll
    for (int u = 0; u < V; ++u) {
        const size_t i = 4 * ((size_t)u * 1024 + t);
        if (i + 4 <= n) {
            const float4u w = *reinterpret_cast<const float4u *>(row + i);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[4 * u + j] = w[j];
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) v[4 * u + j] = i + j < n ? row[i + j] : -INFINITY;
        }
    }
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < 4 * V; ++j) m = fmaxf(m, v[j]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, kWave));
    if (lane == 0) s_m[wave] = m;
    __syncthreads();
    m = s_m[lane % 16];
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, kWave));
    float l = 0.0f;
#pragma unroll
    for (int j = 0; j < 4 * V; ++j) {
        v[j] = v[j] == -INFINITY ? 0.0f : c.exp_diff(v[j], m);
        l = l + v[j];
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) l = l + __shfl_xor(l, o, kWave);
    if (lane == 0) s_l[wave] = l;
    __syncthreads();
    l = s_l[lane % 16];
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) l = l + __shfl_xor(l, o, kWave);
    // (every logit -inf: zeros)
    const float inv = m == INFINITY ? NAN : m == -INFINITY && l == 0.0f ? 0.0f : 1.0f / l;
    float *to = out + (size_t)blockIdx.x * os;
#pragma unroll
    for (int u = 0; u < V; ++u) {
        const size_t i = 4 * ((size_t)u * 1024 + t);
        if (i + 4 <= n) {
            float4u p;
#pragma unroll
            for (int j = 0; j < 4; ++j) p[j] = v[4 * u + j] * inv;
            *reinterpret_cast<float4u *>(to + i) = p;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (i + j < n) to[i + j] = v[4 * u + j] * inv;
        }
    }
}

constexpr int kPartThreads = 256;
// (max, sum) of x[lo, hi) over 256 threads, t of them this one; s_ms: four entries.
__device__ inline MaxSum part_stats(const float *x, size_t lo, size_t hi, int t, Temp c,
                                    MaxSum *s_ms) {
    MaxSum a{-INFINITY, 0.0f};
    for (size_t i0 = lo; i0 < hi; i0 += 16 * kPartThreads) {
        float v[16];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const size_t i = i0 + 4 * ((size_t)u * kPartThreads + t);
            if (i + 4 <= hi) {
                const float4u w = *reinterpret_cast<const float4u *>(x + i);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[4 * u + j] = w[j];
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) v[4 * u + j] = i + j < hi ? x[i + j] : -INFINITY;
            }
        }
        float m = a.m;
#pragma unroll
        for (int j = 0; j < 16; ++j) m = fmaxf(m, v[j]);
        float l = a.m == m ? a.l : a.l * c.exp_diff(a.m, m);
#pragma unroll
        for (int j = 0; j < 16; ++j)
            l = l + (v[j] == -INFINITY ? 0.0f : c.exp_diff(v[j], m));
        a = MaxSum{m, l};
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1)
        a = join(a, MaxSum{__shfl_xor(a.m, o, kWave), __shfl_xor(a.l, o, kWave)}, c);
    if (t % kWave == 0) s_ms[t / kWave] = a;
    __syncthreads();
    a = join(join(s_ms[0], s_ms[1], c), join(s_ms[2], s_ms[3], c), c);
    __syncthreads();
    return a;
}

// A row's probabilities x[lo, hi) from its (max, sum), over n_t threads.
__device__ inline void write_probs(const float *x, size_t lo, size_t hi, int t, int n_t, Temp c,
                                   MaxSum a, float *out) {
    const bool none = a.m == -INFINITY && a.l == 0.0f;  // every logit -inf
    const float inv = a.m == INFINITY ? NAN : 1.0f / a.l;
    for (size_t i = lo + 4 * (size_t)t; i < hi; i += 4 * (size_t)n_t) {
        if (i + 4 <= hi) {
            const float4u w = *reinterpret_cast<const float4u *>(x + i);
            float4u p;
#pragma unroll
            for (int j = 0; j < 4; ++j) p[j] = none ? 0.0f : c.exp_diff(w[j], a.m) * inv;
            *reinterpret_cast<float4u *>(out + i) = p;
        } else {
            for (size_t j = i; j < hi; ++j)
                out[j] = none ? 0.0f : c.exp_diff(x[j], a.m) * inv;
        }
    }
}

constexpr int kMaxParts = 64;
constexpr size_t kSplitRows = 512;
static_assert(kSplitRows * kMaxParts * sizeof(MaxSum) <= kSoftmaxWsBytes, "parts' workspace");
__device__ inline MaxSum join_parts(const MaxSum *p, int parts, Temp c) {
    MaxSum a = p[0];
    for (int i = 1; i < parts; ++i) a = join(a, p[i], c);
    return a;
}

__global__ __launch_bounds__(1024) void k_softmax_row(const float *x, size_t n, size_t xs, Temp c,
                                                      size_t len, int parts, float *out,
                                                      size_t os) {
    __shared__ MaxSum s_ms[4][4], s_part[kMaxParts];
    const float *row = x + (size_t)blockIdx.x * xs;
    const int sub = threadIdx.x / kPartThreads, t = threadIdx.x % kPartThreads;
    for (int i0 = 0; i0 < parts; i0 += 4) {
        const int i = i0 + sub;
        const size_t lo = min(n, i * len), hi = min(n, lo + len);
        const MaxSum a = part_stats(row, lo, hi, t, c, s_ms[sub]);
        if (t == 0 && i < parts) s_part[i] = a;
    }
    __syncthreads();
    write_probs(row, 0, n, threadIdx.x, 1024, c, join_parts(s_part, parts, c),
                out + (size_t)blockIdx.x * os);
}

__global__ __launch_bounds__(kPartThreads) void k_softmax_stats(const float *__restrict__ x,
                                                                size_t n, size_t xs, Temp c,
                                                                size_t len, int parts,
                                                                MaxSum *__restrict__ ws) {
    __shared__ MaxSum s_ms[4];
    const size_t row = blockIdx.x / parts, lo = blockIdx.x % parts * len;
    const MaxSum a = part_stats(x + row * xs, lo, min(n, lo + len), threadIdx.x, c, s_ms);
    if (threadIdx.x == 0) ws[blockIdx.x] = a;
}

__global__ __launch_bounds__(kPartThreads) void k_softmax_write(const float *x, size_t n,
                                                                size_t xs, Temp c, size_t len,
                                                                int parts,
                                                                const MaxSum *__restrict__ ws,
                                                                float *out, size_t os) {
    __shared__ MaxSum s_part[kMaxParts];
    const size_t row = blockIdx.x / parts, lo = blockIdx.x % parts * len;
    if ((int)threadIdx.x < parts) s_part[threadIdx.x] = ws[row * parts + threadIdx.x];
    __syncthreads();
    write_probs(x + row * xs, lo, min(n, lo + len), threadIdx.x, kPartThreads, c,
                join_parts(s_part, parts, c), out + row * os);
}

// ---- verification of drafted tokens ----------------------------------------------
// One workgroup a sequence.  The acceptance tests are products of two floats
// in f64, which are exact.  The row that the token is drawn from is summed in f64 by
// chunks, a chunk a wave at a time, sixteen values a lane in flight; the chunk in
// which the cumulative sum passes the target is read again, a value a thread, until
// it is no longer than the workgroup.
// 4 drafts of 32000 tokens: 9 us, the latency of the loads in turn (ids, their
// probabilities, the row, the chunk).  64 x 7 of 100003: 16.4 us, what 64 CUs can
// read (3.1 TB/s); the next 1024 loaded ahead takes 18.6.
struct Residual {
    const float *p, *q;  // q null: nothing is taken away, or 1 at `hot`
    size_t hot;
    __device__ static double pos(double r) { return r > 0.0 ? r : 0.0; }  // (NaN: 0)
    __device__ double operator()(size_t i) const {
        double r = (double)p[i];
        if (q) r = r - (double)q[i];
        else if (i == hot) r = r - 1.0;
        return pos(r);
    }
};

constexpr int kVerWaves = 16, kVerThreads = kVerWaves * kWave, kVerChunks = 128;

// Another lane's value, as DPP control CTRL picks it in the rows ROWS; 0 elsewhere.
template <int CTRL, int ROWS>
__device__ inline double dpp_f64(double v) {
    const int2 x = __builtin_bit_cast(int2, v);
    return __builtin_bit_cast(
        double, int2{__builtin_amdgcn_update_dpp(0, x.x, CTRL, ROWS, 0xf, false),
                     __builtin_amdgcn_update_dpp(0, x.y, CTRL, ROWS, 0xf, false)});
}
__device__ inline double read_lane_f64(double v, int l) {
    const int2 x = __builtin_bit_cast(int2, v);
    return __builtin_bit_cast(
        double, int2{__builtin_amdgcn_readlane(x.x, l), __builtin_amdgcn_readlane(x.y, l)});
}
// Sums of the lanes up to each: in rows of 16, then over the rows before.  (Moves
// between lanes through LDS: 10.1 and 18.5 us a call for 8.9 and 17.4.)
__device__ inline double wave_scan_f64(double v) {
    v += dpp_f64<0x111, 0xf>(v);  // row_shr 1, 2, 4, 8
    v += dpp_f64<0x112, 0xf>(v);
    v += dpp_f64<0x114, 0xf>(v);
    v += dpp_f64<0x118, 0xf>(v);
    v += dpp_f64<0x142, 0xa>(v);  // lane 15 to row 1, 47 to row 3
    v += dpp_f64<0x143, 0xc>(v);  // lane 31 to rows 2 and 3
    return v;
}
__device__ inline double wave_sum_f64(double v) { return read_lane_f64(wave_scan_f64(v), 63); }
// The first lane at which base and the lanes' values so far exceed the goal, or the
// last one with a value; base becomes the sum before it.
__device__ inline int find_lane(double v, double goal, double *base) {
    const double c = wave_scan_f64(v);
    const unsigned long long mass = __ballot(v > 0.0),
                             over = __ballot(v > 0.0 && *base + c > goal);
    const int l = over ? __ffsll((long long)over) - 1 : mass ? 63 - __clzll((long long)mass) : 0;
    if (l > 0) *base += read_lane_f64(c, l - 1);
    return l;
}

// A lane's sixteen values of 1024, 4 at 4 (lane + 64 u).
struct VerBlock {
    float4u p[4], q[4];
    // zeros from hi on
    __device__ void load(const Residual &r, size_t i0, size_t hi, int lane) {
#pragma unroll
        for (int u = 0; u < 4; ++u) p[u] = q[u] = float4u{0.0f, 0.0f, 0.0f, 0.0f};
        load_row(p, r.p, i0, hi, lane);
        if (r.q) load_row(q, r.q, i0, hi, lane);
    }
    static __device__ void load_row(float4u (&v)[4], const float *x, size_t i0, size_t hi,
                                    int lane) {
        if (i0 + 1024 <= hi) {
#pragma unroll
            for (int u = 0; u < 4; ++u)
                v[u] = *reinterpret_cast<const float4u *>(x + i0 + 4 * (u * kWave + lane));
        } else {
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const size_t i = i0 + 4 * (u * kWave + lane) + j;
                    if (i < hi) v[u][j] = x[i];
                }
        }
    }
    __device__ double sum() const {
        double s = 0.0;
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                s += Residual::pos((double)p[u][j] - (double)q[u][j]);
        return s;
    }
    // Takes out the value that 1 is taken from, if it is the lane's: what is left of it.
    __device__ double take(size_t hot, int lane) {
        double s = 0.0;
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (4 * (u * kWave + lane) + j == (int)hot) {
                    s = Residual::pos((double)p[u][j] - 1.0);
                    p[u][j] = 0.0f;
                }
        return s;
    }
};

__global__ __launch_bounds__(kVerThreads) void k_verify(
    const uint32_t *__restrict__ drafts, const float *__restrict__ dp,
    const float *__restrict__ tp, const float *__restrict__ us,
    const uint32_t *__restrict__ n_drafts, unsigned k, size_t n, uint32_t *__restrict__ tokens,
    uint32_t *__restrict__ accepted) {
    __shared__ double s_sum[kVerChunks];
    __shared__ unsigned s_first, s_tok;
    const int lane = threadIdx.x % kWave, wv = threadIdx.x / kWave;
    const size_t b = blockIdx.x;
    const unsigned count = n_drafts ? min(n_drafts[b], k) : k;
    const uint32_t *x = drafts + b * k;
    const float *u = us + b * (k + 1);
    const double draw = (double)u[k];
    if (threadIdx.x == 0) {
        s_first = count;
        s_tok = MRI_NO_TOKEN;
    }
    __syncthreads();
    for (unsigned i = threadIdx.x; i < count; i += kVerThreads) {
        const size_t t = x[i];
        bool ok = t < n;
        if (ok) {
            const double q = dp ? (double)dp[(b * k + i) * n + t] : 1.0;
            ok = (double)u[i] * q < (double)tp[(b * (k + 1) + i) * n + t];
        }
        if (!ok) atomicMin(&s_first, i);
    }
    __syncthreads();
    const unsigned a = s_first;
    Residual r{tp + (b * (k + 1) + a) * n, nullptr, n};
    if (a < count) {
        if (dp) r.q = dp + (b * k + a) * n;
        else r.hot = x[a];
    }
    double goal = -1.0, base = 0.0;  // (below 0: the total is not known yet)
    size_t lo = 0, hi = n;
    for (;;) {
        // the sums of the chunks of [lo, hi), `len` values each (whole 1024s), zeros past them;
        const size_t len = ((hi - lo + kVerChunks - 1) / kVerChunks + 1023) / 1024 * 1024;
        __syncthreads();
        for (int c = wv; c < kVerChunks; c += kVerWaves) {
            const size_t l0 = min(lo + c * len, hi), l1 = min(l0 + len, hi);
            double s = 0.0;
            for (size_t i = l0; i < l1; i += 1024) {
                VerBlock cur;
                cur.load(r, i, hi, lane);
                if (r.hot - i < 1024) s += cur.take(r.hot - i, lane);
                s += cur.sum();
            }
            if (l0 < l1) s = wave_sum_f64(s);
            if (lane == 0) s_sum[c] = s;
        }
        __syncthreads();
        const double c0 = s_sum[2 * lane], c1 = s_sum[2 * lane + 1];
        if (goal < 0.0) {
            const double total = wave_sum_f64(c0 + c1);
            if (!(total > 0.0)) {
                if (!(a < count) || (!r.q && r.hot == n)) break;  // no mass
                r.q = nullptr;  // the draft covers the target: draw from the target
                r.hot = n;
                continue;
            }
            goal = draw * total;
        }
        const int l = find_lane(c0 + c1, goal, &base);
        const double f0 = read_lane_f64(c0, l), f1 = read_lane_f64(c1, l);
        const bool second = f1 > 0.0 && !(f0 > 0.0 && base + f0 > goal);
        if (second) base += f0;
        lo = lo + (size_t)(2 * l + second) * len;
        hi = min(lo + len, hi);
        if (hi - lo > kVerThreads) continue;
        // a value a thread: the wave that passes the goal, then its lane
        const size_t i = lo + threadIdx.x;
        const double v = i < hi ? r(i) : 0.0;
        const double w = wave_sum_f64(v);
        __syncthreads();
        if (lane == 0) s_sum[wv] = w;
        __syncthreads();
        const int at = find_lane(lane < kVerWaves ? s_sum[lane] : 0.0, goal, &base);
        if (wv == at) {
            const int l = find_lane(v, goal, &base);
            if (lane == 0) s_tok = (unsigned)(lo + wv * kWave + l);
        }
        break;
    }
    __syncthreads();
    for (unsigned i = threadIdx.x; i <= k; i += kVerThreads)
        tokens[b * (k + 1) + i] = i < a ? x[i] : i == a ? s_tok : MRI_NO_TOKEN;
    if (threadIdx.x == 0) accepted[b] = a;
}

}  // namespace

mri_status launch_softmax(const float *x, size_t rows, size_t n, size_t x_stride,
                          float temperature, float *out, size_t out_stride, hipStream_t s) {
    if (!rows) return MRI_OK;
    const float half = temperature >= 1.0f ? 0.5f : 1.0f;
    const Temp c{half, (float)fmin(1.4426950408889634074 / half / (double)temperature,
                                   (double)FLT_MAX)};
    // Held: 5 x 32000 5.8 us a call against 8.6 in parts (two launches) and 10 in row
    // form, 320 rows 24 against 27, 512 rows 31 against 41.  Twice as many values a
    // thread do not fit its registers beside the addresses: 50000 11 against 8.4.
    const auto held = [&](auto v) {
        hipLaunchKernelGGL(k_softmax_held<decltype(v)::value>, dim3((unsigned)rows), dim3(1024), 0,
                           s, x, n, x_stride, c, out, out_stride);
        MRI_LAUNCHED("k_softmax_held");
        return MRI_OK;
    };
    if (n <= 4096) return held(std::integral_constant<int, 1>());
    if (n <= 2 * 4096) return held(std::integral_constant<int, 2>());
    if (n <= 4 * 4096) return held(std::integral_constant<int, 4>());
    if (n <= 8 * 4096) return held(std::integral_constant<int, 8>());
    // parts of 4096 values at least, 64 of them at most
    const size_t len = round_up(std::max<size_t>((n + kMaxParts - 1) / kMaxParts, 4096), 4);
    const size_t parts = (n + len - 1) / len;
    // Rows in parts where whole rows leave CUs idle (100003 logits: 5 rows 9 us against
    // 28, 128 rows 33 against 44, 320 rows 76 against 89, 512 rows 125 against 126).
    // The parts' workspace is the stream's: a call that is being captured uses none,
    // so that graphs recorded on one stream may run side by side.
    if (rows < kSplitRows) {
        const StreamTurn turn(s);  // no other thread's parts between this call's launches
        hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
        void *ws = nullptr;
        if (hipStreamIsCapturing(s, &capture) != hipSuccess) {
            (void)hipGetLastError();
        } else if (capture == hipStreamCaptureStatusNone) {
            const mri_status st = softmax_ws_get(s, &ws);
            if (st) return st;
        }
        if (ws) {
            hipLaunchKernelGGL(k_softmax_stats, dim3((unsigned)(rows * parts)),
                               dim3(kPartThreads), 0, s, x, n, x_stride, c, len, (int)parts,
                               static_cast<MaxSum *>(ws));
            MRI_LAUNCHED("k_softmax_stats");
            hipLaunchKernelGGL(k_softmax_write, dim3((unsigned)(rows * parts)),
                               dim3(kPartThreads), 0, s, x, n, x_stride, c, len, (int)parts,
                               static_cast<const MaxSum *>(ws), out, out_stride);
            MRI_LAUNCHED("k_softmax_write");
            return MRI_OK;
        }
    }
    hipLaunchKernelGGL(k_softmax_row, dim3((unsigned)rows), dim3(1024), 0, s, x, n, x_stride, c,
                       len, (int)parts, out, out_stride);
    MRI_LAUNCHED("k_softmax_row");
    return MRI_OK;
}

mri_status launch_verify(const uint32_t *drafts, const float *draft_probs,
                         const float *target_probs, const float *uniforms,
                         const uint32_t *n_drafts, size_t n_seqs, size_t k, size_t n,
                         uint32_t *tokens, uint32_t *accepted, hipStream_t s) {
    if (!n_seqs) return MRI_OK;
    hipLaunchKernelGGL(k_verify, dim3((unsigned)n_seqs), dim3(kVerThreads), 0, s, drafts,
                       draft_probs, target_probs, uniforms, n_drafts, (unsigned)k, n, tokens,
                       accepted);
    MRI_LAUNCHED("k_verify");
    return MRI_OK;
}

}  // namespace mri
