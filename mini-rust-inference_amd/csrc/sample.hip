// sample.hip — probabilities of logit rows and the verification of drafted
// tokens against them.
#include <hip/hip_runtime.h>

#include <cfloat>

#include "kv4.hpp"

namespace mri {
namespace {

constexpr int kWave = 64;

// ---- softmax with a temperature ----------------------------------------------
// p_i = exp((x_i - max x) / T) / sum: one workgroup a row, which is read
// twice (the second time from cache) and written once.  Each thread keeps a
// running maximum and the sum of exponentials under it.
__device__ inline float exp_scaled(float d, float c) {
    return __builtin_amdgcn_exp2f(d * c);  // c = log2(e) / T
}

template <int NT>
__global__ __launch_bounds__(NT) void k_softmax(const float *x, size_t n, size_t xs, float c,
                                                float *out, size_t os) {
    __shared__ float s_m[NT / kWave], s_l[NT / kWave];
    const float *row = x + (size_t)blockIdx.x * xs;
    float *orow = out + (size_t)blockIdx.x * os;
    float m = -INFINITY, l = 0.0f;
    for (size_t i = threadIdx.x; i < n; i += NT) {
        const float v = row[i];
        if (v > m) {
            l = l * exp_scaled(m - v, c) + 1.0f;
            m = v;
        } else if (!(v == -INFINITY)) {
            l = l + exp_scaled(v - m, c);  // NaN stays in the sum
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const float m2 = __shfl_xor(m, o, kWave), l2 = __shfl_xor(l, o, kWave);
        const float mm = fmaxf(m, m2);
        l = (m == mm ? l : l * exp_scaled(m - mm, c)) + (m2 == mm ? l2 : l2 * exp_scaled(m2 - mm, c));
        m = mm;
    }
    if (threadIdx.x % kWave == 0) {
        s_m[threadIdx.x / kWave] = m;
        s_l[threadIdx.x / kWave] = l;
    }
    __syncthreads();
    m = s_m[0];
    for (int w = 1; w < NT / kWave; ++w) m = fmaxf(m, s_m[w]);
    l = 0.0f;
    for (int w = 0; w < NT / kWave; ++w)
        l = l + (s_m[w] == m ? s_l[w] : s_l[w] * exp_scaled(s_m[w] - m, c));
    const bool none = m == -INFINITY && l == 0.0f;  // every logit -inf
    const float inv = m == INFINITY ? NAN : 1.0f / l;
    for (size_t i = threadIdx.x; i < n; i += NT)
        orow[i] = none ? 0.0f : exp_scaled(row[i] - m, c) * inv;
}

// ---- verification of drafted tokens ----------------------------------------------
// One workgroup a sequence.  The acceptance tests are products of two floats
// in f64, which are exact.  The drawn token is found by halving: the waves sum
// contiguous sixteenths of a range (f64), the one in which the cumulative
// sum passes the target is the next range, down to one wave's width.
struct Residual {
    const float *p, *q;  // q null: nothing is taken away, or 1 at `hot`
    size_t hot;
    __device__ double operator()(size_t i) const {
        double r = (double)p[i];
        if (q) r = r - (double)q[i];
        else if (i == hot) r = r - 1.0;
        return r > 0.0 ? r : 0.0;  // (NaN: 0)
    }
};

constexpr int kVerWaves = 16;

__device__ inline double wave_sum_f64(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, kWave);
    return v;
}

// The sums of the sixteen parts of [lo, hi), `part` elements each, in s_sum.
__device__ inline void part_sums(const Residual &r, size_t lo, size_t hi, size_t part,
                                 double *s_sum) {
    const int lane = threadIdx.x % kWave, wv = threadIdx.x / kWave;
    const size_t a = min(lo + (size_t)wv * part, hi), b = min(a + part, hi);
    double s = 0.0;
    for (size_t i = a + lane; i < b; i += kWave) s += r(i);
    s = wave_sum_f64(s);
    __syncthreads();
    if (lane == 0) s_sum[wv] = s;
    __syncthreads();
}

__global__ __launch_bounds__(kVerWaves *kWave) void k_verify(
    const uint32_t *__restrict__ drafts, const float *__restrict__ dp,
    const float *__restrict__ tp, const float *__restrict__ us,
    const uint32_t *__restrict__ n_drafts, unsigned k, size_t n, uint32_t *__restrict__ tokens,
    uint32_t *__restrict__ accepted) {
    __shared__ double s_sum[kVerWaves];
    __shared__ unsigned s_first, s_tok;
    const size_t b = blockIdx.x;
    const unsigned count = n_drafts ? min(n_drafts[b], k) : k;
    const uint32_t *x = drafts + b * k;
    const float *u = us + b * (k + 1);
    if (threadIdx.x == 0) {
        s_first = count;
        s_tok = MRI_NO_TOKEN;
    }
    __syncthreads();
    for (unsigned i = threadIdx.x; i < count; i += kVerWaves * kWave) {
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
    auto part_of = [](size_t len) {
        return ((len + kVerWaves - 1) / kVerWaves + kWave - 1) / kWave * kWave;
    };
    size_t lo = 0, hi = n, part = part_of(n);
    auto total_of = [&]() {
        part_sums(r, lo, hi, part, s_sum);
        double t = 0.0;
        for (int w = 0; w < kVerWaves; ++w) t += s_sum[w];
        return t;
    };
    double total = total_of();
    if (a < count && !(total > 0.0)) {  // the draft covers the target: draw from the target
        r.q = nullptr;
        r.hot = n;
        total = total_of();
    }
    if (total > 0.0) {
        const double goal = (double)u[k] * total;
        double base = 0.0;
        for (;;) {
            // the first part in which the sum passes the goal, else the last with mass
            int at = 0;
            double before = base, run = base;
            for (int w = 0; w < kVerWaves; ++w) {
                if (s_sum[w] > 0.0) {
                    at = w;
                    before = run;
                    run += s_sum[w];
                    if (run > goal) break;
                }
            }
            base = before;
            lo = lo + (size_t)at * part;
            hi = min(lo + part, hi);
            if (hi - lo <= kWave) break;
            part = part_of(hi - lo);
            part_sums(r, lo, hi, part, s_sum);
        }
        if (threadIdx.x < kWave) {
            const size_t i = lo + threadIdx.x;
            const double v = i < hi ? r(i) : 0.0;
            double c = v;
#pragma unroll
            for (int o = 1; o < kWave; o <<= 1) {
                const double y = __shfl_up(c, o, kWave);
                if ((int)threadIdx.x >= o) c += y;
            }
            const unsigned long long mass = __ballot(v > 0.0),
                                     over = __ballot(v > 0.0 && base + c > goal);
            const int lane = over ? __ffsll((long long)over) - 1 : 63 - __clzll((long long)mass);
            if (threadIdx.x == 0) s_tok = (unsigned)(lo + lane);
        }
    }
    __syncthreads();
    for (unsigned i = threadIdx.x; i <= k; i += kVerWaves * kWave)
        tokens[b * (k + 1) + i] = i < a ? x[i] : i == a ? s_tok : MRI_NO_TOKEN;
    if (threadIdx.x == 0) accepted[b] = a;
}

}  // namespace

mri_status launch_softmax(const float *x, size_t rows, size_t n, size_t x_stride,
                          float temperature, float *out, size_t out_stride, hipStream_t s) {
    if (!rows) return MRI_OK;
    const float c = (float)fmin(1.4426950408889634074 / (double)temperature, (double)FLT_MAX);
    hipLaunchKernelGGL(k_softmax<1024>, dim3((unsigned)rows), dim3(1024), 0, s, x, n, x_stride, c,
                       out, out_stride);
    MRI_LAUNCHED("k_softmax");
    return MRI_OK;
}

mri_status launch_verify(const uint32_t *drafts, const float *draft_probs,
                         const float *target_probs, const float *uniforms,
                         const uint32_t *n_drafts, size_t n_seqs, size_t k, size_t n,
                         uint32_t *tokens, uint32_t *accepted, hipStream_t s) {
    if (!n_seqs) return MRI_OK;
    hipLaunchKernelGGL(k_verify, dim3((unsigned)n_seqs), dim3(kVerWaves * kWave), 0, s, drafts,
                       draft_probs, target_probs, uniforms, n_drafts, (unsigned)k, n, tokens,
                       accepted);
    MRI_LAUNCHED("k_verify");
    return MRI_OK;
}

}  // namespace mri
