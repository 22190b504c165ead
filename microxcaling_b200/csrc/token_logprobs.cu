// Log probabilities of given tokens from a row of logits, the row's entropy and its best alternatives; and the gradient
// (sm_100a).
//
// With x the logits times 1 / temperature, m = max x, z = sum exp(x - m), s = sum exp(x - m) (x - m):
//     log p_t = (x_t - m) - log z,     H = log z - s / z,     p_j = exp(x_j - lse),  lse = m + log z
//     dx_j = g_lp (1[j = t] - p_j) - g_H p_j (log p_j + H)  =  p_j (A + B log p_j) + g_lp 1[j = t],
//     A = -g_lp - g_H H,  B = -g_H
//
// Forward is one pass over the row: every thread keeps its own running m, z and s (rescaled when 16 bytes of the row bring a new
// maximum), joined at the end.  Both directions are bound by HBM, forward close to the issue rate of the
// exponentials as well.  -inf logits (barred tokens) have probability 0 and add 0 to s; a row of nothing else has log
// probability -inf, entropy 0 and gradient 0.  A NaN or +inf makes its row NaN.
//
// Alternatives: the maxima of 64 interleaved parts of the row come out of the same pass, and the k-th largest of them is a
// bound that at least k logits reach (k <= 32).  Only threads of parts that reach it read their logits again (from
// L2) and collect those at or above the bound, a few dozen as a rule, which are ranked by (value, lowest index first).  When
// too many reach it (equal logits), k rounds over the row find them one by one.
#include <algorithm>
#include <float.h>
#include <math.h>
#include "mxq_common.cuh"

namespace mxq {

constexpr int kParts = 64;                 // parts of a row whose maxima bound the k-th largest logit
constexpr int kMaxTop = 32;
constexpr int kCand = 1024;                // candidates that are ranked in shared memory

struct LogprobArgs {
    const void* x;
    const int64_t* tokens;                 // [rows] or null
    float* logprob;                        // [rows] (with tokens)
    float* entropy;                        // [rows] or null
    float* lse;                            // [rows] or null: kept for the gradient (+inf: no finite logit)
    float* top_logprob;                    // [rows, top]
    int64_t* top_token;
    int64_t rows, vocab, stride, ignore;
    float inv_t;
    int top;
};

template <int DT, int VEC>
__device__ __forceinline__ void load_logits(const typename Store<DT>::T* p, int64_t i, float (&v)[VEC]) {
    if constexpr (VEC == 1) {
        v[0] = Store<DT>::load(p[i]);
    } else {
        uint32_t b[VEC];
        VecIO<DT, 16>::load(p, i, b);
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[j] = __uint_as_float(b[j]);
    }
}

constexpr float kLog2e = 1.4426950408889634f;
// 2^x by the hardware's approximation (relative error about 2^-22, results below 2^-126 are 0)
__device__ __forceinline__ float exp2_approx(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// Larger key = larger logit, the lowest index first among equals (-0 = +0); a NaN is above everything.
__device__ __forceinline__ uint32_t value_key(float v) {
    const uint32_t u = __float_as_uint(v + 0.f);
    if (v != v) return 0xfffffffeu;                                 // so that no key has every bit set
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ unsigned long long full_key(float v, int64_t i) {
    return ((unsigned long long)value_key(v) << 32) | (0xffffffffu - (uint32_t)i);
}

template <int THREADS>
__device__ __forceinline__ unsigned long long cta_max(unsigned long long v, unsigned long long* red) {
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) { const unsigned long long o = __shfl_xor_sync(0xffffffffu, v, s); v = o > v ? o : v; }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = red[0];
    for (int w = 1; w < THREADS / 32; ++w) v = red[w] > v ? red[w] : v;
    return v;
}

template <int DT, int VEC, int THREADS, bool ENT>
__global__ void __launch_bounds__(THREADS) token_logprobs_kernel(const LogprobArgs g) {
    using T = typename Store<DT>::T;
    __shared__ float red_m[THREADS / 32], red_z[THREADS / 32], red_s[THREADS / 32];
    __shared__ float part_max[kParts];
    __shared__ unsigned long long cand[kCand];
    __shared__ unsigned long long red_k[THREADS / 32];
    __shared__ float bound;
    __shared__ int n_cand;
    const int64_t row = blockIdx.x;
    const T* x = reinterpret_cast<const T*>(g.x) + row * g.stride;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    // raw: largest logit of this thread, a finite number below every logit that counts until one is seen
    float raw = -FLT_MAX, m = -FLT_MAX, z = 0.f, s = 0.f;
    bool nan = false;
    for (int64_t c = (int64_t)threadIdx.x * VEC; c < g.vocab; c += THREADS * VEC) {
        float v[VEC];
        load_logits<DT, VEC>(x, c, v);
        float best = v[0];
#pragma unroll
        for (int j = 1; j < VEC; ++j) best = fmaxf(best, v[j]);
        raw = fmaxf(raw, best);
        if (best * g.inv_t > m) {
            const float up = best * g.inv_t, d = m - up, f = exp2_approx(d * kLog2e);
            if (ENT) s = f > 0.f ? (s + z * d) * f : 0.f;
            z *= f;
            m = up;
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const float t = __fmaf_rn(v[j], g.inv_t, -m), e = exp2_approx(t * kLog2e);
            z += e;
            if (ENT) s = __fmaf_rn(e, fmaxf(t, -1e4f), s);        // e is 0 there, and -inf * 0 is not
            if (g.top) nan |= v[j] != v[j];
        }
    }
    // join: over the warp, then over the warps
    float mm = m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, o));
    {
        const float d = m - mm, f = exp2_approx(d * kLog2e);
        if (ENT) s = f > 0.f ? (s + z * d) * f : 0.f;
        z *= f;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            z += __shfl_xor_sync(0xffffffffu, z, o);
            if (ENT) s += __shfl_xor_sync(0xffffffffu, s, o);
        }
        if (lane == 0) { red_m[warp] = mm; red_z[warp] = z; if (ENT) red_s[warp] = s; }
    }
    if (g.top) {
        constexpr int W = THREADS / kParts;                        // threads of a part
        float pm = nan ? INFINITY : raw;
#pragma unroll
        for (int o = W / 2; o > 0; o >>= 1) pm = fmaxf(pm, __shfl_xor_sync(0xffffffffu, pm, o));
        if (threadIdx.x % W == 0) part_max[threadIdx.x / W] = pm;
        if (threadIdx.x == 0) n_cand = 0;
    }
    __syncthreads();
    mm = red_m[0];
#pragma unroll
    for (int w = 1; w < THREADS / 32; ++w) mm = fmaxf(mm, red_m[w]);
    z = s = 0.f;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
        const float d = red_m[w] - mm, f = exp2_approx(d * kLog2e);
        if (ENT && f > 0.f) s += (red_s[w] + red_z[w] * d) * f;
        z += red_z[w] * f;
    }
    const bool empty = z == 0.f;                                    // no logit above -inf
    const float log_z = logf(z);
    if (threadIdx.x == 0) {
        if (g.lse) g.lse[row] = empty ? INFINITY : mm + log_z;
        if (ENT) g.entropy[row] = empty ? 0.f : log_z - s / z;
        if (g.tokens) {
            const int64_t t = g.tokens[row];
            float lp;
            if (t == g.ignore) lp = 0.f;
            else if (t < 0 || t >= g.vocab) lp = NAN;
            else lp = empty ? -INFINITY : __fmaf_rn(Store<DT>::load(x[t]), g.inv_t, -mm) - log_z;
            g.logprob[row] = lp;
        }
    }
    if (!g.top) return;

    if (threadIdx.x < kParts) {
        const float mine = part_max[threadIdx.x];
        int rank = 0;
#pragma unroll
        for (int j = 0; j < kParts; ++j) rank += part_max[j] > mine || (part_max[j] == mine && j < (int)threadIdx.x);
        if (rank == g.top - 1) bound = mine;
    }
    __syncthreads();
    if (part_max[threadIdx.x / (THREADS / kParts)] >= bound) {
        for (int64_t c = (int64_t)threadIdx.x * VEC; c < g.vocab; c += THREADS * VEC) {
            float v[VEC];
            load_logits<DT, VEC>(x, c, v);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                if (!(v[j] < bound) && v[j] != -INFINITY) {
                    const int at = atomicAdd(&n_cand, 1);
                    if (at < kCand) cand[at] = full_key(v[j], c + j);
                }
            }
        }
    }
    __syncthreads();
    const int n = n_cand;
    auto write = [&](int rank, unsigned long long key) {
        const int64_t i = 0xffffffffu - (uint32_t)key;
        g.top_token[row * g.top + rank] = i;
        g.top_logprob[row * g.top + rank] = empty ? -INFINITY : __fmaf_rn(Store<DT>::load(x[i]), g.inv_t, -mm) - log_z;
    };
    if (n >= g.top && n <= kCand) {
        for (int i = threadIdx.x; i < n; i += THREADS) {
            const unsigned long long key = cand[i];
            int rank = 0;
            for (int j = 0; j < n && rank < g.top; ++j) rank += cand[j] > key;
            if (rank < g.top) write(rank, key);
        }
    } else {
        unsigned long long last = ~0ull;                            // above every key: an index is below 2^32 - 1
        for (int r = 0; r < g.top; ++r) {
            unsigned long long best = 0;
            for (int64_t c = (int64_t)threadIdx.x * VEC; c < g.vocab; c += THREADS * VEC) {
                float v[VEC];
                load_logits<DT, VEC>(x, c, v);
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const unsigned long long key = full_key(v[j], c + j);
                    if (key < last && key > best) best = key;
                }
            }
            last = cta_max<THREADS>(best, red_k);
            if (threadIdx.x == 0) write(r, last);
        }
    }
}

struct LogprobGradArgs {
    const void* x;
    const int64_t* tokens;
    const float* lse;
    const float* entropy;                  // [rows], read where g_h is given
    const float* g_lp;                     // [rows] or null
    const float* g_h;                      // [rows] or null
    void* dx;                              // [rows, vocab]
    int64_t rows, vocab, stride, ignore, chunks;
    float inv_t;
};

constexpr int kGradThreads = 256;
constexpr int kGradSteps = 8;              // vectors a thread

template <int DT, int VEC, bool ENT>
__global__ void __launch_bounds__(kGradThreads) token_logprobs_grad_kernel(const LogprobGradArgs g) {
    using T = typename Store<DT>::T;
    const int64_t row = blockIdx.x / g.chunks, first = (blockIdx.x % g.chunks) * (kGradThreads * VEC * kGradSteps);
    const T* x = reinterpret_cast<const T*>(g.x) + row * g.stride;
    T* dx = reinterpret_cast<T*>(g.dx) + row * g.vocab;
    const float lse = g.lse[row], gh = ENT ? g.g_h[row] : 0.f;
    const int64_t t = g.tokens ? g.tokens[row] : g.ignore;
    float glp = g.g_lp && t != g.ignore ? g.g_lp[row] : 0.f;
    if (t != g.ignore && (t < 0 || t >= g.vocab) && g.g_lp) glp = NAN;      // as the log probability is
    const float A = -(glp + (ENT ? gh * g.entropy[row] : 0.f)), B = -gh;
    const bool empty = lse == INFINITY;
#pragma unroll
    for (int i = 0; i < kGradSteps; ++i) {
        const int64_t c = first + (int64_t)(i * kGradThreads + threadIdx.x) * VEC;
        if (c >= g.vocab) break;
        float v[VEC];
        load_logits<DT, VEC>(x, c, v);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const float lp = __fmaf_rn(v[j], g.inv_t, -lse), p = exp2_approx(lp * kLog2e);
            float d = ENT ? p * __fmaf_rn(B, fmaxf(lp, -1e4f), A) : p * A;  // p is 0 where lp is below
            if (c + j == t) d += glp;
            v[j] = empty ? 0.f : d * g.inv_t;
        }
        if constexpr (VEC == 1) {
            dx[c] = Store<DT>::make(v[0]);
        } else if constexpr (DT == DT_F32) {
            *reinterpret_cast<float4*>(dx + c) = make_float4(v[0], v[1], v[2], v[3]);
        } else {
            T o[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) o[j] = Store<DT>::make(v[j]);
            *reinterpret_cast<uint4*>(dx + c) = *reinterpret_cast<const uint4*>(o);
        }
    }
}

template <int DT, int VEC, int THREADS>
static int launch_logprobs(const LogprobArgs& g, cudaStream_t st) {
    if (g.entropy) token_logprobs_kernel<DT, VEC, THREADS, true><<<(int)g.rows, THREADS, 0, st>>>(g);
    else token_logprobs_kernel<DT, VEC, THREADS, false><<<(int)g.rows, THREADS, 0, st>>>(g);
    return check_launch();
}
template <int DT>
static int dispatch_logprobs(const LogprobArgs& g, cudaStream_t st) {
    constexpr int V = DT == DT_F32 ? 4 : 8;
    const bool vec = g.vocab % V == 0 && aligned16(g.x) && (g.stride * (16 / V)) % 16 == 0;
    if (g.vocab <= 8192) return vec ? launch_logprobs<DT, V, 256>(g, st) : launch_logprobs<DT, 1, 256>(g, st);
    return vec ? launch_logprobs<DT, V, 1024>(g, st) : launch_logprobs<DT, 1, 1024>(g, st);
}

template <int DT, int VEC>
static int launch_logprobs_grad(LogprobGradArgs g, cudaStream_t st) {
    const int64_t per = kGradThreads * VEC * kGradSteps;
    g.chunks = (g.vocab + per - 1) / per;
    if (g.rows * g.chunks > 0x7fffffff) return MXQ_ERR_TOO_LARGE;
    const int grid = (int)(g.rows * g.chunks);
    if (g.g_h) token_logprobs_grad_kernel<DT, VEC, true><<<grid, kGradThreads, 0, st>>>(g);
    else token_logprobs_grad_kernel<DT, VEC, false><<<grid, kGradThreads, 0, st>>>(g);
    return check_launch();
}
template <int DT>
static int dispatch_logprobs_grad(const LogprobGradArgs& g, cudaStream_t st) {
    constexpr int V = DT == DT_F32 ? 4 : 8;
    const bool vec = g.vocab % V == 0 && aligned16(g.x) && aligned16(g.dx) && (g.stride * (16 / V)) % 16 == 0;
    return vec ? launch_logprobs_grad<DT, V>(g, st) : launch_logprobs_grad<DT, 1>(g, st);
}

}  // namespace mxq

extern "C" int mxq_token_logprobs(const void* logits, int dtype, int64_t stride, const int64_t* tokens, int64_t ignore_index,
                                  float inv_temperature, float* logprobs, float* entropy, float* lse, int top, float* top_logprobs,
                                  int64_t* top_tokens, int64_t rows, int64_t vocab, void* stream) {
    using namespace mxq;
    if (rows < 0 || vocab <= 0 || dtype < 0 || dtype > 2 || top < 0 || top > vocab || !(inv_temperature > 0.f)) return MXQ_ERR_BAD_ARG;
    if (top > kMaxTop || vocab > 0x7fffffff || rows > 0x7fffffff) return MXQ_ERR_TOO_LARGE;
    if (rows == 0) return MXQ_OK;
    if (!logits || (rows > 1 && stride < vocab) || (tokens && !logprobs) || (top && (!top_logprobs || !top_tokens))) return MXQ_ERR_BAD_ARG;
    LogprobArgs g = {logits, tokens, logprobs, entropy, lse, top_logprobs, top_tokens, rows, vocab, stride, ignore_index, inv_temperature, top};
    cudaStream_t st = (cudaStream_t)stream;
    if (dtype == MXQ_F32) return dispatch_logprobs<DT_F32>(g, st);
    if (dtype == MXQ_F16) return dispatch_logprobs<DT_F16>(g, st);
    return dispatch_logprobs<DT_BF16>(g, st);
}

extern "C" int mxq_token_logprobs_grad(const void* logits, int dtype, int64_t stride, const int64_t* tokens, int64_t ignore_index,
                                       float inv_temperature, const float* lse, const float* entropy, const float* g_logprobs,
                                       const float* g_entropy, void* grad, int64_t rows, int64_t vocab, void* stream) {
    using namespace mxq;
    if (rows < 0 || vocab <= 0 || dtype < 0 || dtype > 2 || !(inv_temperature > 0.f)) return MXQ_ERR_BAD_ARG;
    if (vocab > 0x7fffffff || rows > 0x7fffffff) return MXQ_ERR_TOO_LARGE;
    if (rows == 0) return MXQ_OK;
    if (!logits || !lse || !grad || (rows > 1 && stride < vocab) || (g_logprobs && !tokens) || (g_entropy && !entropy)) return MXQ_ERR_BAD_ARG;
    LogprobGradArgs g = {logits, tokens, lse, entropy, g_logprobs, g_entropy, grad, rows, vocab, stride, ignore_index, 0, inv_temperature};
    cudaStream_t st = (cudaStream_t)stream;
    if (dtype == MXQ_F32) return dispatch_logprobs_grad<DT_F32>(g, st);
    if (dtype == MXQ_F16) return dispatch_logprobs_grad<DT_F16>(g, st);
    return dispatch_logprobs_grad<DT_BF16>(g, st);
}
