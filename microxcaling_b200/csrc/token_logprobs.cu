// Log probabilities of given tokens from a row of logits, the row's entropy and its best alternatives; and the gradient
// (sm_100a).
//
// With x the logits times 1 / temperature, m = max x, z = sum exp(x - m), s = sum exp(x - m) (x - m):
//     log p_t = (x_t - m) - log z,     H = log z - s / z,     p_j = exp(x_j - lse),  lse = m + log z
//     dx_j = g_lp (1[j = t] - p_j) - g_H p_j (log p_j + H)  =  p_j (A + B log p_j) + g_lp 1[j = t],
//     A = -g_lp - g_H H,  B = -g_H
//
// Forward is one pass over the row: every thread keeps its own running m, z and s (rescaled when 16 bytes of the row bring a new
// maximum), joined at the end; in units of log 2, which is what the hardware's exponential takes.  Both directions are bound
// by HBM, forward close to the rate of the exponentials (16 a cycle and SM) as well.  -inf logits (barred tokens) have
// probability 0 and add 0 to s; a row of nothing else has log probability -inf, entropy 0 and gradient 0.  A NaN or +inf
// makes its row NaN.  The gradient gets m and log z apart, so that neither is rounded by the other.
//
// Alternatives: the maxima of 64 interleaved parts of the row come out of the same pass, and the k-th largest of them is a
// bound that at least k logits reach (k <= 32).  Only the parts that reach it, k of 64 as a rule, are read again (from L2), and
// what is at or above the bound, a few dozen values, is ranked by (value, lowest index first).  When too many reach it
// (equal logits) or too few are finite, and in rows with a NaN or +inf, k rounds over the row find them one by one.
#include <algorithm>
#include <float.h>
#include <math.h>
#include "mxq_common.cuh"
#include "sm100_ptx.cuh"

namespace mxq {

constexpr int kParts = 64;                 // parts of a row whose maxima bound the k-th largest logit
constexpr int kMaxTop = 32;
constexpr int kCand = 1024;                // candidates that are ranked in shared memory

struct LogprobArgs {
    const void* x;
    const int64_t* tokens;                 // [rows] or null
    float* logprob;                        // [rows] (with tokens)
    float* entropy;                        // [rows] or null
    float2* stats;                         // [rows] or null, for the gradient: largest logit, log2 of z (+inf: no finite logit)
    float* top_logprob;                    // [rows, top]
    int64_t* top_token;
    int64_t rows, vocab, stride, ignore;
    float inv_t;
    int top;
};

// A row as 16-byte vectors wherever it starts: `head` single values up to the first 16-byte border, whole vectors, the rest.
template <int DT>
struct Row {
    using T = typename Store<DT>::T;
    static constexpr int VEC = 16 / (int)sizeof(T);
    const T* p;
    int head, vecs, len;
    __device__ __forceinline__ Row(const T* row, int64_t n) : p(row), len((int)n) {
        head = min(len, (int)((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / (int)sizeof(T));
        vecs = (len - head) / VEC;
    }
    __device__ __forceinline__ int first(int i) const { return head + i * VEC; }      // column of vector i
    __device__ __forceinline__ uint4 raw(int i) const { return __ldg(reinterpret_cast<const uint4*>(p + first(i))); }
    // the head (which = 0) or the rest (1), filled up with -inf
    __device__ __forceinline__ int edge_first(int which) const { return which == 0 ? 0 : first(vecs); }
    __device__ __forceinline__ int edge_count(int which) const { return which == 0 ? head : len - first(vecs); }
    __device__ __forceinline__ void edge(int which, float (&v)[VEC]) const {
        const int from = edge_first(which), n = edge_count(which);
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[j] = j < n ? Store<DT>::load(p[from + j]) : -INFINITY;
    }
    static __device__ __forceinline__ void values(const uint4& q, float (&v)[VEC]) {
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (DT == DT_F32) {
                v[i] = __uint_as_float(w[i]);
            } else if constexpr (DT == DT_BF16) {
                v[2 * i] = __uint_as_float(w[i] << 16);
                v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            } else {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
                v[2 * i] = f.x;
                v[2 * i + 1] = f.y;
            }
        }
    }
};

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
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

// Running maximum, sum and entropy sum of one thread: m = max x, z = sum 2^((x - m) c), s = sum 2^((x - m) c) (x - m) c with
// c = log2(e) / temperature; two values to an instruction.  m starts at a finite number below every logit that counts.
template <bool ENT>
struct Running {
    float m = -FLT_MAX;
    uint64_t z = 0, s = 0;
    template <int N>
    __device__ __forceinline__ void add(const float (&v)[N], float c, float best) {
        if (best > m) {
            const float d = (m - best) * c, f = exp2_approx(d);
            const uint64_t f2 = ptx::pack2f(f, f);
            if (ENT) s = f > 0.f ? ptx::mul2(ptx::fma2_to(z, ptx::pack2f(d, d), s), f2) : 0;
            z = ptx::mul2(z, f2);
            m = best;
        }
        const uint64_t c2 = ptx::pack2f(c, c), m2 = ptx::pack2f(-m, -m);
#pragma unroll
        for (int j = 0; j < N; j += 2) {
            float t0, t1;
            ptx::unpack2f(ptx::mul2(ptx::add2(ptx::pack2f(v[j], v[j + 1]), m2), c2), t0, t1);
            const uint64_t e = ptx::pack2f(exp2_approx(t0), exp2_approx(t1));
            z = ptx::add2(z, e);
            if (ENT) ptx::fma2(s, e, ptx::pack2f(fmaxf(t0, -1e4f), fmaxf(t1, -1e4f)));   // e is 0 there, and 0 * -inf is not
        }
    }
};

template <int DT, int THREADS, bool ENT, bool TOP>
__global__ void __launch_bounds__(THREADS, 1536 / THREADS) token_logprobs_kernel(const LogprobArgs g) {
    constexpr int VEC = Row<DT>::VEC, U = 4;                       // vectors of a thread in flight
    __shared__ float red_m[THREADS / 32], red_z[THREADS / 32], red_s[THREADS / 32];
    __shared__ float part_max[kParts];
    __shared__ unsigned long long cand[kCand];
    __shared__ unsigned long long red_k[THREADS / 32];
    __shared__ float bound;
    __shared__ int n_cand, n_parts, parts[kParts];
    const int64_t row = blockIdx.x;
    const Row<DT> x(reinterpret_cast<const typename Store<DT>::T*>(g.x) + row * g.stride, g.vocab);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const float c = g.inv_t * kLog2e;

    Running<ENT> run;
    float raw = -FLT_MAX;                                          // largest logit of this thread
    auto take = [&](const float (&v)[VEC]) {
        float best = v[0];
#pragma unroll
        for (int j = 1; j < VEC; ++j) best = fmaxf(best, v[j]);
        raw = fmaxf(raw, best);
        run.add(v, c, best);
    };
    int i = tid;
    for (; i + (U - 1) * THREADS < x.vecs; i += U * THREADS) {
        uint4 q[U];
#pragma unroll
        for (int u = 0; u < U; ++u) q[u] = x.raw(i + u * THREADS);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float v[VEC];
            Row<DT>::values(q[u], v);
            take(v);
        }
    }
    for (; i < x.vecs; i += THREADS) {
        float v[VEC];
        Row<DT>::values(x.raw(i), v);
        take(v);
    }
    if (tid < 2 && x.edge_count(tid) > 0) {
        float v[VEC];
        x.edge(tid, v);
        take(v);
    }
    // join: over the warp, then over the warps
    float m = run.m, z, s, hi;
    ptx::unpack2f(run.z, z, hi);
    z += hi;
    ptx::unpack2f(run.s, s, hi);
    s += hi;
    float mm = m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, o));
    {
        const float d = (m - mm) * c, f = exp2_approx(d);
        if (ENT) s = f > 0.f ? (s + z * d) * f : 0.f;
        z *= f;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            z += __shfl_xor_sync(0xffffffffu, z, o);
            if (ENT) s += __shfl_xor_sync(0xffffffffu, s, o);
        }
        if (lane == 0) { red_m[warp] = mm; red_z[warp] = z; if (ENT) red_s[warp] = s; }
    }
    if constexpr (TOP) {
        constexpr int W = THREADS / kParts;                        // threads of a part
        float pm = raw;
#pragma unroll
        for (int o = W / 2; o > 0; o >>= 1) pm = fmaxf(pm, __shfl_xor_sync(0xffffffffu, pm, o));
        if (tid % W == 0) part_max[tid / W] = pm;
        if (tid == 0) n_cand = n_parts = 0;
    }
    __syncthreads();
    mm = red_m[0];
#pragma unroll
    for (int w = 1; w < THREADS / 32; ++w) mm = fmaxf(mm, red_m[w]);
    z = s = 0.f;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
        const float d = (red_m[w] - mm) * c, f = exp2_approx(d);
        if (ENT && f > 0.f) s += (red_s[w] + red_z[w] * d) * f;
        z += red_z[w] * f;
    }
    const bool empty = z == 0.f;                                    // no logit above -inf
    const float log_z = log2f(z);
    auto logprob = [&](float v) { return empty ? -INFINITY : kLn2 * ((v - mm) * c - log_z); };
    if (tid == 0) {
        if (g.stats) g.stats[row] = make_float2(mm, empty ? INFINITY : log_z);
        if (ENT) g.entropy[row] = empty ? 0.f : kLn2 * (log_z - s / z);
        if (g.tokens) {
            const int64_t t = g.tokens[row];
            g.logprob[row] = t == g.ignore ? 0.f : t < 0 || t >= g.vocab ? NAN : logprob(Store<DT>::load(x.p[t]));
        }
    }
    if constexpr (TOP) {
        if (tid < kParts) {
            const float mine = part_max[tid];
            int rank = 0;
#pragma unroll
            for (int j = 0; j < kParts; ++j) rank += part_max[j] > mine || (part_max[j] == mine && j < tid);
            if (rank == g.top - 1) bound = mine;
        }
        __syncthreads();
        // the parts that reach the bound, their vectors spread over all threads
        constexpr int W = THREADS / kParts;
        if (tid < kParts && part_max[tid] >= bound) parts[atomicAdd(&n_parts, 1)] = tid;
        __syncthreads();
        auto collect = [&](const float (&v)[VEC], int first) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                if (v[j] >= bound) {
                    const int at = atomicAdd(&n_cand, 1);
                    if (at < kCand) cand[at] = full_key(v[j], first + j);
                }
            }
        };
        const bool clean = z == z;                                      // a NaN or +inf: one by one, below
        if (clean) {
            const int np = n_parts, rounds = (x.vecs + THREADS - 1) / THREADS;
            for (int k = tid; k < np * W * rounds; k += THREADS) {
                const int slot = k / W, at = slot / np * THREADS + parts[slot % np] * W + k % W;
                if (at >= x.vecs) continue;
                float v[VEC];
                Row<DT>::values(x.raw(at), v);
                collect(v, x.first(at));
            }
            if (tid < 2 && x.edge_count(tid) > 0) {
                float v[VEC];
                x.edge(tid, v);
                collect(v, x.edge_first(tid));
            }
        }
        __syncthreads();
        const int n = n_cand;
        auto write = [&](int rank, unsigned long long key) {
            const int64_t k = 0xffffffffu - (uint32_t)key;
            g.top_token[row * g.top + rank] = k;
            g.top_logprob[row * g.top + rank] = logprob(Store<DT>::load(x.p[k]));
        };
        if (clean && n >= g.top && n <= kCand) {
            for (int k = tid; k < n; k += THREADS) {
                const unsigned long long key = cand[k];
                int rank = 0;
                for (int j = 0; j < n && rank < g.top; ++j) rank += cand[j] > key;
                if (rank < g.top) write(rank, key);
            }
        } else {
            unsigned long long last = ~0ull;                            // above every key
            for (int r = 0; r < g.top; ++r) {
                unsigned long long best = 0;
                auto look = [&](const float (&v)[VEC], int first, int count) {
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        const unsigned long long key = full_key(v[j], first + j);
                        if (j < count && key < last && key > best) best = key;
                    }
                };
                float v[VEC];
                for (int k = tid; k < x.vecs; k += THREADS) {
                    Row<DT>::values(x.raw(k), v);
                    look(v, x.first(k), VEC);
                }
                if (tid < 2 && x.edge_count(tid) > 0) {
                    x.edge(tid, v);
                    look(v, x.edge_first(tid), x.edge_count(tid));
                }
                last = cta_max<THREADS>(best, red_k);
                if (tid == 0) write(r, last);
            }
        }
    }
}

struct LogprobGradArgs {
    const void* x;
    const int64_t* tokens;
    const float2* stats;
    const float* entropy;                  // [rows], read where g_h is given
    const float* g_lp;                     // [rows] or null
    const float* g_h;                      // [rows] or null
    void* dx;                              // [rows, vocab]
    int64_t rows, vocab, stride, ignore, chunks;
    float inv_t;
};

constexpr int kGradThreads = 256;
constexpr int kGradSteps = 8;              // vectors a thread

// VECTORS: rows of x and dx meet 16-byte borders at the same columns
template <int DT, bool ENT, bool VECTORS>
__global__ void __launch_bounds__(kGradThreads) token_logprobs_grad_kernel(const LogprobGradArgs g) {
    using T = typename Store<DT>::T;
    constexpr int VEC = Row<DT>::VEC;
    const int64_t row = blockIdx.x / g.chunks, chunk = blockIdx.x % g.chunks;
    const Row<DT> x(reinterpret_cast<const T*>(g.x) + row * g.stride, g.vocab);
    T* dx = reinterpret_cast<T*>(g.dx) + row * g.vocab;
    const float2 st = g.stats[row];
    const bool empty = st.y == INFINITY;
    const float gh = ENT ? g.g_h[row] : 0.f, c = g.inv_t * kLog2e;
    const int64_t t = g.tokens ? g.tokens[row] : g.ignore;
    float glp = g.g_lp && t != g.ignore ? g.g_lp[row] : 0.f;
    if (t != g.ignore && (t < 0 || t >= g.vocab) && g.g_lp) glp = NAN;      // as the log probability is
    // p (A + B log p) with log p in units of log 2, everything times 1 / temperature
    const float A = -(glp + (ENT ? gh * g.entropy[row] : 0.f)) * g.inv_t, B = -gh * kLn2 * g.inv_t;
    auto gradient = [&](float v, int64_t col) {
        const float lp = (v - st.x) * c - st.y, p = exp2_approx(lp);
        float d = ENT ? p * __fmaf_rn(B, fmaxf(lp, -1e4f), A) : p * A;      // p is 0 where lp is below
        if (col == t) d += glp * g.inv_t;
        return empty ? 0.f : d;
    };
    const int64_t per = kGradThreads * kGradSteps;
    if constexpr (VECTORS) {
        for (int k = 0; k < kGradSteps; ++k) {
            const int64_t i = chunk * per + k * kGradThreads + threadIdx.x;
            if (i >= x.vecs) break;
            float v[VEC];
            Row<DT>::values(x.raw((int)i), v);
            const int first = x.first((int)i);
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[j] = gradient(v[j], first + j);
            if constexpr (DT == DT_F32) {
                *reinterpret_cast<float4*>(dx + first) = make_float4(v[0], v[1], v[2], v[3]);
            } else {
                T o[VEC];
#pragma unroll
                for (int j = 0; j < VEC; ++j) o[j] = Store<DT>::make(v[j]);
                *reinterpret_cast<uint4*>(dx + first) = *reinterpret_cast<const uint4*>(o);
            }
        }
        if (chunk == 0 && threadIdx.x < 2 * VEC) {                          // the values before and behind the whole vectors
            const int which = threadIdx.x / VEC, j = threadIdx.x % VEC, col = x.edge_first(which) + j;
            if (j < x.edge_count(which)) dx[col] = Store<DT>::make(gradient(Store<DT>::load(x.p[col]), col));
        }
    } else {
        for (int k = 0; k < kGradSteps * VEC; ++k) {
            const int64_t col = chunk * per * VEC + k * kGradThreads + threadIdx.x;
            if (col >= g.vocab) break;
            dx[col] = Store<DT>::make(gradient(Store<DT>::load(x.p[col]), col));
        }
    }
}

template <int DT, int THREADS>
static int launch_logprobs(const LogprobArgs& g, cudaStream_t st) {
    const int grid = (int)g.rows;
    if (g.entropy && g.top) token_logprobs_kernel<DT, THREADS, true, true><<<grid, THREADS, 0, st>>>(g);
    else if (g.entropy) token_logprobs_kernel<DT, THREADS, true, false><<<grid, THREADS, 0, st>>>(g);
    else if (g.top) token_logprobs_kernel<DT, THREADS, false, true><<<grid, THREADS, 0, st>>>(g);
    else token_logprobs_kernel<DT, THREADS, false, false><<<grid, THREADS, 0, st>>>(g);
    return check_launch();
}
template <int DT>
static int dispatch_logprobs(const LogprobArgs& g, cudaStream_t st) {
    // 512 threads a row let two rows share an SM, one working while the other's sums meet; few long rows get 1024 each
    const bool wide = g.rows <= sm_count() && g.vocab > 8192;
    if (g.vocab <= 8192) return launch_logprobs<DT, 256>(g, st);
    return wide ? launch_logprobs<DT, 1024>(g, st) : launch_logprobs<DT, 512>(g, st);
}

template <int DT>
static int dispatch_logprobs_grad(LogprobGradArgs g, cudaStream_t st) {
    constexpr int V = Row<DT>::VEC, ES = 16 / V;
    const int64_t per = kGradThreads * V * kGradSteps;
    g.chunks = (g.vocab + per - 1) / per;
    if (g.rows * g.chunks > 0x7fffffff) return MXQ_ERR_TOO_LARGE;
    const int grid = (int)(g.rows * g.chunks);
    const bool vec = ((reinterpret_cast<uintptr_t>(g.x) ^ reinterpret_cast<uintptr_t>(g.dx)) & 15) == 0 &&
                     (g.rows == 1 || (g.stride - g.vocab) * ES % 16 == 0);
#define MXQ_GRAD(ENT) (vec ? token_logprobs_grad_kernel<DT, ENT, true><<<grid, kGradThreads, 0, st>>>(g) \
                           : token_logprobs_grad_kernel<DT, ENT, false><<<grid, kGradThreads, 0, st>>>(g))
    if (g.g_h) MXQ_GRAD(true);
    else MXQ_GRAD(false);
#undef MXQ_GRAD
    return check_launch();
}

}  // namespace mxq

extern "C" int mxq_token_logprobs(const void* logits, int dtype, int64_t stride, const int64_t* tokens, int64_t ignore_index,
                                  float inv_temperature, float* logprobs, float* entropy, float* stats, int top, float* top_logprobs,
                                  int64_t* top_tokens, int64_t rows, int64_t vocab, void* stream) {
    using namespace mxq;
    if (rows < 0 || vocab <= 0 || dtype < 0 || dtype > 2 || top < 0 || top > vocab || !(inv_temperature > 0.f)) return MXQ_ERR_BAD_ARG;
    if (top > kMaxTop || vocab > 0x7fffffff || rows > 0x7fffffff) return MXQ_ERR_TOO_LARGE;
    if (rows == 0) return MXQ_OK;
    if (!logits || (rows > 1 && stride < vocab) || (tokens && !logprobs) || (top && (!top_logprobs || !top_tokens))) return MXQ_ERR_BAD_ARG;
    LogprobArgs g = {logits, tokens, logprobs, entropy, (float2*)stats, top_logprobs, top_tokens, rows, vocab, stride, ignore_index, inv_temperature, top};
    cudaStream_t st = (cudaStream_t)stream;
    if (dtype == MXQ_F32) return dispatch_logprobs<DT_F32>(g, st);
    if (dtype == MXQ_F16) return dispatch_logprobs<DT_F16>(g, st);
    return dispatch_logprobs<DT_BF16>(g, st);
}

extern "C" int mxq_token_logprobs_grad(const void* logits, int dtype, int64_t stride, const int64_t* tokens, int64_t ignore_index,
                                       float inv_temperature, const float* stats, const float* entropy, const float* g_logprobs,
                                       const float* g_entropy, void* grad, int64_t rows, int64_t vocab, void* stream) {
    using namespace mxq;
    if (rows < 0 || vocab <= 0 || dtype < 0 || dtype > 2 || !(inv_temperature > 0.f)) return MXQ_ERR_BAD_ARG;
    if (vocab > 0x7fffffff || rows > 0x7fffffff) return MXQ_ERR_TOO_LARGE;
    if (rows == 0) return MXQ_OK;
    if (!logits || !stats || !grad || (rows > 1 && stride < vocab) || (g_logprobs && !tokens) || (g_entropy && !entropy)) return MXQ_ERR_BAD_ARG;
    LogprobGradArgs g = {logits, tokens, (const float2*)stats, entropy, g_logprobs, g_entropy, grad, rows, vocab, stride, ignore_index, 0, inv_temperature};
    cudaStream_t st = (cudaStream_t)stream;
    if (dtype == MXQ_F32) return dispatch_logprobs_grad<DT_F32>(g, st);
    if (dtype == MXQ_F16) return dispatch_logprobs_grad<DT_F16>(g, st);
    return dispatch_logprobs_grad<DT_BF16>(g, st);
}
