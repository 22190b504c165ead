// Layer normalisation over the last dimension, forward and backward, each value rounded once (sm_100a).
//
//     y = (x - mean) * rstd * w + b,   rstd = 1 / sqrt(var + eps)
//     with g = dy * w and n = (x - mean) * rstd:   dx = rstd * (g - mean(g) - n * mean(g * n)),
//     dw = sum over rows of dy * n,   db = sum over rows of dy
//
// Bound by HBM: forward reads x and writes y, backward reads x and dy and writes dx; with 16-bit types the arithmetic is close
// behind, hence pairs of fp32 in one instruction (add, mul, fma .f32x2) wherever a row is read in vectors.  A row stays in the
// registers of one group of threads (a warp for short rows, a CTA for long ones) as it was read, so that the variance is
// that of the centred values, not a difference of two sums.  Backward CTAs walk the rows with a stride, the next rows streaming
// into a ring in shared memory, and keep the sums for dw and db of "their" rows in fp32 registers, column by column (each
// thread owns the same columns of every row); they write them once, [CTA, 2, cols], and a second kernel adds these in a fixed order.
// Rows longer than the registers hold are read again (from L2) and their column sums are kept in shared memory or, longer still,
// in the workspace itself.
//
// Measured (share of the copy rate of 6567 GB/s): forward 16384 x 8192 bf16 91.9 us (0.89), 65536 x 2048 bf16 88.8 us (0.92),
// 8192 x 8192 fp32 83.1 us (0.98); backward 16384 x 8192 bf16 134.9 us (0.91; 232 us with rows read straight into registers,
// 168 us with the ring and scalar arithmetic), 32768 x 4096 bf16 129.7 us (0.95), 8192 x 8192 fp32 134.8 us (0.91).
#include <algorithm>
#include "fp8_block.cuh"
#include "mxq_common.cuh"
#include "sm100_ptx.cuh"

namespace mxq {

__device__ int g_norm_status;            // MXQ_ERR_DEVICE once a kernel has given up on a wait

struct NormArgs {
    const void* x;
    const void* dy;              // backward
    const void* w;               // [cols] or null
    const void* b;               // [cols] or null (forward)
    void* out;                   // y or dx (backward: or null)
    float* mean;                 // [rows], forward: or null
    float* rstd;
    float* part;                 // backward: [CTAs, 2, cols] or null
    int64_t rows, cols, x_stride, dy_stride;
    float eps;
};

// VEC consecutive values as fp32
template <int DT, int VEC>
__device__ __forceinline__ void load_vec(const void* base, int64_t i, float (&v)[VEC]) {
    if constexpr (VEC == 1) {
        v[0] = load1<DT>(base, i);
    } else {
        constexpr int N = VecIO<DT, 16>::N;
#pragma unroll
        for (int j = 0; j < VEC; j += N) {
            uint32_t b[N];
            VecIO<DT, 16>::load(base, i + j, b);
#pragma unroll
            for (int k = 0; k < N; ++k) v[j + k] = __uint_as_float(b[k]);
        }
    }
}
template <int DT, int VEC>
__device__ __forceinline__ void store_vec(void* base, int64_t i, const float (&v)[VEC]) {
    if constexpr (VEC == 1) {
        store1<DT>(base, i, v[0]);
    } else if constexpr (DT == DT_F32) {
        float4* p = reinterpret_cast<float4*>(reinterpret_cast<float*>(base) + i);
#pragma unroll
        for (int j = 0; j < VEC; j += 4) p[j / 4] = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
    } else {
        uint32_t w[VEC / 2];
#pragma unroll
        for (int j = 0; j < VEC / 2; ++j) {
            if constexpr (DT == DT_BF16) {
                const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
                w[j] = *reinterpret_cast<const uint32_t*>(&h);
            } else {
                const __half2 h = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
                w[j] = *reinterpret_cast<const uint32_t*>(&h);
            }
        }
        static_assert(VEC == 8, "one 16-byte store");
        *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(base) + i) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// Sums of a and b over the TPR threads of a row, in every one of them.  Groups longer than a warp are the whole CTA;
// `buf` alternates between two halves of `red`, so one barrier a call is enough.
template <int TPR>
__device__ __forceinline__ void row_sum2(float& a, float& b, float2 (*red)[32], int buf) {
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) {
        a += __shfl_xor_sync(0xffffffffu, a, s);
        b += __shfl_xor_sync(0xffffffffu, b, s);
    }
    if constexpr (TPR > 32) {
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        if (lane == 0) red[buf][warp] = make_float2(a, b);
        __syncthreads();
        const float2 t = lane < TPR / 32 ? red[buf][lane] : make_float2(0.f, 0.f);
        a = t.x; b = t.y;
#pragma unroll
        for (int s = TPR / 64; s > 0; s >>= 1) {
            a += __shfl_xor_sync(0xffffffffu, a, s);
            b += __shfl_xor_sync(0xffffffffu, b, s);
        }
        a = __shfl_sync(0xffffffffu, a, 0);
        b = __shfl_sync(0xffffffffu, b, 0);
    }
}

// The same for one value; `half` names the half of `red` to use, another one each time.
template <int TPR>
__device__ __forceinline__ float row_sum(float a, float2 (*red)[32], int half) {
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) a += __shfl_xor_sync(0xffffffffu, a, s);
    if constexpr (TPR > 32) {
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        if (lane == 0) red[half][warp].x = a;
        __syncthreads();
        a = lane < TPR / 32 ? red[half][lane].x : 0.f;
#pragma unroll
        for (int s = TPR / 64; s > 0; s >>= 1) a += __shfl_xor_sync(0xffffffffu, a, s);
        a = __shfl_sync(0xffffffffu, a, 0);
    }
    return a;
}

// 16 bytes of a row as they lie in memory (VEC > 1), or one value
template <int DT, int VEC> struct Raw {
    uint4 q;
    __device__ __forceinline__ void load(const void* row, int64_t c) {
        q = *reinterpret_cast<const uint4*>(reinterpret_cast<const typename Store<DT>::T*>(row) + c);
    }
    __device__ __forceinline__ void zero() { q = make_uint4(0, 0, 0, 0); }
    __device__ __forceinline__ void get(float (&v)[VEC]) const {
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
        if constexpr (DT == DT_F32) {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(w[i]);
        } else if constexpr (DT == DT_BF16) {
#pragma unroll
            for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(w[i] << 16); v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
                v[2 * i] = f.x; v[2 * i + 1] = f.y;
            }
        }
    }
};
// The values of a Raw as pairs of fp32, two to a 64-bit register.
template <int DT, int VEC>
__device__ __forceinline__ void pairs(const Raw<DT, VEC>& r, uint64_t (&p)[VEC / 2]) {
    const uint32_t w[4] = {r.q.x, r.q.y, r.q.z, r.q.w};
    if constexpr (DT == DT_F32) {
        p[0] = ptx::pack2f(w[0], w[1]);
        p[1] = ptx::pack2f(w[2], w[3]);
    } else if constexpr (DT == DT_BF16) {
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = ptx::pack2f(w[i] << 16, w[i] & 0xffff0000u);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            p[i] = ptx::pack2f(f.x, f.y);
        }
    }
}
template <int DT> struct Raw<DT, 1> {
    float f;
    __device__ __forceinline__ void load(const void* row, int64_t c) { f = load1<DT>(row, c); }
    __device__ __forceinline__ void zero() { f = 0.f; }
    __device__ __forceinline__ void get(float (&v)[1]) const { v[0] = f; }
};

// threads of a CTA: four rows of a warp each, or one row
template <int TPR> constexpr int kNormThreads = TPR == 32 ? 128 : TPR;

// A row in registers: thread t of the row's TPR threads owns the NV groups of VEC columns at (i * TPR + t) * VEC.
template <int DT, int WDT, int VEC, int TPR, int NV>
__global__ void __launch_bounds__(kNormThreads<TPR>) layer_norm_fwd_kernel(const NormArgs g) {
    __shared__ float2 red[2][32];
    const int t = threadIdx.x % TPR;
    const int64_t row = (int64_t)blockIdx.x * (kNormThreads<TPR> / TPR) + threadIdx.x / TPR;
    if (TPR == 32 && row >= g.rows) return;                    // a warp on its own; a CTA-wide row always exists
    using T = typename Store<DT>::T;
    const T* x = reinterpret_cast<const T*>(g.x) + row * g.x_stride;
    Raw<DT, VEC> raw[NV];                                      // as it came: half the registers of fp32 for 16-bit types
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * TPR + t) * VEC;
        if (c < g.cols) raw[i].load(x, c);
        else raw[i].zero();
    }
    const float inv = 1.f / (float)g.cols;
    float mean, rstd;
    if constexpr (VEC > 1) {                                   // pairs of values, two operations an instruction
        uint64_t p[VEC / 2], s2 = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            pairs(raw[i], p);
#pragma unroll
            for (int j = 0; j < VEC / 2; ++j) s2 = ptx::add2(s2, p[j]);
        }
        float s, hi;
        ptx::unpack2f(s2, s, hi);
        mean = row_sum<TPR>(s + hi, red, 0) * inv;
        const uint64_t off = ptx::pack2f(-mean, -mean);
        s2 = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if ((i * TPR + t) * VEC >= g.cols) continue;
            pairs(raw[i], p);
#pragma unroll
            for (int j = 0; j < VEC / 2; ++j) { const uint64_t d = ptx::add2(p[j], off); ptx::fma2(s2, d, d); }
        }
        ptx::unpack2f(s2, s, hi);
        rstd = 1.f / sqrtf(row_sum<TPR>(s + hi, red, 1) * inv + g.eps);
        const uint64_t scale = ptx::pack2f(rstd, rstd), shift = ptx::pack2f(-mean * rstd, -mean * rstd);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * TPR + t) * VEC;
            if (c >= g.cols) continue;
            float w[VEC], b[VEC], o[VEC];
            if (g.w) load_vec<WDT, VEC>(g.w, c, w);
            if (g.b) load_vec<WDT, VEC>(g.b, c, b);
            pairs(raw[i], p);
#pragma unroll
            for (int j = 0; j < VEC / 2; ++j) {
                uint64_t n = ptx::fma2_to(p[j], scale, shift);
                if (g.w && g.b) n = ptx::fma2_to(n, ptx::pack2f(w[2 * j], w[2 * j + 1]), ptx::pack2f(b[2 * j], b[2 * j + 1]));
                else if (g.w) n = ptx::mul2(n, ptx::pack2f(w[2 * j], w[2 * j + 1]));
                else if (g.b) n = ptx::add2(n, ptx::pack2f(b[2 * j], b[2 * j + 1]));
                ptx::unpack2f(n, o[2 * j], o[2 * j + 1]);
            }
            store_vec<DT, VEC>(g.out, row * g.cols + c, o);
        }
    } else {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) s += raw[i].f;
        mean = row_sum<TPR>(s, red, 0) * inv;
        s = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const float d = raw[i].f - mean;
            if (i * TPR + t < g.cols) s = __fmaf_rn(d, d, s);
        }
        rstd = 1.f / sqrtf(row_sum<TPR>(s, red, 1) * inv + g.eps);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = i * TPR + t;
            if (c >= g.cols) continue;
            float n = (raw[i].f - mean) * rstd;
            if (g.w) n *= load1<WDT>(g.w, c);
            if (g.b) n += load1<WDT>(g.b, c);
            store1<DT>(g.out, row * g.cols + c, n);
        }
    }
    if (t == 0 && g.mean) { g.mean[row] = mean; g.rstd[row] = rstd; }
}

// Rows of any length: read three times, the later ones from L2.
template <int DT, int WDT>
__global__ void __launch_bounds__(1024) layer_norm_fwd_long_kernel(const NormArgs g) {
    __shared__ float2 red[2][32];
    const int64_t row = blockIdx.x;
    using T = typename Store<DT>::T;
    const T* x = reinterpret_cast<const T*>(g.x) + row * g.x_stride;
    float s = 0.f, z = 0.f;
    for (int64_t c = threadIdx.x; c < g.cols; c += 1024) s += load1<DT>(x, c);
    row_sum2<1024>(s, z, red, 0);
    const float mean = s / (float)g.cols;
    s = z = 0.f;
    for (int64_t c = threadIdx.x; c < g.cols; c += 1024) { const float d = load1<DT>(x, c) - mean; s = __fmaf_rn(d, d, s); }
    row_sum2<1024>(s, z, red, 1);
    const float rstd = 1.f / sqrtf(s / (float)g.cols + g.eps);
    if (threadIdx.x == 0 && g.mean) { g.mean[row] = mean; g.rstd[row] = rstd; }
    for (int64_t c = threadIdx.x; c < g.cols; c += 1024) {
        float n = (load1<DT>(x, c) - mean) * rstd;
        if (g.w) n *= load1<WDT>(g.w, c);
        if (g.b) n += load1<WDT>(g.b, c);
        store1<DT>(g.out, row * g.cols + c, n);
    }
}

// Long rows whose layout allows bulk copies: the CTA's next rows of x and dy stream into a ring in shared memory
// while it works on one, so that copies are always in flight whatever the row's two sums wait for.  A thread takes its values of
// a row into registers; once the row's sums have met at the barrier everyone has, and the row's place is refilled.
template <int DT, int WDT, int TPR, int NV, int STAGES>
__global__ void __launch_bounds__(TPR) layer_norm_bwd_ring_kernel(const NormArgs g) {
    constexpr int VEC = DT == DT_F32 ? 4 : 8;
    extern __shared__ __align__(128) uint8_t ring[];           // [STAGES][2][row]
    __shared__ float2 red[2][32];
    __shared__ uint64_t full[STAGES];
    __shared__ int abort_word;
    volatile int* abort_flag = &abort_word;
    using T = typename Store<DT>::T;
    const int t = threadIdx.x;
    const uint32_t row_bytes = (uint32_t)g.cols * sizeof(T);
    auto fetch = [&](int64_t row, int s) {
        const uint32_t bar = ptx::smem_u32(&full[s]), dst = ptx::smem_u32(ring) + 2 * s * row_bytes;
        ptx::mbar_expect_tx(bar, 2 * row_bytes);
        ptx::bulk_load(dst, reinterpret_cast<const T*>(g.x) + row * g.x_stride, row_bytes, bar);
        ptx::bulk_load(dst + row_bytes, reinterpret_cast<const T*>(g.dy) + row * g.dy_stride, row_bytes, bar);
    };
    if (t == 0) {
        for (int s = 0; s < STAGES; ++s) ptx::mbar_init(ptx::smem_u32(&full[s]), 1);
        abort_word = 0;
        ptx::fence_mbar_init();
        ptx::fence_proxy_async();
        for (int s = 0; s < STAGES; ++s)
            if (blockIdx.x + (int64_t)s * gridDim.x < g.rows) fetch(blockIdx.x + (int64_t)s * gridDim.x, s);
    }
    __syncthreads();
    constexpr bool KEEP = TPR * NV * VEC <= 8192;              // longer rows leave no registers for the weights
    uint64_t dw[NV][VEC / 2], db[NV][VEC / 2], w[KEEP ? NV : 1][VEC / 2];  // pairs of fp32; two sums or products an instruction
    auto weights = [&](int i, uint64_t (&to)[VEC / 2]) {
        const int c = (i * TPR + t) * VEC;
        float f[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) f[j] = 1.f;
        if (g.w && c < g.cols) load_vec<WDT, VEC>(g.w, c, f);
#pragma unroll
        for (int j = 0; j < VEC / 2; ++j) to[j] = ptx::pack2f(f[2 * j], f[2 * j + 1]);
    };
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        if constexpr (KEEP) weights(i, w[i]);
#pragma unroll
        for (int j = 0; j < VEC / 2; ++j) dw[i][j] = db[i][j] = 0;
    }
    const float inv = 1.f / (float)g.cols;
    float mean = 0.f, rstd = 0.f;
    if (blockIdx.x < g.rows) { mean = g.mean[blockIdx.x]; rstd = g.rstd[blockIdx.x]; }
    int it = 0;
    for (int64_t row = blockIdx.x; row < g.rows; row += gridDim.x, ++it) {
        const int s = it % STAGES;
        float mean_next = 0.f, rstd_next = 0.f;
        if (row + gridDim.x < g.rows) { mean_next = g.mean[row + gridDim.x]; rstd_next = g.rstd[row + gridDim.x]; }
        const uint64_t scale = ptx::pack2f(rstd, rstd), shift = ptx::pack2f(-mean * rstd, -mean * rstd);
        ptx::mbar_wait(ptx::smem_u32(&full[s]), (it / STAGES) & 1, abort_flag);
        const uint8_t* px = ring + 2 * s * row_bytes;
        Raw<DT, VEC> x[NV], d[NV];
        uint64_t sg2 = 0, sn2 = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * TPR + t) * VEC;
            if (c >= g.cols) continue;
            x[i].load(px, c);
            d[i].load(px + row_bytes, c);
            uint64_t xv[VEC / 2], dv[VEC / 2];
            pairs(x[i], xv);
            pairs(d[i], dv);
            uint64_t (&wi)[VEC / 2] = w[KEEP ? i : 0];
            if constexpr (!KEEP) weights(i, wi);
#pragma unroll
            for (int j = 0; j < VEC / 2; ++j) {
                const uint64_t n = ptx::fma2_to(xv[j], scale, shift), h = ptx::mul2(dv[j], wi[j]);
                ptx::fma2(dw[i][j], dv[j], n);
                db[i][j] = ptx::add2(db[i][j], dv[j]);
                sg2 = ptx::add2(sg2, h);
                ptx::fma2(sn2, h, n);
            }
        }
        float sg, sn, hi;
        ptx::unpack2f(sg2, sg, hi);
        sg += hi;
        ptx::unpack2f(sn2, sn, hi);
        sn += hi;
        row_sum2<TPR>(sg, sn, red, it & 1);
        if (t == 0 && row + (int64_t)STAGES * gridDim.x < g.rows) fetch(row + (int64_t)STAGES * gridDim.x, s);
        if (g.out) {
            const float a0 = -sg * inv * rstd, a1 = -sn * inv * rstd;
            const uint64_t k0 = ptx::pack2f(a0, a0), k1 = ptx::pack2f(a1, a1);
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (i * TPR + t) * VEC;
                if (c >= g.cols) continue;
                uint64_t xv[VEC / 2], dv[VEC / 2];
                float o[VEC];
                pairs(x[i], xv);
                pairs(d[i], dv);
                uint64_t (&wi)[VEC / 2] = w[KEEP ? i : 0];
                if constexpr (!KEEP) weights(i, wi);
#pragma unroll
                for (int j = 0; j < VEC / 2; ++j) {
                    const uint64_t n = ptx::fma2_to(xv[j], scale, shift), h = ptx::mul2(dv[j], wi[j]);
                    ptx::unpack2f(ptx::fma2_to(n, k1, ptx::fma2_to(h, scale, k0)), o[2 * j], o[2 * j + 1]);
                }
                store_vec<DT, VEC>(g.out, row * g.cols + c, o);
            }
        }
        mean = mean_next; rstd = rstd_next;
    }
    if (*abort_flag && t == 0) {                               // copies still in flight get a bounded time to land
        for (int s = 0; s < STAGES; ++s)
            for (uint32_t i = 0; i < 4096 && !ptx::mbar_try_wait(ptx::smem_u32(&full[s]), 0) &&
                                 !ptx::mbar_try_wait(ptx::smem_u32(&full[s]), 1); ++i) __nanosleep(64);
        atomicExch(&g_norm_status, MXQ_ERR_DEVICE);
    }
    if (!g.part) return;
    float* part = g.part + (int64_t)blockIdx.x * 2 * g.cols;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * TPR + t) * VEC;
        if (c >= g.cols) continue;
#pragma unroll
        for (int j = 0; j < VEC / 2; ++j) {
            *reinterpret_cast<uint64_t*>(part + c + 2 * j) = dw[i][j];
            *reinterpret_cast<uint64_t*>(part + g.cols + c + 2 * j) = db[i][j];
        }
    }
}

template <int DT, int WDT, int VEC, int TPR, int NV>
__global__ void __launch_bounds__(kNormThreads<TPR>) layer_norm_bwd_kernel(const NormArgs g) {
    constexpr int ROWS = kNormThreads<TPR> / TPR;
    __shared__ float2 red[2][32];
    const int t = threadIdx.x % TPR, group = threadIdx.x / TPR;
    using T = typename Store<DT>::T;
    float dw[NV][VEC], db[NV][VEC];
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < VEC; ++j) dw[i][j] = db[i][j] = 0.f;
    const float inv = 1.f / (float)g.cols;
    int buf = 0;
    for (int64_t row = (int64_t)blockIdx.x * ROWS + group; row < g.rows; row += (int64_t)gridDim.x * ROWS, buf ^= 1) {
        const T* x = reinterpret_cast<const T*>(g.x) + row * g.x_stride;
        const T* dy = reinterpret_cast<const T*>(g.dy) + row * g.dy_stride;
        const float mean = g.mean[row], rstd = g.rstd[row];
        float n[NV][VEC], d[NV][VEC];
        float s = 0.f, sn = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int64_t c = (int64_t)(i * TPR + t) * VEC;
            if (c < g.cols) {
                load_vec<DT, VEC>(x, c, n[i]);
                load_vec<DT, VEC>(dy, c, d[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int64_t c = (int64_t)(i * TPR + t) * VEC;
            if (c >= g.cols) continue;
            float w[VEC];
            if (g.w) load_vec<WDT, VEC>(g.w, c, w);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                n[i][j] = (n[i][j] - mean) * rstd;
                dw[i][j] = __fmaf_rn(d[i][j], n[i][j], dw[i][j]);
                db[i][j] += d[i][j];
                if (g.w) d[i][j] *= w[j];
                s += d[i][j];
                sn = __fmaf_rn(d[i][j], n[i][j], sn);
            }
        }
        if (!g.out) continue;                                  // the same for every thread
        row_sum2<TPR>(s, sn, red, buf);
        s *= inv; sn *= inv;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int64_t c = (int64_t)(i * TPR + t) * VEC;
            if (c >= g.cols) continue;
#pragma unroll
            for (int j = 0; j < VEC; ++j) d[i][j] = rstd * (d[i][j] - s - n[i][j] * sn);
            store_vec<DT, VEC>(g.out, row * g.cols + c, d[i]);
        }
    }
    if (!g.part) return;
    float* part = g.part + (int64_t)blockIdx.x * 2 * g.cols;
    if constexpr (ROWS == 1) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int64_t c = (int64_t)(i * TPR + t) * VEC;
            if (c >= g.cols) continue;
#pragma unroll
            for (int j = 0; j < VEC; ++j) { part[c + j] = dw[i][j]; part[g.cols + c + j] = db[i][j]; }
        }
    } else {
        // the CTA's warps add their sums one after the other
        __shared__ float acc[2][TPR * NV * VEC];
        for (int r = 0; r < ROWS; ++r) {
            if (group == r) {
#pragma unroll
                for (int i = 0; i < NV; ++i)
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        const int c = (i * TPR + t) * VEC + j;
                        acc[0][c] = r ? acc[0][c] + dw[i][j] : dw[i][j];
                        acc[1][c] = r ? acc[1][c] + db[i][j] : db[i][j];
                    }
            }
            __syncthreads();
        }
        for (int c = threadIdx.x; c < g.cols; c += kNormThreads<TPR>) { part[c] = acc[0][c]; part[g.cols + c] = acc[1][c]; }
    }
}

// Rows of any length: read twice; column sums in shared memory (SMEM) or in this CTA's rows of the workspace.
template <int DT, int WDT, bool SMEM>
__global__ void __launch_bounds__(1024) layer_norm_bwd_long_kernel(const NormArgs g) {
    extern __shared__ float sums[];
    __shared__ float2 red[2][32];
    using T = typename Store<DT>::T;
    float* part = g.part ? g.part + (int64_t)blockIdx.x * 2 * g.cols : nullptr;
    float* aw = SMEM ? sums : part;
    float* ab = aw ? aw + g.cols : nullptr;
    const bool keep = g.part != nullptr;
    if (keep)
        for (int64_t c = threadIdx.x; c < g.cols; c += 1024) aw[c] = ab[c] = 0.f;
    const float inv = 1.f / (float)g.cols;
    int buf = 0;
    for (int64_t row = blockIdx.x; row < g.rows; row += gridDim.x, buf ^= 1) {
        const T* x = reinterpret_cast<const T*>(g.x) + row * g.x_stride;
        const T* dy = reinterpret_cast<const T*>(g.dy) + row * g.dy_stride;
        const float mean = g.mean[row], rstd = g.rstd[row];
        float s = 0.f, sn = 0.f;
        for (int64_t c = threadIdx.x; c < g.cols; c += 1024) {
            const float n = (load1<DT>(x, c) - mean) * rstd, d = load1<DT>(dy, c);
            if (keep) { aw[c] = __fmaf_rn(d, n, aw[c]); ab[c] += d; }
            const float h = g.w ? d * load1<WDT>(g.w, c) : d;
            s += h;
            sn = __fmaf_rn(h, n, sn);
        }
        if (!g.out) continue;
        row_sum2<1024>(s, sn, red, buf);
        s *= inv; sn *= inv;
        for (int64_t c = threadIdx.x; c < g.cols; c += 1024) {
            const float n = (load1<DT>(x, c) - mean) * rstd, d = load1<DT>(dy, c);
            const float h = g.w ? d * load1<WDT>(g.w, c) : d;
            store1<DT>(g.out, row * g.cols + c, rstd * (h - s - n * sn));
        }
    }
    if (SMEM && keep)
        for (int64_t c = threadIdx.x; c < g.cols; c += 1024) { part[c] = aw[c]; part[g.cols + c] = ab[c]; }   // a thread's own columns
}

// Threads a row and values a thread: the smallest group that holds the row at 16 values a thread (8 for a warp's
// shortest rows), so that registers leave room for several CTAs on an SM.
struct NormShape { int tpr, vals; };
static NormShape norm_shape(int64_t cols) {
    if (cols <= 256) return {32, 8};
    if (cols <= 512) return {32, 16};
    if (cols <= 1024) return {128, 8};
    if (cols <= 2048) return {128, 16};
    if (cols <= 4096) return {256, 16};
    if (cols <= 8192) return {512, 16};
    return {0, 0};
}

static int64_t norm_bwd_ctas(int64_t rows, int64_t cols) {
    const NormShape s = norm_shape(cols);
    const int64_t per = s.tpr == 32 ? 4 : 1, resident = s.tpr == 0 || s.tpr >= 512 ? 1 : s.tpr >= 256 ? 2 : s.tpr == 128 && s.vals == 8 ? 8 : s.tpr == 32 ? 8 : 4;
    return std::max<int64_t>(1, std::min<int64_t>((rows + per - 1) / per, sm_count() * resident));
}

// Pairs of rows in the ring: 128 KB of them at 8192 16-bit columns; two of 64 KB at 8192 fp32 columns.
template <int DT, int WDT, int TPR, int VALS, int STAGES = ((TPR * VALS > 8192) ? 3 : (DT == DT_F32 && TPR * VALS == 8192) ? 2 : 4)>
static int launch_ring(const NormArgs& g, cudaStream_t st) {
    constexpr int VEC = DT == DT_F32 ? 4 : 8;
    auto kern = layer_norm_bwd_ring_kernel<DT, WDT, TPR, VALS / VEC, STAGES>;
    const int bytes = STAGES * 2 * (int)g.cols * (DT == DT_F32 ? 4 : 2);
    static_assert(STAGES * 2 * TPR * VALS * (DT == DT_F32 ? 4 : 2) <= 200 * 1024, "shared memory");
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) { cudaGetLastError(); return MXQ_ERR_CUDA; }
    kern<<<(int)norm_bwd_ctas(g.rows, g.cols), TPR, bytes, st>>>(g);
    return check_launch();
}

template <int DT, int WDT, int VEC, int TPR, int VALS>
static int launch_norm_fwd(const NormArgs& g, cudaStream_t st) {
    constexpr int per = kNormThreads<TPR> / TPR;
    const int64_t grid = (g.rows + per - 1) / per;
    if (grid > 0x7fffffff) return MXQ_ERR_TOO_LARGE;
    layer_norm_fwd_kernel<DT, WDT, VEC, TPR, VALS / VEC><<<(int)grid, kNormThreads<TPR>, 0, st>>>(g);
    return check_launch();
}

template <int DT, int WDT, int VEC, int TPR, int VALS>
static int launch_norm(const NormArgs& g, bool bwd, cudaStream_t st) {
    constexpr int threads = kNormThreads<TPR>;
    if (bwd) {
        layer_norm_bwd_kernel<DT, WDT, VEC, TPR, VALS / VEC><<<(int)norm_bwd_ctas(g.rows, g.cols), threads, 0, st>>>(g);
    } else {
        return launch_norm_fwd<DT, WDT, VEC, TPR, VALS>(g, st);
    }
    return check_launch();
}

template <int DT, int WDT, int VEC>
static int launch_norm_vec(const NormArgs& g, bool bwd, cudaStream_t st) {
    const NormShape s = norm_shape(g.cols);
    if (s.tpr == 32 && s.vals == 8) return launch_norm<DT, WDT, VEC, 32, 8>(g, bwd, st);
    if (s.tpr == 32) return launch_norm<DT, WDT, VEC, 32, 16>(g, bwd, st);
    if constexpr (VEC == 1) {
        if (s.tpr == 128 && s.vals == 8) return launch_norm<DT, WDT, VEC, 128, 8>(g, bwd, st);
        if (s.tpr == 128) return launch_norm<DT, WDT, VEC, 128, 16>(g, bwd, st);
        if (s.tpr == 256) return launch_norm<DT, WDT, VEC, 256, 16>(g, bwd, st);
        return launch_norm<DT, WDT, VEC, 512, 16>(g, bwd, st);
    } else if (bwd) {                                          // whole vectors and 16-byte aligned rows
        if (s.tpr == 128 && s.vals == 8) return launch_ring<DT, WDT, 128, 8>(g, st);
        if (s.tpr == 128) return launch_ring<DT, WDT, 128, 16>(g, st);
        if (s.tpr == 256) return launch_ring<DT, WDT, 256, 16>(g, st);
        return launch_ring<DT, WDT, 512, 16>(g, st);
    } else if (g.rows >= 4 * sm_count()) {
        // few barriers and many rows in flight: 32 or, packed two to a register, 64 values a thread.  16384 x 8192 bf16:
        // 512 threads x 16 values 143 us, 256 x 32 107 us, 128 x 64 92 us; 65536 x 2048: 128 x 16 108, 64 x 32 89
        if (g.cols <= 1024) return launch_norm_fwd<DT, WDT, VEC, 32, 32>(g, st);
        if (g.cols <= 2048) return launch_norm_fwd<DT, WDT, VEC, 64, 32>(g, st);
        if constexpr (DT == DT_F32) {
            if (g.cols <= 4096) return launch_norm_fwd<DT, WDT, VEC, 128, 32>(g, st);
            return launch_norm_fwd<DT, WDT, VEC, 256, 32>(g, st);
        } else {
            if (g.cols <= 4096) return launch_norm_fwd<DT, WDT, VEC, 64, 64>(g, st);
            return launch_norm_fwd<DT, WDT, VEC, 128, 64>(g, st);
        }
    } else {                                                   // few rows: many threads on each
        if (s.tpr == 128 && s.vals == 8) return launch_norm_fwd<DT, WDT, VEC, 128, 8>(g, st);
        if (s.tpr == 128) return launch_norm_fwd<DT, WDT, VEC, 128, 16>(g, st);
        if (s.tpr == 256) return launch_norm_fwd<DT, WDT, VEC, 256, 16>(g, st);
        return launch_norm_fwd<DT, WDT, VEC, 512, 16>(g, st);
    }
}

template <int DT, int WDT>
static int launch_norm_long(const NormArgs& g, bool bwd, cudaStream_t st) {
    if (!bwd) {
        if (g.rows > 0x7fffffff) return MXQ_ERR_TOO_LARGE;
        layer_norm_fwd_long_kernel<DT, WDT><<<(int)g.rows, 1024, 0, st>>>(g);
        return check_launch();
    }
    const int grid = (int)norm_bwd_ctas(g.rows, g.cols);
    const int64_t bytes = g.part ? 8 * g.cols : 0;
    if (bytes <= 200 * 1024) {
        auto kern = layer_norm_bwd_long_kernel<DT, WDT, true>;
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024) != cudaSuccess) { cudaGetLastError(); return MXQ_ERR_CUDA; }
        kern<<<grid, 1024, (size_t)bytes, st>>>(g);
    } else {
        layer_norm_bwd_long_kernel<DT, WDT, false><<<grid, 1024, 0, st>>>(g);
    }
    return check_launch();
}

template <int DT, int WDT>
static int launch_norm_dt(const NormArgs& g, bool bwd, cudaStream_t st) {
    constexpr int VEC = DT == DT_F32 ? 4 : 8;
    const int es = DT == DT_F32 ? 4 : 2;
    // 16-byte accesses: whole vectors in a row, aligned rows, aligned weights
    const bool vec = g.cols % VEC == 0 && aligned16(g.x) && aligned16(g.out) && (g.rows == 1 || g.x_stride * es % 16 == 0) &&
                     aligned16(g.w) && aligned16(g.b) && (!bwd || (aligned16(g.dy) && (g.rows == 1 || g.dy_stride * es % 16 == 0)));
    if constexpr (DT != DT_F32) {
        if (vec && g.cols > 8192 && g.cols <= 16384) {         // 32 or 64 packed values a thread
            if (bwd) return launch_ring<DT, WDT, 512, 32>(g, st);
            return launch_norm_fwd<DT, WDT, VEC, 256, 64>(g, st);
        }
    }
    if (norm_shape(g.cols).tpr) return vec ? launch_norm_vec<DT, WDT, VEC>(g, bwd, st) : launch_norm_vec<DT, WDT, 1>(g, bwd, st);
    return launch_norm_long<DT, WDT>(g, bwd, st);
}

int norm_status(int clear) {
    int v = 0;
    if (cudaMemcpyFromSymbol(&v, g_norm_status, sizeof v) != cudaSuccess) { cudaGetLastError(); return MXQ_ERR_CUDA; }
    if (clear && v != 0) {
        const int zero = 0;
        cudaMemcpyToSymbol(g_norm_status, &zero, sizeof zero);
    }
    return v;
}

static int norm_dispatch(const NormArgs& g, int dtype, int wdtype, bool bwd, cudaStream_t st) {
    if (dtype == MXQ_F32) return wdtype == MXQ_F32 ? launch_norm_dt<DT_F32, DT_F32>(g, bwd, st) : MXQ_ERR_UNSUPPORTED;
    if (dtype == MXQ_F16) {
        if (wdtype == MXQ_F16) return launch_norm_dt<DT_F16, DT_F16>(g, bwd, st);
        return wdtype == MXQ_F32 ? launch_norm_dt<DT_F16, DT_F32>(g, bwd, st) : MXQ_ERR_UNSUPPORTED;
    }
    if (wdtype == MXQ_BF16) return launch_norm_dt<DT_BF16, DT_BF16>(g, bwd, st);
    return wdtype == MXQ_F32 ? launch_norm_dt<DT_BF16, DT_F32>(g, bwd, st) : MXQ_ERR_UNSUPPORTED;
}

}  // namespace mxq

extern "C" int mxq_layer_norm_fwd(const void* x, int dtype, int64_t x_stride, const void* w, const void* b, int w_dtype, void* y,
                                  float* mean, float* rstd, int64_t rows, int64_t cols, float eps, void* stream) {
    using namespace mxq;
    if (rows < 0 || cols <= 0 || dtype < 0 || dtype > 2 || w_dtype < 0 || w_dtype > 2 || !mean != !rstd) return MXQ_ERR_BAD_ARG;
    if (rows == 0) return MXQ_OK;
    if (!x || !y || (rows > 1 && x_stride < cols)) return MXQ_ERR_BAD_ARG;
    NormArgs g = {};
    g.x = x; g.w = w; g.b = b; g.out = y; g.mean = mean; g.rstd = rstd;
    g.rows = rows; g.cols = cols; g.x_stride = x_stride; g.eps = eps;
    return norm_dispatch(g, dtype, w_dtype, false, (cudaStream_t)stream);
}

extern "C" int64_t mxq_layer_norm_workspace_bytes(int64_t rows, int64_t cols) {
    return rows <= 0 || cols <= 0 ? 0 : mxq::norm_bwd_ctas(rows, cols) * 8 * cols;
}

extern "C" int mxq_layer_norm_bwd(const void* dy, const void* x, int dtype, int64_t dy_stride, int64_t x_stride, const void* w, int w_dtype,
                                  const float* mean, const float* rstd, void* dx, void* dw, void* db, int sums_dtype, void* workspace,
                                  int64_t workspace_bytes, int64_t rows, int64_t cols, void* stream) {
    using namespace mxq;
    if (rows < 0 || cols <= 0 || dtype < 0 || dtype > 2 || w_dtype < 0 || w_dtype > 2 || sums_dtype < 0 || sums_dtype > 2) return MXQ_ERR_BAD_ARG;
    if (!dx && !dw && !db) return MXQ_OK;
    cudaStream_t st = (cudaStream_t)stream;
    const bool sums = dw || db;
    if (rows == 0) return sum_partials(nullptr, 0, cols, 2, dw, db, sums_dtype, st);
    if (!x || !dy || !mean || !rstd || (rows > 1 && (x_stride < cols || dy_stride < cols))) return MXQ_ERR_BAD_ARG;
    if (sums && (!workspace || workspace_bytes < mxq_layer_norm_workspace_bytes(rows, cols))) return MXQ_ERR_BAD_ARG;
    if (sums && !aligned16(workspace)) return MXQ_ERR_ALIGN;
    NormArgs g = {};
    g.x = x; g.dy = dy; g.w = w; g.out = dx; g.mean = const_cast<float*>(mean); g.rstd = const_cast<float*>(rstd);
    g.part = sums ? (float*)workspace : nullptr;
    g.rows = rows; g.cols = cols; g.x_stride = x_stride; g.dy_stride = dy_stride;
    const int rc = norm_dispatch(g, dtype, w_dtype, true, st);
    return rc || !sums ? rc : sum_partials(g.part, norm_bwd_ctas(rows, cols), cols, 2, dw, db, sums_dtype, st);
}
