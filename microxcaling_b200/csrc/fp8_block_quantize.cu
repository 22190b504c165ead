// 8-bit quantization with one fp32 scale per 128 values (sm_100a).
//
// A block of 128 values with maximum magnitude a has the scale s = max(a, 2^-100) * (1 / top), the inverse r = 1 / s
// and the codes RNE(v * r) in e4m3 (top 448) or e5m2 (top 57344); s, r and v * r are fp32, each rounded to nearest.
// The bound 2^-100 keeps r finite for blocks of zeros and of tiny values (their codes are then 0).  A block that holds
// an infinity or a NaN has the scale Inf / NaN, and every product with it is NaN.
//
// One CTA of 256 threads takes a 128 x 128 tile, one thread 8 consecutive rows x 8 consecutive columns of it in
// registers.  The tile is what both block directions have in common: row blocks (1 x 128) are maxima over 16 lanes,
// column blocks (128 x 1) maxima over the thread's own rows, one shuffle and eight warps, and a 128 x 128 block is
// all of them, so x is read once whatever is asked for.  The transposed codes pass through shared memory as 8-byte
// pieces (8 rows of one column), XOR-swizzled by the column group so that neither side has bank conflicts, and leave
// as whole 128-byte rows of the transposed operand.
#include "mxq_common.cuh"
#include "fp8_block.cuh"
#include "sm100_ptx.cuh"

namespace mxq {

struct QuantArgs {
    const void* x;
    int64_t rows, cols, stride;      // stride in elements
    uint8_t* codes;                  // [rows, pitch] or null
    int64_t pitch;
    float* scales;                   // [col blocks, rows] (tile: [col blocks, row blocks])
    uint8_t* codes_t;                // [cols, pitch_t] or null
    int64_t pitch_t;
    float* scales_t;                 // [row blocks, cols] (tile: [row blocks, col blocks])
    float* colsum;                   // [row blocks, cols] sums over the tile's rows, or null
    int64_t row_blocks, col_blocks;
    float inv_top;                   // 1 / (largest value of the format), rounded to fp32
    int vec;                         // 16-byte loads: base and row stride aligned
};

__device__ __forceinline__ void load8(const QuantArgs& g, int64_t row, int64_t col, float (&v)[8]) {
    const float* p = reinterpret_cast<const float*>(g.x) + row * g.stride + col;
    if (row < g.rows && col + 8 <= g.cols && g.vec) {
        const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
        v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (row < g.rows && col + i < g.cols) ? p[i] : 0.f;
    }
}

// max that keeps a NaN
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

template <bool E5M2>
__device__ __forceinline__ uint32_t code2(float lo, float hi) {
    uint16_t r;
    if (E5M2) asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
template <bool E5M2>
__device__ __forceinline__ uint2 code8(const float (&v)[8]) {
    return make_uint2(code2<E5M2>(v[0], v[1]) | (code2<E5M2>(v[2], v[3]) << 16),
                      code2<E5M2>(v[4], v[5]) | (code2<E5M2>(v[6], v[7]) << 16));
}

__device__ __forceinline__ float block_scale(float amax, float inv_top) {
    return __fmul_rn(max_nan(amax, 0x1p-100f), inv_top);
}

// fp32 inputs
template <bool E5M2>
__global__ void __launch_bounds__(256)
fp8_quantize_kernel(const QuantArgs g, const bool tile) {
    __shared__ float col_part[8][128];          // per-warp column maxima
    __shared__ float col_sum[8][128];
    __shared__ float warp_part[8];
    __shared__ float col_r[128];
    __shared__ uint2 stage[128][16];
    ptx::grid_launch_dependents();               // a product launched to overlap waits for this grid before it reads its results
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int l16 = lane & 15, h = lane >> 4;
    const int64_t cb = blockIdx.x % g.col_blocks, rb = blockIdx.x / g.col_blocks;
    const int64_t row0 = rb * 128 + 16 * warp + 8 * h, col0 = cb * 128 + 8 * l16;

    float v[8][8];
#pragma unroll
    for (int i = 0; i < 8; ++i) load8(g, row0 + i, col0, v[i]);

    float rmax[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        rmax[i] = fabsf(v[i][0]);
#pragma unroll
        for (int j = 1; j < 8; ++j) rmax[i] = max_nan(rmax[i], fabsf(v[i][j]));
    }
    if (g.colsum) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) s += v[i][j];
            s += __shfl_xor_sync(0xffffffffu, s, 16);
            if (h == 0) col_sum[warp][8 * l16 + j] = s;
        }
    }
    float tile_s = 0.f, tile_r = 0.f;
    if (tile) {
        float m = rmax[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) m = max_nan(m, rmax[i]);
#pragma unroll
        for (int s = 16; s > 0; s >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, s));
        if (lane == 0) warp_part[warp] = m;
        __syncthreads();
        m = warp_part[0];
#pragma unroll
        for (int w = 1; w < 8; ++w) m = max_nan(m, warp_part[w]);
        tile_s = block_scale(m, g.inv_top);
        tile_r = __fdiv_rn(1.f, tile_s);
        if (threadIdx.x == 0) {
            if (g.scales) g.scales[cb * g.row_blocks + rb] = tile_s;
            if (g.scales_t) g.scales_t[rb * g.col_blocks + cb] = tile_s;
        }
    }
    // row blocks
    if (g.codes) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float r = tile_r;
            if (!tile) {
                float m = rmax[i];
#pragma unroll
                for (int s = 8; s > 0; s >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, s));
                const float sc = block_scale(m, g.inv_top);
                r = __fdiv_rn(1.f, sc);
                if (l16 == 0 && row0 + i < g.rows) g.scales[cb * g.rows + row0 + i] = sc;
            }
            float q[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) q[j] = __fmul_rn(v[i][j], r);
            // whole 8-byte groups: the row pitch is a multiple of 16, so a group that starts inside the row ends inside it
            if (row0 + i < g.rows && col0 < g.cols)
                *reinterpret_cast<uint2*>(g.codes + (row0 + i) * g.pitch + col0) = code8<E5M2>(q);
        }
    }
    if (!g.codes_t && !g.colsum) return;
    // column blocks
    if (g.codes_t && !tile) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float m = fabsf(v[0][j]);
#pragma unroll
            for (int i = 1; i < 8; ++i) m = max_nan(m, fabsf(v[i][j]));
            m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, 16));
            if (h == 0) col_part[warp][8 * l16 + j] = m;
        }
    }
    __syncthreads();
    if (threadIdx.x < 128) {
        const int64_t col = cb * 128 + threadIdx.x;
        if (g.codes_t && !tile) {
            float m = col_part[0][threadIdx.x];
#pragma unroll
            for (int w = 1; w < 8; ++w) m = max_nan(m, col_part[w][threadIdx.x]);
            const float sc = block_scale(m, g.inv_top);
            col_r[threadIdx.x] = __fdiv_rn(1.f, sc);
            if (col < g.cols) g.scales_t[rb * g.cols + col] = sc;
        }
        if (g.colsum && col < g.cols) {
            float s = col_sum[0][threadIdx.x];
#pragma unroll
            for (int w = 1; w < 8; ++w) s += col_sum[w][threadIdx.x];
            g.colsum[rb * g.cols + col] = s;
        }
    }
    if (!g.codes_t) return;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int c = 8 * l16 + j;
        const float r = tile ? tile_r : col_r[c];
        float q[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) q[i] = __fmul_rn(v[i][j], r);
        stage[c][(2 * warp + h) ^ l16] = code8<E5M2>(q);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int c = 16 * i + 2 * warp + h;                  // one column of the tile = one row of the result
        const int64_t col = cb * 128 + c, row = rb * 128 + 8 * l16;
        const uint2 w = stage[c][l16 ^ (c >> 3)];
        if (col < g.cols && row < g.rows) *reinterpret_cast<uint2*>(g.codes_t + col * g.pitch_t + row) = w;
    }
}

// ---- 16-bit inputs: the tile stays packed, two values to a register, and so do the maxima --------------------------------
template <int DT> __device__ __forceinline__ uint32_t max2_nan(uint32_t a, uint32_t b) {
    uint32_t r;
    if (DT == DT_BF16) asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
template <int DT> __device__ __forceinline__ void unpack16(uint32_t w, float& lo, float& hi) {
    if (DT == DT_BF16) {
        lo = __uint_as_float(w << 16);
        hi = __uint_as_float(w & 0xffff0000u);
    } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
        lo = f.x;
        hi = f.y;
    }
}
template <int DT> __device__ __forceinline__ float max_of_pair(uint32_t w) {
    float lo, hi;
    unpack16<DT>(w, lo, hi);
    return max_nan(lo, hi);
}
template <bool E5M2>
__device__ __forceinline__ uint32_t code2_scaled(float lo, float hi, uint64_t r) {
    ptx::unpack2f(ptx::mul2(ptx::pack2f(lo, hi), r), lo, hi);
    return code2<E5M2>(lo, hi);
}

// The work of fp8_quantize_kernel with 64 instead of 106 registers a thread, so that four CTAs share an SM and one loads
// while another reduces or stores.  Both directions of a bf16 tensor, at 2 + 2 bytes a value: 8192 x 4096 27.8 us (0.74 of the
// copy rate; 51 us with fp32 values in registers and two CTAs an SM), 16384 x 8192 96 us (0.85); one direction of the
// latter 63 us (0.97).
template <int DT, bool E5M2, bool TILE>
__global__ void __launch_bounds__(256, 4) fp8_quantize16_kernel(const QuantArgs g) {
    __shared__ uint32_t col_part[8][64];        // per-warp column maxima, two columns to a word
    __shared__ float col_sum[8][128];
    __shared__ float warp_part[8];
    __shared__ float col_r[128];
    __shared__ uint2 stage[128][16];
    ptx::grid_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int l16 = lane & 15, h = lane >> 4;
    const int64_t cb = blockIdx.x % g.col_blocks, rb = blockIdx.x / g.col_blocks;
    const int64_t row0 = rb * 128 + 16 * warp + 8 * h, col0 = cb * 128 + 8 * l16;

    uint32_t w[8][4];
    const uint16_t* base = reinterpret_cast<const uint16_t*>(g.x) + row0 * g.stride + col0;
    const bool whole = g.vec && col0 + 8 <= g.cols;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if (row0 + i < g.rows && whole) {
            const uint4 q = __ldg(reinterpret_cast<const uint4*>(base + i * g.stride));
            w[i][0] = q.x; w[i][1] = q.y; w[i][2] = q.z; w[i][3] = q.w;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                w[i][j] = 0;
                if (row0 + i < g.rows && col0 + 2 * j < g.cols) w[i][j] = base[i * g.stride + 2 * j];
                if (row0 + i < g.rows && col0 + 2 * j + 1 < g.cols) w[i][j] |= (uint32_t)base[i * g.stride + 2 * j + 1] << 16;
            }
        }
    }
    if (g.colsum) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float s0 = 0.f, s1 = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float lo, hi;
                unpack16<DT>(w[i][j], lo, hi);
                s0 += lo;
                s1 += hi;
            }
            s0 += __shfl_xor_sync(0xffffffffu, s0, 16);
            s1 += __shfl_xor_sync(0xffffffffu, s1, 16);
            if (h == 0) *reinterpret_cast<float2*>(&col_sum[warp][8 * l16 + 2 * j]) = make_float2(s0, s1);
        }
    }
    // maxima of the thread's 8 rows (two halves to a word) and of its 4 pairs of columns
    uint32_t cmax[4];
    float mine = 0.f;                           // lane l16 = i < 8: the maximum of row i of this half warp
    if (TILE || g.codes) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            uint32_t m = w[i][0] & 0x7fff7fffu;
#pragma unroll
            for (int j = 1; j < 4; ++j) m = max2_nan<DT>(m, w[i][j] & 0x7fff7fffu);
            if (!TILE) {
#pragma unroll
                for (int s = 8; s > 0; s >>= 1) m = max2_nan<DT>(m, __shfl_xor_sync(0xffffffffu, m, s));
                if (l16 == i) mine = max_of_pair<DT>(m);
            } else {
                mine = max_nan(mine, max_of_pair<DT>(m));
            }
        }
    }
    float tile_r = 0.f;
    if (TILE) {
#pragma unroll
        for (int s = 16; s > 0; s >>= 1) mine = max_nan(mine, __shfl_xor_sync(0xffffffffu, mine, s));
        if (lane == 0) warp_part[warp] = mine;
        __syncthreads();
        mine = warp_part[0];
#pragma unroll
        for (int k = 1; k < 8; ++k) mine = max_nan(mine, warp_part[k]);
        const float sc = block_scale(mine, g.inv_top);
        tile_r = __fdiv_rn(1.f, sc);
        if (threadIdx.x == 0) {
            if (g.scales) g.scales[cb * g.row_blocks + rb] = sc;
            if (g.scales_t) g.scales_t[rb * g.col_blocks + cb] = sc;
        }
    } else if (g.codes_t) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            cmax[j] = w[0][j] & 0x7fff7fffu;
#pragma unroll
            for (int i = 1; i < 8; ++i) cmax[j] = max2_nan<DT>(cmax[j], w[i][j] & 0x7fff7fffu);
            cmax[j] = max2_nan<DT>(cmax[j], __shfl_xor_sync(0xffffffffu, cmax[j], 16));
        }
        if (h == 0) *reinterpret_cast<uint4*>(&col_part[warp][4 * l16]) = make_uint4(cmax[0], cmax[1], cmax[2], cmax[3]);
    }
    if (g.codes) {
        float r = tile_r;
        if (!TILE) {                            // one division a row, by the lane that holds its maximum
            const float sc = block_scale(mine, g.inv_top);
            r = __fdiv_rn(1.f, sc);
            if (l16 < 8 && row0 + l16 < g.rows) g.scales[cb * g.rows + row0 + l16] = sc;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float ri = TILE ? tile_r : __shfl_sync(0xffffffffu, r, (lane & 16) + i);
            const uint64_t r2 = ptx::pack2f(ri, ri);
            uint32_t c[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float lo, hi;
                unpack16<DT>(w[i][j], lo, hi);
                c[j] = code2_scaled<E5M2>(lo, hi, r2);
            }
            // whole 8-byte groups: the row pitch is a multiple of 16, so a group that starts inside the row ends inside it
            if (row0 + i < g.rows && col0 < g.cols)
                *reinterpret_cast<uint2*>(g.codes + (row0 + i) * g.pitch + col0) = make_uint2(c[0] | (c[1] << 16), c[2] | (c[3] << 16));
        }
    }
    if (!g.codes_t && !g.colsum) return;
    __syncthreads();
    if (threadIdx.x < 128) {
        const int64_t col = cb * 128 + threadIdx.x;
        if (g.codes_t && !TILE) {
            uint32_t m = col_part[0][threadIdx.x >> 1];
#pragma unroll
            for (int k = 1; k < 8; ++k) m = max2_nan<DT>(m, col_part[k][threadIdx.x >> 1]);
            float lo, hi;
            unpack16<DT>(m, lo, hi);
            const float sc = block_scale(threadIdx.x & 1 ? hi : lo, g.inv_top);
            col_r[threadIdx.x] = __fdiv_rn(1.f, sc);
            if (col < g.cols) g.scales_t[rb * g.cols + col] = sc;
        }
        if (g.colsum && col < g.cols) {
            float s = col_sum[0][threadIdx.x];
#pragma unroll
            for (int k = 1; k < 8; ++k) s += col_sum[k][threadIdx.x];
            g.colsum[rb * g.cols + col] = s;
        }
    }
    if (!g.codes_t) return;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int c = 8 * l16 + 2 * j;
        const float ra = TILE ? tile_r : col_r[c], rc = TILE ? tile_r : col_r[c + 1];
        const uint64_t r2 = ptx::pack2f(ra, rc);
        uint32_t a[2] = {0, 0}, b[2] = {0, 0};  // 8 codes of column c, of column c + 1
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            float l0, h0, l1, h1;
            unpack16<DT>(w[i][j], l0, h0);
            unpack16<DT>(w[i + 1][j], l1, h1);
            ptx::unpack2f(ptx::mul2(ptx::pack2f(l0, h0), r2), l0, h0);
            ptx::unpack2f(ptx::mul2(ptx::pack2f(l1, h1), r2), l1, h1);
            a[i >> 2] |= code2<E5M2>(l0, l1) << (8 * (i & 2));
            b[i >> 2] |= code2<E5M2>(h0, h1) << (8 * (i & 2));
        }
        stage[c][(2 * warp + h) ^ l16] = make_uint2(a[0], a[1]);
        stage[c + 1][(2 * warp + h) ^ l16] = make_uint2(b[0], b[1]);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int c = 16 * i + 2 * warp + h;
        const int64_t col = cb * 128 + c, row = rb * 128 + 8 * l16;
        const uint2 v = stage[c][l16 ^ (c >> 3)];
        if (col < g.cols && row < g.rows) *reinterpret_cast<uint2*>(g.codes_t + col * g.pitch_t + row) = v;
    }
}

// Column sums of part [n, pitch]: 32 columns a CTA, each of its WARPS warps adds every WARPS-th row (four at a time in flight),
// and the warps' sums are added in order.  Many rows need many warps (1184 x 2002, bound by the latency of a warp's loads one
// after the other: 8.2 us with 8 warps, 5.4 us with 32), few do not (148 x 16384: 4.5 us with 8, 6.7 us with 32).
template <int DT, int WARPS>
__global__ void __launch_bounds__(32 * WARPS)
sum_partials_kernel(const float* part, int64_t n, int64_t cols, int64_t pitch, void* out0, void* out1) {
    const int set = blockIdx.y;
    void* out = set ? out1 : out0;
    const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t c = (int64_t)blockIdx.x * 32 + lane;
    __shared__ float s[WARPS][32];
    if (!out) return;
    const float* p = part + set * cols + c;
    float a[4] = {0.f, 0.f, 0.f, 0.f};
    if (c < cols) {
        int64_t i = w;
        for (; i + 3 * WARPS < n; i += 4 * WARPS) {
#pragma unroll
            for (int j = 0; j < 4; ++j) a[j] += p[(i + WARPS * j) * pitch];
        }
        for (; i < n; i += WARPS) a[0] += p[i * pitch];
    }
    s[w][lane] = (a[0] + a[1]) + (a[2] + a[3]);
    __syncthreads();
    if (w == 0 && c < cols) {
        float v = s[0][lane];
#pragma unroll
        for (int i = 1; i < WARPS; ++i) v += s[i][lane];
        store1<DT>(out, c, v);
    }
}

int sum_partials(const float* part, int64_t n, int64_t cols, int sets, void* out0, void* out1, int dtype, cudaStream_t st) {
    if (cols <= 0) return MXQ_OK;
    const int64_t grid = (cols + 31) / 32;
    if (grid > 0x7fffffff) return MXQ_ERR_TOO_LARGE;
    const dim3 g((unsigned)grid, (unsigned)sets);
    const int64_t pitch = sets * cols;
#define MXQ_SUM(DT) (n > 512 ? sum_partials_kernel<DT, 32><<<g, 1024, 0, st>>>(part, n, cols, pitch, out0, out1) \
                             : sum_partials_kernel<DT, 8><<<g, 256, 0, st>>>(part, n, cols, pitch, out0, out1))
    if (dtype == MXQ_F32) MXQ_SUM(DT_F32);
    else if (dtype == MXQ_F16) MXQ_SUM(DT_F16);
    else if (dtype == MXQ_BF16) MXQ_SUM(DT_BF16);
    else return MXQ_ERR_BAD_ARG;
#undef MXQ_SUM
    return check_launch();
}

}  // namespace mxq

extern "C" int mxq_fp8_quantize(const void* x, int dtype, int64_t rows, int64_t cols, int64_t row_stride, int fmt, int tile,
                                void* codes, int64_t codes_pitch, float* scales, void* codes_t, int64_t codes_t_pitch,
                                float* scales_t, float* colsum, void* stream) {
    using namespace mxq;
    if (rows < 0 || cols < 0 || fmt < 0 || fmt > 1 || dtype < 0 || dtype > 2) return MXQ_ERR_BAD_ARG;
    if (rows == 0 || cols == 0) return MXQ_OK;
    if (!x || row_stride < cols || (!codes && !codes_t) || (codes && !scales) || (codes_t && !scales_t)) return MXQ_ERR_BAD_ARG;
    if (codes && (codes_pitch < cols || codes_pitch % 16 || !aligned16(codes))) return MXQ_ERR_ALIGN;
    if (codes_t && (codes_t_pitch < rows || codes_t_pitch % 16 || !aligned16(codes_t))) return MXQ_ERR_ALIGN;
    QuantArgs g;
    g.x = x; g.rows = rows; g.cols = cols; g.stride = row_stride;
    g.codes = (uint8_t*)codes; g.pitch = codes_pitch; g.scales = scales;
    g.codes_t = (uint8_t*)codes_t; g.pitch_t = codes_t_pitch; g.scales_t = scales_t; g.colsum = colsum;
    g.row_blocks = (rows + 127) / 128; g.col_blocks = (cols + 127) / 128;
    g.inv_top = fmt ? (float)(1.0 / 57344.0) : (float)(1.0 / 448.0);
    g.vec = aligned16(x) && (row_stride * dtype_size(dtype)) % 16 == 0;
    const int64_t grid = g.row_blocks * g.col_blocks;
    if (grid > 0x7fffffff) return MXQ_ERR_TOO_LARGE;
    cudaStream_t st = (cudaStream_t)stream;
    const int n = (int)grid;
    if (dtype == MXQ_F32) {
        if (fmt) fp8_quantize_kernel<true><<<n, 256, 0, st>>>(g, tile != 0);
        else fp8_quantize_kernel<false><<<n, 256, 0, st>>>(g, tile != 0);
        return check_launch();
    }
#define MXQ_LAUNCH(DT, TILE) (fmt ? fp8_quantize16_kernel<DT, true, TILE><<<n, 256, 0, st>>>(g) \
                                  : fp8_quantize16_kernel<DT, false, TILE><<<n, 256, 0, st>>>(g))
    if (dtype == MXQ_F16) { if (tile) MXQ_LAUNCH(DT_F16, true); else MXQ_LAUNCH(DT_F16, false); }
    else { if (tile) MXQ_LAUNCH(DT_BF16, true); else MXQ_LAUNCH(DT_BF16, false); }
#undef MXQ_LAUNCH
    return check_launch();
}

extern "C" int mxq_sum_partials(const float* part, int64_t n, int64_t cols, void* out, int dtype, void* stream) {
    if (n < 0 || cols < 0 || (cols > 0 && (!out || (n > 0 && !part)))) return MXQ_ERR_BAD_ARG;
    return mxq::sum_partials(part, n, cols, 1, out, nullptr, dtype, (cudaStream_t)stream);
}
