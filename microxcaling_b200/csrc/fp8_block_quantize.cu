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

template <int DT>
__device__ __forceinline__ void load8(const QuantArgs& g, int64_t row, int64_t col, float (&v)[8]) {
    using T = typename Store<DT>::T;
    const T* p = reinterpret_cast<const T*>(g.x) + row * g.stride + col;
    if (row < g.rows && col + 8 <= g.cols && g.vec) {
        uint32_t b[VecIO<DT, 16>::N];
        VecIO<DT, 16>::load(p, 0, b);
#pragma unroll
        for (int i = 0; i < VecIO<DT, 16>::N; ++i) v[i] = __uint_as_float(b[i]);
        if constexpr (DT == DT_F32) {
            VecIO<DT, 16>::load(p, 4, b);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[4 + i] = __uint_as_float(b[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (row < g.rows && col + i < g.cols) ? Store<DT>::load(p[i]) : 0.f;
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

template <int DT, bool E5M2>
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
    for (int i = 0; i < 8; ++i) load8<DT>(g, row0 + i, col0, v[i]);

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

// Column sums of part [n, pitch]: 32 columns a CTA, each of its 8 warps adds every eighth row (four at a time in flight),
// and the warps' sums are added in order.
template <int DT>
__global__ void __launch_bounds__(256)
sum_partials_kernel(const float* part, int64_t n, int64_t cols, int64_t pitch, void* out0, void* out1) {
    const int set = blockIdx.y;
    void* out = set ? out1 : out0;
    const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t c = (int64_t)blockIdx.x * 32 + lane;
    __shared__ float s[8][32];
    if (!out) return;
    const float* p = part + set * cols + c;
    float a[4] = {0.f, 0.f, 0.f, 0.f};
    if (c < cols) {
        int64_t i = w;
        for (; i + 24 < n; i += 32) {
#pragma unroll
            for (int j = 0; j < 4; ++j) a[j] += p[(i + 8 * j) * pitch];
        }
        for (; i < n; i += 8) a[0] += p[i * pitch];
    }
    s[w][lane] = (a[0] + a[1]) + (a[2] + a[3]);
    __syncthreads();
    if (w == 0 && c < cols) {
        float v = s[0][lane];
#pragma unroll
        for (int i = 1; i < 8; ++i) v += s[i][lane];
        store1<DT>(out, c, v);
    }
}

int sum_partials(const float* part, int64_t n, int64_t cols, int sets, void* out0, void* out1, int dtype, cudaStream_t st) {
    if (cols <= 0) return MXQ_OK;
    const int64_t grid = (cols + 31) / 32;
    if (grid > 0x7fffffff) return MXQ_ERR_TOO_LARGE;
    const dim3 g((unsigned)grid, (unsigned)sets);
    if (dtype == MXQ_F32) sum_partials_kernel<DT_F32><<<g, 256, 0, st>>>(part, n, cols, sets * cols, out0, out1);
    else if (dtype == MXQ_F16) sum_partials_kernel<DT_F16><<<g, 256, 0, st>>>(part, n, cols, sets * cols, out0, out1);
    else if (dtype == MXQ_BF16) sum_partials_kernel<DT_BF16><<<g, 256, 0, st>>>(part, n, cols, sets * cols, out0, out1);
    else return MXQ_ERR_BAD_ARG;
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
    const bool t = tile != 0;
#define MXQ_LAUNCH(DT) (fmt ? fp8_quantize_kernel<DT, true><<<(int)grid, 256, 0, st>>>(g, t) \
                            : fp8_quantize_kernel<DT, false><<<(int)grid, 256, 0, st>>>(g, t))
    if (dtype == MXQ_F32) MXQ_LAUNCH(DT_F32);
    else if (dtype == MXQ_F16) MXQ_LAUNCH(DT_F16);
    else MXQ_LAUNCH(DT_BF16);
#undef MXQ_LAUNCH
    return check_launch();
}

extern "C" int mxq_sum_partials(const float* part, int64_t n, int64_t cols, void* out, int dtype, void* stream) {
    if (n < 0 || cols < 0 || (cols > 0 && (!out || (n > 0 && !part)))) return MXQ_ERR_BAD_ARG;
    return mxq::sum_partials(part, n, cols, 1, out, nullptr, dtype, (cudaStream_t)stream);
}
