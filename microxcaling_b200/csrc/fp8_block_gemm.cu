// Product of 8-bit operands with an fp32 scale for each block of 128 along the contraction (sm_100a):
//
//     out[m, n] = sum over K blocks kb of  sa[kb, m] * sb[kb, n] * sum over k in kb of a[m, k] * b[n, k]   (+ bias[n])
//
// The inner sums are tcgen05.mma kind::f8f6f4 over 128 bytes of K, each started from zero into an accumulator of its own in
// tensor memory; the epilogue warps multiply it by the block's scales and add it to fp32 registers while the tensor core
// works on the next block.  (The tensor core can apply power-of-two scales itself, but not fp32 ones.)  So a sum of
// products is at most 128 long before it meets fp32 arithmetic on the ordinary cores.
//
// The tensor core's 128 rows are taken from b, so that the 32 lanes of an epilogue warp hold 32 consecutive n
// of one output row and a product with few rows (tokens of a decoding step) wastes nothing: a tile is 128 of b's rows
// x NT of a's rows, NT = 16 .. 128, and what has to be read then is b, once.  When the tiles do not fill the GPU the K blocks
// of a tile are split over the CTAs of a cluster (2, 4 or 8), which join their sums through distributed shared
// memory in the order of their ranks, so that results do not depend on timing.
#include <cuda.h>
#include <algorithm>
#include "fp8_block.cuh"
#include "mxq_common.cuh"
#include "sm100_ptx.cuh"
#include "tma_host.cuh"

namespace mxq {

__device__ int g_fp8_status;                       // MXQ_ERR_DEVICE once a kernel has given up on a wait

struct Fp8Gemm {
    const float* sp;                               // scales of the tensor core's row operand (b), [kb, sp_ld]
    const float* sq;                               // scales of its column operand (a), [kb, sq_ld]
    int64_t sp_ld, sq_ld;
    int sp_shift, sq_shift;                        // 0: a scale a row, 7: a scale for 128 rows
    void* out;                                     // [q, p], p contiguous
    const void* bias;                              // [p] or null
    int out_dtype, bias_dtype;
    int64_t P, Q, kb_total, p_tiles, q_tiles;
    int split;                                     // CTAs of a cluster that share a tile
    uint32_t idesc;
};

__device__ __forceinline__ float load_dyn(const void* p, int dtype, int64_t i) {
    if (dtype == DT_F32) return load1<DT_F32>(p, i);
    if (dtype == DT_F16) return load1<DT_F16>(p, i);
    return load1<DT_BF16>(p, i);
}
__device__ __forceinline__ void store_dyn(void* p, int dtype, int64_t i, float v) {
    if (dtype == DT_F32) store1<DT_F32>(p, i, v);
    else if (dtype == DT_F16) store1<DT_F16>(p, i, v);
    else store1<DT_BF16>(p, i, v);
}

template <int NT>
struct Fp8Tile {
    static constexpr int kWarps = NT >= 64 ? 8 : 4;           // epilogue warps: a lane quarter each, or half of its columns
    static constexpr int kCols = NT >= 64 ? NT / 2 : NT;      // columns of one epilogue warp
    static constexpr int kThreads = 64 + 32 * kWarps;
    static constexpr int kAcc = NT >= 128 ? 2 : 4;            // accumulators in tensor memory
    static constexpr int kTmemCols = kAcc * NT < 32 ? 32 : kAcc * NT;
    static constexpr int kP = 128 * 128, kQ = NT * 128;
    static constexpr int kStage = kP + kQ;
    static constexpr int kStages = NT >= 128 ? 6 : NT == 64 ? 4 : 5;
    static constexpr int kSum = NT * 128 * 4;                 // this CTA's sums, over the stages once they are done with
    static constexpr int kScaleOff = kStages * kStage > kSum ? kStages * kStage : kSum;
    static constexpr int kBarOff = kScaleOff + 2 * NT * 4;
    static constexpr int kTotal = kBarOff + 256 + 1024;
};

template <int NT>
__global__ void __launch_bounds__(Fp8Tile<NT>::kThreads)
fp8_gemm_kernel(const __grid_constant__ CUtensorMap tmap_p, const __grid_constant__ CUtensorMap tmap_q, const Fp8Gemm g) {
    using S = Fp8Tile<NT>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::kBarOff);    // [kStages]
    uint64_t* empty = full + S::kStages;                                // [kStages]
    uint64_t* acc_full = empty + S::kStages;                            // [kAcc]
    uint64_t* acc_empty = acc_full + S::kAcc;                           // [kAcc]
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + S::kAcc);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    float* q_scale = reinterpret_cast<float*>(smem + S::kScaleOff);     // [2][NT]
    float* sums = reinterpret_cast<float*>(smem);                       // [NT][128], after the main loop

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = g.split > 1 ? (int)ptx::cluster_ctarank() : 0;
    const int64_t tile = blockIdx.x / g.split;
    const int64_t pt = tile % g.p_tiles, qt = tile / g.p_tiles;
    const int64_t kb0 = g.kb_total * rank / g.split, kb1 = g.kb_total * (rank + 1) / g.split;

    if (threadIdx.x == 0) {
        for (int s = 0; s < S::kStages; ++s) { ptx::mbar_init(ptx::smem_u32(&full[s]), 1); ptx::mbar_init(ptx::smem_u32(&empty[s]), 1); }
        for (int b = 0; b < S::kAcc; ++b) { ptx::mbar_init(ptx::smem_u32(&acc_full[b]), 1); ptx::mbar_init(ptx::smem_u32(&acc_empty[b]), S::kWarps); }
        *abort_flag = 0;
        ptx::fence_mbar_init();
    }
    if (warp == 1) {
        ptx::tmem_alloc(ptx::smem_u32(tmem_slot), S::kTmemCols);
        ptx::tmem_relinquish();
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    if (warp == 0) {
        if (ptx::elect_one()) {
            uint32_t it = 0;
            bool ok = true;
            for (int64_t kb = kb0; kb < kb1; ++kb, ++it) {
                const int s = it % S::kStages;
                if (it >= (uint32_t)S::kStages && !ptx::mbar_wait(ptx::smem_u32(&empty[s]), ((it / S::kStages) & 1) ^ 1, abort_flag)) { ok = false; break; }
                const uint32_t bar = ptx::smem_u32(&full[s]), st = ptx::smem_u32(smem + s * S::kStage);
                ptx::mbar_expect_tx(bar, S::kStage);
                ptx::tma_load_2d(st, &tmap_p, bar, (int)(kb * 128), (int)(pt * 128));
                ptx::tma_load_2d(st + S::kP, &tmap_q, bar, (int)(kb * 128), (int)(qt * NT));
            }
            if (!ok)                               // give copies already in flight a bounded time to land
                for (int s = 0; s < S::kStages; ++s)
                    for (uint32_t i = 0; i < 4096 && !ptx::mbar_try_wait(ptx::smem_u32(&full[s]), 0) &&
                                         !ptx::mbar_try_wait(ptx::smem_u32(&full[s]), 1); ++i) __nanosleep(64);
        }
    } else if (warp == 1) {
        if (ptx::elect_one()) {
            uint32_t it = 0;
            for (int64_t kb = kb0; kb < kb1; ++kb, ++it) {
                const int s = it % S::kStages, b = it % S::kAcc;
                if (it >= (uint32_t)S::kAcc && !ptx::mbar_wait(ptx::smem_u32(&acc_empty[b]), ((it / S::kAcc) & 1) ^ 1, abort_flag)) break;
                if (!ptx::mbar_wait(ptx::smem_u32(&full[s]), (it / S::kStages) & 1, abort_flag)) break;
                ptx::tc_fence_after();
                const uint32_t pa = ptx::smem_u32(smem + s * S::kStage), qa = pa + S::kP;
#pragma unroll
                for (int k = 0; k < 4; ++k)        // 128-byte swizzle: a K step of 32 moves the start inside the atom
                    ptx::tc_mma_f8(tmem_base + b * NT, ptx::smem_desc(pa + 32 * k, 0, 1024, 2), ptx::smem_desc(qa + 32 * k, 0, 1024, 2),
                                   g.idesc, k > 0);
                ptx::tc_commit(ptx::smem_u32(&empty[s]));
                ptx::tc_commit(ptx::smem_u32(&acc_full[b]));
            }
        }
    } else {
        const int e = warp - 2, quarter = warp & 3, c0 = NT >= 64 ? (e >> 2) * S::kCols : 0;
        const int te = threadIdx.x - 64;                       // 0 .. 32 * kWarps - 1
        const int64_t p = pt * 128 + quarter * 32 + lane;
        const float* spp = g.sp + (min(p, g.P - 1) >> g.sp_shift);
        const bool loads_q = te < NT && qt * NT + te < g.Q;
        const float* sqp = g.sq + ((qt * NT + te) >> g.sq_shift);
        float acc[S::kCols];
#pragma unroll
        for (int i = 0; i < S::kCols; ++i) acc[i] = 0.f;
        float sp_next = 0.f, sq_next = 0.f;
        if (kb0 < kb1) {
            sp_next = __ldg(spp + kb0 * g.sp_ld);
            if (loads_q) sq_next = __ldg(sqp + kb0 * g.sq_ld);
        }
        uint32_t it = 0;
        for (int64_t kb = kb0; kb < kb1; ++kb, ++it) {
            const int b = it % S::kAcc;
            float* qs = q_scale + (it & 1) * NT;
            if (te < NT) qs[te] = sq_next;
            const float sp = sp_next;
            if (kb + 1 < kb1) {
                sp_next = __ldg(spp + (kb + 1) * g.sp_ld);
                if (loads_q) sq_next = __ldg(sqp + (kb + 1) * g.sq_ld);
            }
            asm volatile("bar.sync 1, %0;" ::"n"(32 * S::kWarps) : "memory");   // two buffers: a warp is at most one block ahead
            if (!ptx::mbar_wait(ptx::smem_u32(&acc_full[b]), (it / S::kAcc) & 1, abort_flag)) *abort_flag = 1;
            ptx::tc_fence_after();
            const uint32_t t = tmem_base + ((uint32_t)(quarter * 32) << 16) + b * NT + c0;
#pragma unroll
            for (int c = 0; c < S::kCols; c += 16) {
                uint32_t v[16];
                ptx::tmem_ld_32x32b_x16(t + c, v);
                ptx::tmem_ld_wait();
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[c + i] = __fmaf_rn(__uint_as_float(v[i]), sp * qs[c0 + c + i], acc[c + i]);
            }
            ptx::tc_fence_before();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&acc_empty[b]));
        }
        // every block of this CTA has been multiplied and every copy has landed: the stages are free
        asm volatile("bar.sync 1, %0;" ::"n"(32 * S::kWarps) : "memory");
#pragma unroll
        for (int i = 0; i < S::kCols; ++i) sums[(c0 + i) * 128 + quarter * 32 + lane] = acc[i];
    }
    __syncthreads();
    if (g.split > 1) { ptx::cluster_arrive(); ptx::cluster_wait(); }
    // each CTA of the cluster joins and writes its share of the tile's columns (output rows)
    if (!*abort_flag) {
        const int q_first = NT * rank / g.split, q_last = NT * (rank + 1) / g.split;
        for (int i = q_first * 128 + threadIdx.x; i < q_last * 128; i += S::kThreads) {
            const int64_t q = qt * NT + (i >> 7), p = pt * 128 + (i & 127);
            if (q >= g.Q) break;
            if (p >= g.P) continue;
            float v = 0.f;
            if (g.split > 1) {
                const uint32_t a = ptx::smem_u32(sums + i);
                for (int r = 0; r < g.split; ++r) v += ptx::ld_cluster_f32(ptx::mapa(a, r));
            } else {
                v = sums[i];
            }
            if (g.bias) v += load_dyn(g.bias, g.bias_dtype, p);
            store_dyn(g.out, g.out_dtype, q * g.P + p, v);
        }
    }
    ptx::tc_fence_before();
    __syncthreads();
    if (g.split > 1) { ptx::cluster_arrive(); ptx::cluster_wait(); }       // no CTA leaves while another reads its sums
    if (threadIdx.x == 0 && *abort_flag) atomicExch(&g_fp8_status, MXQ_ERR_DEVICE);
    if (warp == 1) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc(tmem_base, S::kTmemCols);
    }
}

// [rows, K] bytes with a row pitch; box = 128 bytes of K x box_rows rows, zero-filled outside
static int make_map(CUtensorMap* m, const void* base, int64_t rows, int64_t K, int64_t pitch, int box_rows) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return MXQ_ERR_CUDA;
    cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)pitch};
    cuuint32_t box[2] = {128, (cuuint32_t)box_rows};
    cuuint32_t estr[2] = {1, 1};
    return fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
               ? MXQ_OK : MXQ_ERR_CUDA;
}

template <int NT>
static int launch_fp8(const CUtensorMap& tp, const CUtensorMap& tq, const Fp8Gemm& g, cudaStream_t st) {
    using S = Fp8Tile<NT>;
    static_assert(S::kTotal <= 232448, "shared memory");
    auto kern = fp8_gemm_kernel<NT>;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kTotal) != cudaSuccess) { cudaGetLastError(); return MXQ_ERR_CUDA; }
    const int64_t grid = g.p_tiles * g.q_tiles * g.split;
    if (grid > 0x7fffffff) return MXQ_ERR_TOO_LARGE;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(S::kThreads);
    cfg.dynamicSmemBytes = S::kTotal;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = g.split; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, kern, tp, tq, g) != cudaSuccess) { cudaGetLastError(); return MXQ_ERR_CUDA; }
    return check_launch();
}

int fp8_gemm_status(int clear) {
    int v = 0;
    if (cudaMemcpyFromSymbol(&v, g_fp8_status, sizeof v) != cudaSuccess) { cudaGetLastError(); return MXQ_ERR_CUDA; }
    if (clear && v != 0) {
        const int zero = 0;
        cudaMemcpyToSymbol(g_fp8_status, &zero, sizeof zero);
    }
    return v;
}

}  // namespace mxq

extern "C" int mxq_fp8_gemm(const void* a, int64_t a_pitch, const float* a_scales, int a_tile, int a_fmt, const void* b,
                            int64_t b_pitch, const float* b_scales, int b_tile, int b_fmt, void* out, int out_dtype,
                            const void* bias, int bias_dtype, int64_t M, int64_t N, int64_t K, void* stream) {
    using namespace mxq;
    if (M < 0 || N < 0 || K <= 0 || a_fmt < 0 || a_fmt > 1 || b_fmt < 0 || b_fmt > 1) return MXQ_ERR_BAD_ARG;
    if (out_dtype < 0 || out_dtype > 2 || (bias && (bias_dtype < 0 || bias_dtype > 2))) return MXQ_ERR_BAD_ARG;
    if (M == 0 || N == 0) return MXQ_OK;
    if (!a || !b || !a_scales || !b_scales || !out || a_pitch < K || b_pitch < K) return MXQ_ERR_BAD_ARG;
    if (!aligned16(a) || !aligned16(b) || a_pitch % 16 || b_pitch % 16) return MXQ_ERR_ALIGN;
    if (M > 0x7fffff00 || N > 0x7fffff00 || K > 0x7fffff00) return MXQ_ERR_TOO_LARGE;
    const int nt = M <= 16 ? 16 : M <= 32 ? 32 : M <= 64 ? 64 : 128;
    Fp8Gemm g;
    g.sp = b_scales; g.sp_shift = b_tile ? 7 : 0; g.sp_ld = b_tile ? (N + 127) / 128 : N;
    g.sq = a_scales; g.sq_shift = a_tile ? 7 : 0; g.sq_ld = a_tile ? (M + 127) / 128 : M;
    g.out = out; g.out_dtype = out_dtype; g.bias = bias; g.bias_dtype = bias_dtype;
    g.P = N; g.Q = M; g.kb_total = (K + 127) / 128;
    g.p_tiles = (N + 127) / 128; g.q_tiles = (M + nt - 1) / nt;
    g.idesc = ptx::idesc_f8(b_fmt, a_fmt, 128, nt);
    // K blocks are split until every SM has a CTA, as long as each CTA keeps two of them
    g.split = 1;
    while (g.split < 8 && g.p_tiles * g.q_tiles * g.split < sm_count() && g.kb_total >= 4 * g.split) g.split *= 2;
    CUtensorMap tp, tq;
    int rc = make_map(&tp, b, N, K, b_pitch, 128);
    if (!rc) rc = make_map(&tq, a, M, K, a_pitch, nt);
    if (rc) return rc;
    g_launch_count[0].fetch_add(1, std::memory_order_relaxed);
    cudaStream_t st = (cudaStream_t)stream;
    if (nt == 16) return launch_fp8<16>(tp, tq, g, st);
    if (nt == 32) return launch_fp8<32>(tp, tq, g, st);
    if (nt == 64) return launch_fp8<64>(tp, tq, g, st);
    return launch_fp8<128>(tp, tq, g, st);
}

extern "C" int64_t mxq_fp8_linear_workspace_bytes(int64_t M, int64_t K) {
    if (M < 0 || K < 0) return -1;
    const int64_t pitch = (K + 15) / 16 * 16;
    return (M * pitch + 255) / 256 * 256 + (K + 127) / 128 * M * 4;
}

extern "C" int mxq_fp8_linear_fwd(const void* x, int x_dtype, int64_t x_stride, int x_fmt, const void* w, int64_t w_pitch,
                                  const float* w_scales, int w_tile, int w_fmt, void* y, int y_dtype, const void* bias,
                                  int bias_dtype, int64_t M, int64_t N, int64_t K, void* workspace, int64_t workspace_bytes,
                                  void* stream) {
    if (M < 0 || N < 0 || K <= 0) return MXQ_ERR_BAD_ARG;
    if (M == 0 || N == 0) return MXQ_OK;
    if (!workspace || workspace_bytes < mxq_fp8_linear_workspace_bytes(M, K)) return MXQ_ERR_BAD_ARG;
    if (reinterpret_cast<uintptr_t>(workspace) & 255) return MXQ_ERR_ALIGN;
    const int64_t pitch = (K + 15) / 16 * 16;
    float* scales = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + (M * pitch + 255) / 256 * 256);
    const int rc = mxq_fp8_quantize(x, x_dtype, M, K, x_stride, x_fmt, 0, workspace, pitch, scales, nullptr, 0, nullptr, nullptr, stream);
    if (rc) return rc;
    return mxq_fp8_gemm(workspace, pitch, scales, 0, x_fmt, w, w_pitch, w_scales, w_tile, w_fmt, y, y_dtype, bias, bias_dtype,
                        M, N, K, stream);
}

// ---------------------------------------------------------------------------------------------------------------
// A linear layer's training step as one call each way.  `saved` holds what the backward pass needs of the forward one's
// operands (x transposed for dw, w transposed for dx), `scratch` what only the running call needs.
// ---------------------------------------------------------------------------------------------------------------
namespace mxq {
struct Carve {                                     // hands out 256-byte aligned parts of one buffer
    uint8_t* base;
    int64_t used = 0;
    explicit Carve(void* p) : base(static_cast<uint8_t*>(p)) {}
    uint8_t* take(int64_t bytes) {
        uint8_t* p = base ? base + used : nullptr;
        used += (bytes + 255) / 256 * 256;
        return p;
    }
};
struct Operand8 { uint8_t* codes = nullptr; int64_t pitch = 0; float* scales = nullptr; };
static Operand8 carve_operand(Carve& c, int64_t rows, int64_t K, bool tile) {
    Operand8 o;
    o.pitch = (K + 15) / 16 * 16;
    o.codes = c.take(rows * o.pitch);
    o.scales = reinterpret_cast<float*>(c.take(4 * ((K + 127) / 128) * (tile ? (rows + 127) / 128 : rows)));
    return o;
}
struct Saved8 { Operand8 xt, wt; int64_t bytes; };
static Saved8 carve_saved(void* p, int64_t M, int64_t N, int64_t K, int need_dx, int need_dw) {
    Carve c(p);
    Saved8 s;
    if (need_dw) s.xt = carve_operand(c, K, M, false);
    if (need_dx) s.wt = carve_operand(c, K, N, true);
    s.bytes = c.used;
    return s;
}
struct Scratch8 { Operand8 x, w; int64_t bytes; };
static Scratch8 carve_fwd(void* p, int64_t M, int64_t N, int64_t K) {
    Carve c(p);
    Scratch8 s;
    s.x = carve_operand(c, M, K, false);
    s.w = carve_operand(c, N, K, true);
    s.bytes = c.used;
    return s;
}
struct Grads8 { Operand8 dy, dyt; float* sums; int64_t bytes; };
static Grads8 carve_bwd(void* p, int64_t M, int64_t N, int64_t K) {
    Carve c(p);
    Grads8 s;
    s.dy = carve_operand(c, M, N, false);
    s.dyt = carve_operand(c, N, M, false);
    s.sums = reinterpret_cast<float*>(c.take(4 * ((M + 127) / 128) * N));
    s.bytes = c.used;
    return s;
}
}  // namespace mxq

extern "C" int64_t mxq_fp8_linear_saved_bytes(int64_t M, int64_t N, int64_t K, int need_dx, int need_dw) {
    return M < 0 || N < 0 || K < 0 ? -1 : mxq::carve_saved(nullptr, M, N, K, need_dx, need_dw).bytes;
}
extern "C" int64_t mxq_fp8_linear_scratch_bytes(int64_t M, int64_t N, int64_t K, int backward) {
    if (M < 0 || N < 0 || K < 0) return -1;
    return backward ? mxq::carve_bwd(nullptr, M, N, K).bytes : mxq::carve_fwd(nullptr, M, N, K).bytes;
}

extern "C" int mxq_fp8_linear_fwd_train(const void* x, int x_dtype, int64_t x_stride, const void* w, int w_dtype, int64_t w_stride,
                                        int fmt, const void* bias, int bias_dtype, void* y, int y_dtype, int need_dx, int need_dw,
                                        void* saved, int64_t saved_bytes, void* scratch, int64_t scratch_bytes, int64_t M, int64_t N,
                                        int64_t K, void* stream) {
    using namespace mxq;
    if (M <= 0 || N <= 0 || K <= 0 || !scratch || ((need_dx || need_dw) && !saved)) return MXQ_ERR_BAD_ARG;
    if ((reinterpret_cast<uintptr_t>(scratch) | reinterpret_cast<uintptr_t>(saved)) & 255) return MXQ_ERR_ALIGN;
    const Scratch8 q = carve_fwd(scratch, M, N, K);
    const Saved8 s = carve_saved(saved, M, N, K, need_dx, need_dw);
    if (scratch_bytes < q.bytes || saved_bytes < s.bytes) return MXQ_ERR_BAD_ARG;
    int rc = mxq_fp8_quantize(x, x_dtype, M, K, x_stride, fmt, 0, q.x.codes, q.x.pitch, q.x.scales, s.xt.codes, s.xt.pitch, s.xt.scales,
                              nullptr, stream);
    if (rc) return rc;
    rc = mxq_fp8_quantize(w, w_dtype, N, K, w_stride, fmt, 1, q.w.codes, q.w.pitch, q.w.scales, s.wt.codes, s.wt.pitch, s.wt.scales,
                          nullptr, stream);
    if (rc) return rc;
    return mxq_fp8_gemm(q.x.codes, q.x.pitch, q.x.scales, 0, fmt, q.w.codes, q.w.pitch, q.w.scales, 1, fmt, y, y_dtype, bias, bias_dtype,
                        M, N, K, stream);
}

extern "C" int mxq_fp8_linear_bwd(const void* dy, int dy_dtype, int64_t dy_stride, int grad_fmt, int fmt, const void* saved,
                                  int64_t saved_bytes, int saved_dx, int saved_dw, void* dx, int dx_dtype, void* dw, int dw_dtype,
                                  void* db, int db_dtype, void* scratch, int64_t scratch_bytes, int64_t M, int64_t N, int64_t K,
                                  void* stream) {
    using namespace mxq;
    if (M <= 0 || N <= 0 || K <= 0 || (dx && !saved_dx) || (dw && !saved_dw)) return MXQ_ERR_BAD_ARG;
    if (!dx && !dw && !db) return MXQ_OK;
    if (!scratch || ((dx || dw) && !saved)) return MXQ_ERR_BAD_ARG;
    if ((reinterpret_cast<uintptr_t>(scratch) | reinterpret_cast<uintptr_t>(saved)) & 255) return MXQ_ERR_ALIGN;
    const Grads8 q = carve_bwd(scratch, M, N, K);
    const Saved8 s = carve_saved(const_cast<void*>(saved), M, N, K, saved_dx, saved_dw);
    if (scratch_bytes < q.bytes || ((dx || dw) && saved_bytes < s.bytes)) return MXQ_ERR_BAD_ARG;
    int rc = mxq_fp8_quantize(dy, dy_dtype, M, N, dy_stride, grad_fmt, 0, dx || !dw ? q.dy.codes : nullptr, q.dy.pitch, q.dy.scales,
                              dw ? q.dyt.codes : nullptr, q.dyt.pitch, q.dyt.scales, db ? q.sums : nullptr, stream);
    if (!rc && dx)
        rc = mxq_fp8_gemm(q.dy.codes, q.dy.pitch, q.dy.scales, 0, grad_fmt, s.wt.codes, s.wt.pitch, s.wt.scales, 1, fmt, dx, dx_dtype,
                          nullptr, 0, M, K, N, stream);
    if (!rc && dw)
        rc = mxq_fp8_gemm(q.dyt.codes, q.dyt.pitch, q.dyt.scales, 0, grad_fmt, s.xt.codes, s.xt.pitch, s.xt.scales, 0, fmt, dw, dw_dtype,
                          nullptr, 0, N, K, M, stream);
    if (!rc && db) rc = mxq_sum_partials(q.sums, (M + 127) / 128, N, db, db_dtype, stream);
    return rc;
}
