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
// of a tile are split over the CTAs of a cluster (2, 4 or 8): each sends its sums to the CTA that owns those output rows, through
// distributed shared memory, and the owner adds them in the order of the ranks, so that results do not depend on timing.
#include <cuda.h>
#include <math.h>
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
    int early;                                     // launched while the kernel that writes a's operand may still run
    uint32_t idesc;
};

// After a wait that gave up: the status word, and a millisecond in which copies still in flight land before the CTA leaves.
__device__ __forceinline__ void give_up(int aborted) {
    if (!aborted) return;
    atomicExch(&g_fp8_status, MXQ_ERR_DEVICE);
    for (int i = 0; i < 64; ++i) __nanosleep(16384);
}

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

__device__ __forceinline__ uint32_t pack2(float lo, float hi, int dtype) {
    if (dtype == DT_BF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// four consecutive values of an output row, bias added; `whole`: rows are a multiple of four values long
__device__ __forceinline__ void store4(const Fp8Gemm& g, int64_t row, int64_t p, float4 f, bool whole) {
    float v[4] = {f.x, f.y, f.z, f.w};
    if (g.bias) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (p + j < g.P) v[j] += load_dyn(g.bias, g.bias_dtype, p + j);
    }
    if (!whole) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (p + j < g.P) store_dyn(g.out, g.out_dtype, row + p + j, v[j]);
    } else if (g.out_dtype == DT_F32) {
        *reinterpret_cast<float4*>(reinterpret_cast<float*>(g.out) + row + p) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
        *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(g.out) + row + p) =
            make_uint2(pack2(v[0], v[1], g.out_dtype), pack2(v[2], v[3], g.out_dtype));
    }
}

template <int NT, bool SPLIT>
struct Fp8Tile {
    static constexpr int kWarps = NT >= 64 ? 8 : 4;           // epilogue warps: a lane quarter each, or half of its columns
    static constexpr int kCols = NT >= 64 ? NT / 2 : NT;      // columns of one epilogue warp
    static constexpr int kThreads = 64 + 32 * kWarps;
    static constexpr int kAcc = NT >= 128 ? 2 : 4;            // accumulators in tensor memory
    static constexpr int kTmemCols = kAcc * NT < 32 ? 32 : kAcc * NT;
    static constexpr int kP = 128 * 128, kQ = NT * 128;
    static constexpr int kStage = kP + kQ;
    // As many stages as let two CTAs live on an SM (one with NT = 128).  Sums from other CTAs need memory of their own, beside
    // the stages that may still be in use; a CTA that has the tile to itself passes its sums through the stages.
    static constexpr int kStages = NT == 128 ? (SPLIT ? 4 : 6) : NT == 64 ? (SPLIT ? 3 : 4) : NT == 32 ? (SPLIT ? 4 : 5) : (SPLIT ? 5 : 6);
    static constexpr int kJoinOff = SPLIT ? kStages * kStage : 0;   // [rank][own columns][128] sums sent to this CTA
    static constexpr int kScaleOff = kStages * kStage + (SPLIT ? NT * 128 * 4 : 0);
    static_assert(NT * 128 * 4 <= kStages * kStage, "the sums fit into the stages");
    static constexpr int kBarOff = kScaleOff + 2 * NT * 4;
    static constexpr int kTotal = kBarOff + 256 + 1024;
};

template <int NT, bool SPLIT>
__global__ void __launch_bounds__(Fp8Tile<NT, SPLIT>::kThreads)
fp8_gemm_kernel(const __grid_constant__ CUtensorMap tmap_p, const __grid_constant__ CUtensorMap tmap_q, const Fp8Gemm g) {
    using S = Fp8Tile<NT, SPLIT>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::kBarOff);    // [kStages]
    uint64_t* empty = full + S::kStages;                                // [kStages]
    uint64_t* acc_full = empty + S::kStages;                            // [kAcc]
    uint64_t* acc_empty = acc_full + S::kAcc;                           // [kAcc]
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + S::kAcc);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    float* q_scale = reinterpret_cast<float*>(smem + S::kScaleOff);     // [2][NT]
    float* join = reinterpret_cast<float*>(smem + S::kJoinOff);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = SPLIT ? (int)ptx::cluster_ctarank() : 0;
    const uint32_t tile = blockIdx.x / g.split;
    const int64_t pt = tile / (uint32_t)g.q_tiles, qt = tile % (uint32_t)g.q_tiles;   // tiles that share rows of b side by side
    const int blocks = (int)g.kb_total, kb0 = blocks * rank / g.split, n_kb = blocks * (rank + 1) / g.split - kb0;

    // The producer's thread makes the barriers and sends for the first stages before anyone else is ready.
    const bool producer = warp == 0 && ptx::elect_one();
    auto load_p = [&](int i) {
        const int s = i % S::kStages;
        const uint32_t bar = ptx::smem_u32(&full[s]);
        ptx::mbar_expect_tx(bar, S::kStage);
        ptx::tma_load_2d(ptx::smem_u32(smem + s * S::kStage), &tmap_p, bar, (kb0 + i) * 128, (int)(pt * 128));
    };
    auto load_q = [&](int i) {
        const int s = i % S::kStages;
        ptx::tma_load_2d(ptx::smem_u32(smem + s * S::kStage + S::kP), &tmap_q, ptx::smem_u32(&full[s]), (kb0 + i) * 128, (int)(qt * NT));
    };
    if (producer) {
        for (int s = 0; s < S::kStages; ++s) { ptx::mbar_init(ptx::smem_u32(&full[s]), 1); ptx::mbar_init(ptx::smem_u32(&empty[s]), 1); }
        for (int b = 0; b < S::kAcc; ++b) { ptx::mbar_init(ptx::smem_u32(&acc_full[b]), 1); ptx::mbar_init(ptx::smem_u32(&acc_empty[b]), S::kWarps); }
        *abort_flag = 0;
        ptx::fence_mbar_init();
        ptx::fence_proxy_async();
        const int ahead = min((int)S::kStages, n_kb);
        for (int i = 0; i < ahead; ++i) load_p(i);
        if (g.early) ptx::grid_wait();                        // b was there before the kernel in front of this one began, a was not
        for (int i = 0; i < ahead; ++i) load_q(i);
    }
    if (warp == 1) {
        ptx::tmem_alloc(ptx::smem_u32(tmem_slot), S::kTmemCols);
        ptx::tmem_relinquish();
    }
    __syncwarp();
    ptx::tc_fence_before();
    __syncthreads();
    if constexpr (SPLIT) ptx::cluster_arrive();                   // waited for before the first store to another CTA's memory
    ptx::tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    if (warp == 0) {
        if (producer) {
            for (int i = S::kStages; i < n_kb; ++i) {
                if (!ptx::mbar_wait(ptx::smem_u32(&empty[i % S::kStages]), ((i / S::kStages) & 1) ^ 1, abort_flag)) break;
                load_p(i);
                load_q(i);
            }
        }
        __syncwarp();
        if constexpr (SPLIT) ptx::cluster_wait();
    } else if (warp == 1) {
        if (ptx::elect_one()) {
            for (int it = 0; it < n_kb; ++it) {
                const int s = it % S::kStages, b = it % S::kAcc;
                if (it >= S::kAcc && !ptx::mbar_wait(ptx::smem_u32(&acc_empty[b]), ((it / S::kAcc) & 1) ^ 1, abort_flag)) break;
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
        __syncwarp();
        if constexpr (SPLIT) ptx::cluster_wait();
    } else {
        const int e = warp - 2, quarter = warp & 3, c0 = NT >= 64 ? (e >> 2) * S::kCols : 0;
        const int te = threadIdx.x - 64;                       // 0 .. 32 * kWarps - 1
        const int64_t p = pt * 128 + quarter * 32 + lane;
        const float* spp = g.sp + (min(p, g.P - 1) >> g.sp_shift) + kb0 * g.sp_ld;
        const bool loads_q = te < NT && qt * NT + te < g.Q;
        const float* sqp = g.sq + ((qt * NT + te) >> g.sq_shift) + kb0 * g.sq_ld;
        float acc[S::kCols];
#pragma unroll
        for (int i = 0; i < S::kCols; ++i) acc[i] = 0.f;
        float sp_next = 0.f, sq_next = 0.f;
        if (g.early) ptx::grid_wait();                         // a's scales; and the output may not be written before
        if (n_kb > 0) {
            sp_next = __ldg(spp);
            if (loads_q) sq_next = __ldg(sqp);
        }
        for (int it = 0; it < n_kb; ++it) {
            const int b = it % S::kAcc;
            float* qs = q_scale + (it & 1) * NT;
            if (te < NT) qs[te] = sq_next;
            const float sp = sp_next;
            if (it + 1 < n_kb) {
                sp_next = __ldg(spp += g.sp_ld);
                if (loads_q) sq_next = __ldg(sqp += g.sq_ld);
            }
            asm volatile("bar.sync 1, %0;" ::"n"(32 * S::kWarps) : "memory");   // two buffers: a warp is at most one block ahead
            ptx::mbar_wait(ptx::smem_u32(&acc_full[b]), (it / S::kAcc) & 1, abort_flag);   // a wait that gives up raises the flag
            ptx::tc_fence_after();
            const uint32_t t = tmem_base + ((uint32_t)(quarter * 32) << 16) + b * NT + c0;
#pragma unroll
            for (int c = 0; c < S::kCols; c += 16) {
                uint32_t v[16];
                ptx::tmem_ld_32x32b_x16(t + c, v);
                ptx::tmem_ld_wait();
                if (c + 16 == S::kCols) {                      // the accumulator is out of tensor memory
                    ptx::tc_fence_before();
                    __syncwarp();
                    if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&acc_empty[b]));
                }
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                    const float4 q = *reinterpret_cast<const float4*>(qs + c0 + c + i);
                    acc[c + i] = __fmaf_rn(__uint_as_float(v[i]), sp * q.x, acc[c + i]);
                    acc[c + i + 1] = __fmaf_rn(__uint_as_float(v[i + 1]), sp * q.y, acc[c + i + 1]);
                    acc[c + i + 2] = __fmaf_rn(__uint_as_float(v[i + 2]), sp * q.z, acc[c + i + 2]);
                    acc[c + i + 3] = __fmaf_rn(__uint_as_float(v[i + 3]), sp * q.w, acc[c + i + 3]);
                }
            }
        }
        // send the sums to the CTAs that own their columns (output rows): [rank][own column][128]
        const int own = NT / g.split;                          // a power of two
        const int shift = __ffs(own) - 1;
        const uint32_t mine = ptx::smem_u32(join) + 4 * (rank * own * 128 + quarter * 32 + lane);
        if constexpr (SPLIT) {
            ptx::cluster_wait();                               // the other CTAs are there
#pragma unroll
            for (int i = 0; i < S::kCols; ++i) {
                const int c = c0 + i;
                ptx::st_cluster_f32(ptx::mapa(mine, c >> shift) + (c & (own - 1)) * 512, acc[i]);
            }
        } else {
            asm volatile("bar.sync 1, %0;" ::"n"(32 * S::kWarps) : "memory");   // the last block has been multiplied: the stages are free
#pragma unroll
            for (int i = 0; i < S::kCols; ++i) join[(c0 + i) * 128 + quarter * 32 + lane] = acc[i];
        }
    }
    if constexpr (SPLIT) { __syncwarp(); ptx::cluster_arrive(); ptx::cluster_wait(); }
    else __syncthreads();
    // join and write this CTA's columns, four consecutive values of an output row a thread
    if (!*abort_flag) {
        const int own = NT / g.split;
        const bool whole = g.P % 4 == 0;
        for (int i = threadIdx.x * 4; i < own * 128; i += S::kThreads * 4) {
            const int64_t q = qt * NT + rank * own + (i >> 7), p = pt * 128 + (i & 127);
            if (q >= g.Q) break;
            if (p >= g.P) continue;
            float4 v = *reinterpret_cast<const float4*>(join + i);
            for (int r = 1; r < g.split; ++r) {
                const float4 o = *reinterpret_cast<const float4*>(join + r * own * 128 + i);
                v.x += o.x; v.y += o.y; v.z += o.z; v.w += o.w;
            }
            store4(g, q * g.P, p, v, whole);
        }
    }
    ptx::tc_fence_before();
    __syncthreads();
    if (threadIdx.x == 0) give_up(*abort_flag);
    if (warp == 1) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc(tmem_base, S::kTmemCols);
    }
}

// ---------------------------------------------------------------------------------------------------------------
// Large products: CTA pairs (cta_group::2) on 256 x 256 tiles, persistent.  The tensor core's rows are a's here.  Each CTA
// stages its own 128 rows of a and its half of b's 256 rows (32 KB a K block, five of them in flight), the even CTA issues the
// MMAs for both, and every CTA's eight epilogue warps hold 128 x 256 fp32 sums in registers, 128 a thread.
// The two accumulators of 256 columns fill tensor memory: while the warps scale and add one block's sums the tensor core
// works on the next one.  Beside its 512 cycles a block (128 x 256 x 128 at the peak rate on each SM) stand 32768 fused
// multiply-adds, 256 cycles of the fp32 pipes (twice that with a scale for every row of b as well, B_ROWS: weight gradients).
//
// Measured: 8192 x 4096 x 4096 135 to 145 us (1.9 to 2.0 PFLOP/s), 16384 x 28672 x 8192 3.4 ms (2.25 PFLOP/s, SM clock near
// 1.4 GHz under the power cap); with B_ROWS 4096 x 4096 x 8192 259 us (1.06 PFLOP/s; 281 us when every thread held one row and
// read all column scales).  With the scaling left out the same loop takes 119 us and 2.7 ms: the rest is the hand-over of the accumulators
// (two of them, a round trip of a block's MMAs, drain and arrival each), not the arithmetic.  Tried and dropped: a release
// fence at that hand-over (299 instead of 181 us at that stage), halves of an accumulator handed over apart (194 to 177), the
// block loop unrolled twice (3.5 -> 4.0 ms at the large size), column scales kept in registers across rows (259 -> 325 us: spills).
// ---------------------------------------------------------------------------------------------------------------
struct Fp8Pair {
    const float* sa;
    const float* sb;
    int64_t sa_ld, sb_ld;
    int sa_shift, sb_shift;
    void* out;                                     // [M, N]
    const void* bias;                              // [N] or null
    int out_dtype, bias_dtype, tma_out;
    int64_t M, N, kb_total, m_tiles, n_tiles;
    uint32_t idesc;
};

template <bool B_ROWS>
struct Fp8PairSmem {
    static constexpr int kStages = 5;
    static constexpr int kBoxes = B_ROWS ? 1 : 2;              // b's scales leave no room for a second one
    static constexpr int kA = 128 * 128, kStage = 2 * kA;
    static constexpr int kStgOff = kStages * kStage;           // boxes of 32 rows x 128 bytes for each epilogue warp
    static constexpr int kScaleOff = kStgOff + 8 * kBoxes * 4096;       // b's scales of two blocks
    static constexpr int kBarOff = kScaleOff + (B_ROWS ? 2 * 256 * 4 : 0);
    static constexpr int kTotal = kBarOff + 256 + 1024;
    static_assert(kTotal <= 232448, "shared memory");
};

// Tiles are walked in groups of 16 tile rows, column by column, so that CTAs at work at the same time share panels in L2.
__device__ __forceinline__ void pair_tile(int64_t t, const Fp8Pair& g, int64_t& mt, int64_t& nt) {
    const uint32_t per = 16 * (uint32_t)g.n_tiles, grp = (uint32_t)t / per, i = (uint32_t)t % per;
    const uint32_t rows = min(16u, (uint32_t)g.m_tiles - grp * 16);
    mt = grp * 16 + i % rows;
    nt = i / rows;
}

// acc += (two sums of a block) * (their scales)
__device__ __forceinline__ void scale_add(float2& acc, uint32_t lo, uint32_t hi, uint64_t scale) {
    uint64_t x = ptx::pack2f(acc.x, acc.y);
    ptx::fma2(x, ptx::pack2f(lo, hi), scale);
    ptx::unpack2f(x, acc.x, acc.y);
}

template <bool B_ROWS, bool F32>
__global__ void __launch_bounds__(384, 1)
fp8_gemm_pair_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                     const __grid_constant__ CUtensorMap tmap_c, const Fp8Pair g) {
    using S = Fp8PairSmem<B_ROWS>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::kBarOff);    // [kStages], the even CTA's
    uint64_t* empty = full + S::kStages;                                // [kStages], one in each CTA
    uint64_t* acc_full = empty + S::kStages;                            // [2], one in each CTA
    uint64_t* acc_empty = acc_full + 2;                                 // [2], the even CTA's
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    float* b_scale = reinterpret_cast<float*>(smem + S::kScaleOff);     // [2][256]

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = ptx::cluster_ctarank();
    if (threadIdx.x == 0) {
        for (int s = 0; s < S::kStages; ++s) { ptx::mbar_init(ptx::smem_u32(&full[s]), 1); ptx::mbar_init(ptx::smem_u32(&empty[s]), 1); }
        for (int b = 0; b < 2; ++b) { ptx::mbar_init(ptx::smem_u32(&acc_full[b]), 1); ptx::mbar_init(ptx::smem_u32(&acc_empty[b]), 16); }
        *abort_flag = 0;
        ptx::fence_mbar_init();
    }
    if (warp == 1) {
        ptx::tmem_alloc_pair(ptx::smem_u32(tmem_slot), 512);
        ptx::tmem_relinquish_pair();
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::cluster_arrive();                                    // both CTAs' barriers exist before anyone signals them
    ptx::cluster_wait();
    ptx::tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    const int64_t total = g.m_tiles * g.n_tiles, pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

    // Registers: 384 threads are launched with 168 each (64512); the first warpgroup (producer, MMA issuer, two idle warps)
    // keeps 40 and the epilogue's two take 232 each, 64512 in all.
    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
        if (warp == 0 && ptx::elect_one()) {
            ptx::prefetch_tmap(&tmap_a);
            ptx::prefetch_tmap(&tmap_b);
            uint32_t it = 0;
            bool ok = true;
            for (int64_t t = pair; t < total && ok; t += pairs) {
                int64_t mt, nt;
                pair_tile(t, g, mt, nt);
                const int row_a = (int)(mt * 256 + rank * 128), row_b = (int)(nt * 256 + rank * 128);
                for (int64_t kb = 0; kb < g.kb_total; ++kb, ++it) {
                    const int s = it % S::kStages;
                    if (it >= (uint32_t)S::kStages && !ptx::mbar_wait(ptx::smem_u32(&empty[s]), ((it / S::kStages) & 1) ^ 1, abort_flag)) { ok = false; break; }
                    if (rank == 0) ptx::mbar_expect_tx(ptx::smem_u32(&full[s]), 2 * S::kStage);
                    const uint32_t bar = ptx::mapa(ptx::smem_u32(&full[s]), 0), st = ptx::smem_u32(smem + s * S::kStage);
                    ptx::tma_load_2d_pair(st, &tmap_a, bar, (int)(kb * 128), row_a);
                    ptx::tma_load_2d_pair(st + S::kA, &tmap_b, bar, (int)(kb * 128), row_b);
                }
            }
        }
        if (warp == 1 && rank == 0 && ptx::elect_one()) {
            const uint64_t desc = ptx::smem_desc(ptx::smem_u32(smem), 0, 1024, 2);
            uint32_t it = 0;
            bool ok = true;
            for (int64_t t = pair; t < total && ok; t += pairs) {
                for (int64_t kb = 0; kb < g.kb_total; ++kb, ++it) {
                    const int s = it % S::kStages;
                    const uint32_t b = it & 1;
                    if (!ptx::mbar_wait(ptx::smem_u32(&full[s]), (it / S::kStages) & 1, abort_flag)) { ok = false; break; }
                    const uint64_t ad = desc + (uint64_t)((s * S::kStage) >> 4), bd = ad + (S::kA >> 4);
                    if (it >= 2 && !ptx::mbar_wait(ptx::smem_u32(&acc_empty[b]), ((it >> 1) & 1) ^ 1, abort_flag)) { ok = false; break; }
                    ptx::tc_fence_after();
#pragma unroll
                    for (int k = 0; k < 4; ++k)                // 32 bytes further inside the swizzle atom a step
                        ptx::tc_mma_f8_pair(tmem_base + b * 256, ad + 2 * k, bd + 2 * k, g.idesc, k > 0);
                    ptx::tc_commit_pair(ptx::smem_u32(&acc_full[b]), 3);
                    ptx::tc_commit_pair(ptx::smem_u32(&empty[s]), 3);
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
        const int e = warp - 4, quarter = warp & 3, half = e >> 2;
        const int te = threadIdx.x & 127;                     // one of the 128 threads of this half
        const uint32_t boxes = S::kStgOff + e * (S::kBoxes * 4096);
        uint32_t ring = 0;
        uint32_t it = 0;
        bool ok = true;
        // Which sums a thread holds, as 64 pairs of neighbouring columns.  With one scale of b for the tile's 128 columns: all of one
        // row.  With a scale a column: four rows (lane / 4 + 8 k) and every fourth pair of columns, so that a thread needs 32 of
        // the 128 column scales and not all of them (128 floats to each of 256 threads a block are 1024 cycles of shared memory).
        constexpr int R = B_ROWS ? 4 : 1;
        auto row_of = [&](int k) { return B_ROWS ? (lane >> 2) + 8 * k : lane; };
        // the scales of the next block are fetched a block ahead
        int64_t mt = 0, nt = 0;
        float sa_next[R], sb_next = 0.f;
        const float *sap = nullptr, *sbp = nullptr;
        int sa_row = 0;
        auto fetch_a = [&]() {
#pragma unroll
            for (int k = 0; k < R; ++k) sa_next[k] = __ldg(sap + (min(sa_row + 8 * k, (int)g.M - 1) >> g.sa_shift));
        };
        auto aim = [&](int64_t t) {
            pair_tile(t, g, mt, nt);
            sa_row = (int)(mt * 256 + rank * 128 + quarter * 32) + row_of(0);
            sap = g.sa;
            fetch_a();
            const int64_t col = nt * 256 + half * 128 + (B_ROWS ? te : 0);
            sb_next = __ldg(sbp = g.sb + (min(col, g.N - 1) >> g.sb_shift));
        };
        if (pair < total) aim(pair);
        for (int64_t t = pair; t < total && ok; t += pairs) {
            const int64_t row0 = mt * 256 + rank * 128 + quarter * 32, col0 = nt * 256 + half * 128;
            float2 acc[64];
#pragma unroll
            for (int i = 0; i < 64; ++i) acc[i] = make_float2(0.f, 0.f);
            for (int64_t kb = 0; kb < g.kb_total; ++kb, ++it) {
                const uint32_t b = it & 1;
                uint64_t f[R];
#pragma unroll
                for (int k = 0; k < R; ++k) {
                    const float v = B_ROWS ? sa_next[k] : sa_next[k] * sb_next;
                    f[k] = ptx::pack2f(v, v);
                }
                const float* bs = b_scale + b * 256 + half * 128 + 2 * (lane & 3);
                if constexpr (B_ROWS) b_scale[b * 256 + half * 128 + te] = sb_next;
                if (kb + 1 < g.kb_total) {
                    sap += g.sa_ld;
                    fetch_a();
                    sb_next = __ldg(sbp += g.sb_ld);
                }
                if constexpr (B_ROWS) asm volatile("bar.sync %0, 128;" ::"r"(1 + half) : "memory");   // two buffers: a warp is at most one block ahead
                if (!ptx::mbar_wait(ptx::smem_u32(&acc_full[b]), (it >> 1) & 1, abort_flag))
                    ok = false;                                // counts the blocks to the end all the same: every later wait gives up at once
                ptx::tc_fence_after();
                const uint32_t ta = tmem_base + ((uint32_t)(quarter * 32) << 16) + b * 256 + half * 128;
                auto drained = [&]() {                         // the accumulator is out of tensor memory
                    ptx::tc_fence_before();
                    __syncwarp();
                    if (lane == 0) ptx::mbar_arrive_cluster_tmem(ptx::mapa(ptx::smem_u32(&acc_empty[b]), 0));
                };
                if constexpr (B_ROWS) {
#pragma unroll
                    for (int c = 0; c < 4; ++c) {              // 64 columns of 16 rows: this thread's pairs in two rows
                        uint32_t w[32];
                        ptx::tmem_ld_16x256b_x8(ta + 64 * (c >> 1) + ((c & 1) * 16u << 16), w);
                        ptx::tmem_ld_wait();
                        if (c == 3) drained();
#pragma unroll
                        for (int n = 0; n < 8; ++n) {
                            const uint64_t q = *reinterpret_cast<const uint64_t*>(bs + 64 * (c >> 1) + 8 * n);
#pragma unroll
                            for (int k = 0; k < 2; ++k)
                                scale_add(acc[32 * (c >> 1) + 8 * (2 * (c & 1) + k) + n], w[4 * n + 2 * k], w[4 * n + 2 * k + 1],
                                          ptx::mul2(f[2 * (c & 1) + k], q));
                        }
                    }
                } else {
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        uint32_t w[64];
                        ptx::tmem_ld_32x32b_x32(ta + 64 * c, w);
                        ptx::tmem_ld_32x32b_x32(ta + 64 * c + 32, w + 32);
                        ptx::tmem_ld_wait();
                        if (c == 1) drained();
#pragma unroll
                        for (int i = 0; i < 32; ++i) scale_add(acc[32 * c + i], w[2 * i], w[2 * i + 1], f[0]);
                    }
                }
            }
            if (t + pairs < total) aim(t + pairs);
            if (!ok || row0 >= g.M || col0 >= g.N) continue;
            // first column of pair i
            auto column = [&](int i) { return B_ROWS ? 64 * (i >> 5) + 8 * (i & 7) + 2 * (lane & 3) : 2 * i; };
            if (g.bias) {
#pragma unroll
                for (int i = 0; i < 64; ++i) {
                    acc[i].x += load_dyn(g.bias, g.bias_dtype, min(col0 + column(i), g.N - 1));
                    acc[i].y += load_dyn(g.bias, g.bias_dtype, min(col0 + column(i) + 1, g.N - 1));
                }
            }
            // out through boxes of 32 rows x 128 bytes in the 128-byte swizzle of the output's tensor map
            constexpr int PER = F32 ? 32 : 64;                 // columns of a box
#pragma unroll
            for (int c = 0; c < 128 / PER; ++c) {
                const int64_t col = col0 + PER * c;
                if (col >= g.N) break;
                uint8_t* box = smem + boxes + (ring++ % S::kBoxes) * 4096;
                const uint32_t box_s = ptx::smem_u32(box);
                if (lane == 0) ptx::bulk_wait_read<S::kBoxes - 1>();       // this box's last store has read it
                __syncwarp();
                if constexpr (B_ROWS) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint32_t at = box_s + row_of(k) * 128;       // row % 8 = lane / 4
#pragma unroll
                        for (int n = 0; n < PER / 8; ++n) {
                            const float2 p = F32 ? acc[32 * (c >> 1) + 8 * k + 4 * (c & 1) + n] : acc[32 * c + 8 * k + n];
                            if constexpr (F32)
                                ptx::st_shared_v2(at + (((2 * n + ((lane & 3) >> 1)) ^ (lane >> 2)) << 4) + 8 * (lane & 1), __float_as_uint(p.x), __float_as_uint(p.y));
                            else
                                ptx::st_shared(at + ((n ^ (lane >> 2)) << 4) + 4 * (lane & 3), pack2(p.x, p.y, g.out_dtype));
                        }
                    }
                } else {
#pragma unroll
                    for (int q = 0; q < 8; ++q) {
                        uint32_t w[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            if constexpr (F32) {
                                const float2 p = acc[16 * c + 2 * q + (j >> 1)];
                                w[j] = __float_as_uint(j & 1 ? p.y : p.x);
                            } else {
                                const float2 p = acc[32 * c + 4 * q + j];
                                w[j] = pack2(p.x, p.y, g.out_dtype);
                            }
                        }
                        ptx::st_shared_v4(box_s + lane * 128 + ((q ^ (lane & 7)) << 4), w[0], w[1], w[2], w[3]);
                    }
                }
                if (g.tma_out) {
                    ptx::fence_proxy_async();
                    __syncwarp();
                    if (lane == 0) { ptx::tma_store_2d(&tmap_c, box_s, (int)col, (int)row0); ptx::bulk_commit(); }
                } else {                                       // rows that are no multiple of 16 bytes long
                    __syncwarp();
                    const int n = (int)min((int64_t)32, g.M - row0);
                    for (int r = 0; r < n; ++r) {
                        const uint32_t v = *reinterpret_cast<const uint32_t*>(box + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4);
                        const int64_t at = (row0 + r) * g.N + col;
                        if constexpr (F32) {
                            if (col + lane < g.N) reinterpret_cast<uint32_t*>(g.out)[at + lane] = v;
                        } else {
                            if (col + 2 * lane < g.N) reinterpret_cast<uint16_t*>(g.out)[at + 2 * lane] = (uint16_t)v;
                            if (col + 2 * lane + 1 < g.N) reinterpret_cast<uint16_t*>(g.out)[at + 2 * lane + 1] = (uint16_t)(v >> 16);
                        }
                    }
                    __syncwarp();
                }
            }
        }
        if (lane == 0) ptx::bulk_wait_all();
    }
    ptx::tc_fence_before();
    __syncthreads();
    if (threadIdx.x == 0) give_up(*abort_flag);
    __syncwarp();
    ptx::cluster_arrive();                                    // the partner no longer touches this CTA's memory
    ptx::cluster_wait();
    if (warp == 1) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc_pair(tmem_base, 512);
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

template <int NT, bool SPLIT>
static int launch_fp8_split(const CUtensorMap& tp, const CUtensorMap& tq, const Fp8Gemm& g, cudaStream_t st) {
    using S = Fp8Tile<NT, SPLIT>;
    static_assert(S::kTotal <= (NT == 128 ? 232448 : 115712), "shared memory of one CTA an SM, or of two");
    auto kern = fp8_gemm_kernel<NT, SPLIT>;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kTotal) != cudaSuccess) { cudaGetLastError(); return MXQ_ERR_CUDA; }
    const int64_t grid = g.p_tiles * g.q_tiles * g.split;
    if (grid > 0x7fffffff) return MXQ_ERR_TOO_LARGE;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(S::kThreads);
    cfg.dynamicSmemBytes = S::kTotal;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = g.split; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = g.early ? 2 : 1;
    if (cudaLaunchKernelEx(&cfg, kern, tp, tq, g) != cudaSuccess) { cudaGetLastError(); return MXQ_ERR_CUDA; }
    return check_launch();
}

template <int NT>
static int launch_fp8(const CUtensorMap& tp, const CUtensorMap& tq, const Fp8Gemm& g, cudaStream_t st) {
    return g.split > 1 ? launch_fp8_split<NT, true>(tp, tq, g, st) : launch_fp8_split<NT, false>(tp, tq, g, st);
}

// out [M, N]: boxes of 32 rows x 128 bytes
static int make_out_map(CUtensorMap* m, void* base, int64_t M, int64_t N, int dtype) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return MXQ_ERR_CUDA;
    const cuuint64_t es = (cuuint64_t)dtype_size(dtype);
    cuuint64_t dims[2] = {(cuuint64_t)N, (cuuint64_t)M};
    cuuint64_t strides[1] = {(cuuint64_t)N * es};
    cuuint32_t box[2] = {(cuuint32_t)(128 / es), 32};
    cuuint32_t estr[2] = {1, 1};
    const CUtensorMapDataType t = dtype == MXQ_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16;
    return fn(m, t, 2, base, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
              CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS ? MXQ_OK : MXQ_ERR_CUDA;
}

template <bool B_ROWS, bool F32>
static int launch_fp8_pair(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tc, const Fp8Pair& g, cudaStream_t st) {
    auto kern = fp8_gemm_pair_kernel<B_ROWS, F32>;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Fp8PairSmem<B_ROWS>::kTotal) != cudaSuccess) { cudaGetLastError(); return MXQ_ERR_CUDA; }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2 * (unsigned)std::min<int64_t>(g.m_tiles * g.n_tiles, std::max(gemm_sms() / 2, 1)));
    cfg.blockDim = dim3(384);
    cfg.dynamicSmemBytes = Fp8PairSmem<B_ROWS>::kTotal;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, kern, ta, tb, tc, g) != cudaSuccess) { cudaGetLastError(); return MXQ_ERR_CUDA; }
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

namespace mxq {
// Which kernel and shape.  A kernel's time is the number of rounds its CTAs need on the GPU times what one CTA takes, a fixed part
// (launch, barriers, tensor memory, first loads, join and store: about 4.5 us) and a part for each K block it walks.  The
// latter, measured: 0.45 to 0.47 us with 16, 32 and 64 rows of a to a tile (what a CTA's own loads take from HBM; 0.30 to 0.41
// when b is in L2), 0.66 us with 128 (the scaling of the sums), or what HBM needs for the 16 KB of b that every CTA at work reads;
// 0.60 us for a CTA pair on 256 x 256, 1.0 us where b has a scale a row.  Both sides of each border (us):
// 64 x 4096 x 4096 split 1 / 2 / 4 / 8: 16.8 / 12.1 / 9.4 / 19.0; 1 x 8192 x 8192 (weights from HBM): 28.1 / 20.2 / 18.3 / 20.5,
// 1 x 28672 x 8192: 42.9 / 49.8 / 56.0 / 61.5; 128 x 4096 x 4096
// with 64 rows, split 2: 12.6, with 128 rows, split 4: 12.9; 1024 x 1024 x 1024 64 rows 8.2, 128 rows 11.3;
// 2048 x 2048 x 2048 pair 14.3, 128 rows 31.0.
struct Fp8Plan { int nt, split; };                 // nt 0: CTA pairs
static Fp8Plan plan_fp8(int64_t M, int64_t N, int64_t blocks, bool b_rows, bool tma_out) {
    const double sms = sm_count(), fixed = 4.5, hbm = 5.5e6;       // us, bytes a us
    const double block_us[4] = {0.45, 0.47, 0.47, 0.66};
    Fp8Plan best = {16, 1};
    double best_us = 1e300;
    for (int i = 0; i < 4; ++i) {
        const int nt = 16 << i;
        if (i > 0 && M <= nt / 2) break;           // half of the tile would be empty
        if (M > nt && nt < 64) continue;           // b would be read for several tiles of few rows
        const double p_tiles = (double)((N + 127) / 128), tiles = p_tiles * (double)((M + nt - 1) / nt);
        for (int split = 1; split <= 8; split *= 2) {
            if (split > 1 && blocks < 2 * split) break;
            // two CTAs on an SM below 128 rows; clusters of four and more leave some SMs of a GPC idle
            const double slots = sms * (nt < 128 ? 2 : 1) * (split >= 4 ? 0.875 : 1);
            const double rounds = ceil(tiles * split / slots), busy = tiles * split / rounds;
            const double share = nt < 128 && busy > sms ? 2 : 1;   // two CTAs on an SM share its tensor core and its fp32 pipes
            const double per = fmax(block_us[i] * (nt > 32 ? share : 1), fmin(busy, p_tiles * split / rounds) * 16384 / hbm);
            const double us = rounds * (fixed + (double)((blocks + split - 1) / split) * per);
            if (us < best_us) { best_us = us; best = {nt, split}; }
        }
    }
    if (M > 128 && N > 128) {
        const double rounds = ceil((double)((M + 255) / 256) * (double)((N + 255) / 256) / (sms / 2));
        // rows of no multiple of 16 bytes leave by single stores, 8 us a tile
        if (fixed + rounds * ((double)blocks * (b_rows ? 1.0 : 0.60) + (tma_out ? 0 : 8)) < best_us) best = {0, 1};
    }
    return best;
}

// `early`: b was complete before the kernel in front of this launch began
int fp8_gemm(const void* a, int64_t a_pitch, const float* a_scales, int a_tile, int a_fmt, const void* b, int64_t b_pitch,
             const float* b_scales, int b_tile, int b_fmt, void* out, int out_dtype, const void* bias, int bias_dtype, int64_t M,
             int64_t N, int64_t K, bool early, cudaStream_t st) {
    if (M < 0 || N < 0 || K <= 0 || a_fmt < 0 || a_fmt > 1 || b_fmt < 0 || b_fmt > 1) return MXQ_ERR_BAD_ARG;
    if (out_dtype < 0 || out_dtype > 2 || (bias && (bias_dtype < 0 || bias_dtype > 2))) return MXQ_ERR_BAD_ARG;
    if (M == 0 || N == 0) return MXQ_OK;
    if (!a || !b || !a_scales || !b_scales || !out || a_pitch < K || b_pitch < K) return MXQ_ERR_BAD_ARG;
    if (!aligned16(a) || !aligned16(b) || !aligned16(out) || a_pitch % 16 || b_pitch % 16) return MXQ_ERR_ALIGN;
    // coordinates are 32-bit, and a block or eight times a block count is added to them
    if (M > 0x7fffff00 || N > 0x7fffff00 || K > 0x7fffff00) return MXQ_ERR_TOO_LARGE;
    const int64_t blocks = (K + 127) / 128;
    const bool tma_out = (N * dtype_size(out_dtype)) % 16 == 0;
    const Fp8Plan plan = plan_fp8(M, N, blocks, !b_tile, tma_out);
    CUtensorMap ta, tb, tc;
    int rc;
    if (plan.nt == 0) {
        Fp8Pair g;
        g.sa = a_scales; g.sa_shift = a_tile ? 7 : 0; g.sa_ld = a_tile ? (M + 127) / 128 : M;
        g.sb = b_scales; g.sb_shift = b_tile ? 7 : 0; g.sb_ld = b_tile ? (N + 127) / 128 : N;
        g.out = out; g.out_dtype = out_dtype; g.bias = bias; g.bias_dtype = bias_dtype;
        g.M = M; g.N = N; g.kb_total = blocks;
        g.m_tiles = (M + 255) / 256; g.n_tiles = (N + 255) / 256;
        g.idesc = ptx::idesc_f8(a_fmt, b_fmt, 256, 256);
        g.tma_out = tma_out;
        if (g.m_tiles * g.n_tiles + sm_count() > 0x7fffffff) return MXQ_ERR_TOO_LARGE;
        rc = make_map(&ta, a, M, K, a_pitch, 128);
        if (!rc) rc = make_map(&tb, b, N, K, b_pitch, 128);
        tc = ta;
        if (!rc && g.tma_out) rc = make_out_map(&tc, out, M, N, out_dtype);
        if (rc) return rc;
        g_launch_count[0].fetch_add(1, std::memory_order_relaxed);
        if (out_dtype == MXQ_F32) return g.sb_shift ? launch_fp8_pair<false, true>(ta, tb, tc, g, st) : launch_fp8_pair<true, true>(ta, tb, tc, g, st);
        return g.sb_shift ? launch_fp8_pair<false, false>(ta, tb, tc, g, st) : launch_fp8_pair<true, false>(ta, tb, tc, g, st);
    }
    const int nt = plan.nt;
    Fp8Gemm g;
    g.sp = b_scales; g.sp_shift = b_tile ? 7 : 0; g.sp_ld = b_tile ? (N + 127) / 128 : N;
    g.sq = a_scales; g.sq_shift = a_tile ? 7 : 0; g.sq_ld = a_tile ? (M + 127) / 128 : M;
    g.out = out; g.out_dtype = out_dtype; g.bias = bias; g.bias_dtype = bias_dtype;
    g.P = N; g.Q = M; g.kb_total = blocks;
    g.p_tiles = (N + 127) / 128; g.q_tiles = (M + nt - 1) / nt;
    g.idesc = ptx::idesc_f8(b_fmt, a_fmt, 128, nt);
    g.split = plan.split;
    g.early = early;
    rc = make_map(&tb, b, N, K, b_pitch, 128);
    if (!rc) rc = make_map(&ta, a, M, K, a_pitch, nt);
    if (rc) return rc;
    g_launch_count[0].fetch_add(1, std::memory_order_relaxed);
    if (nt == 16) return launch_fp8<16>(tb, ta, g, st);
    if (nt == 32) return launch_fp8<32>(tb, ta, g, st);
    if (nt == 64) return launch_fp8<64>(tb, ta, g, st);
    return launch_fp8<128>(tb, ta, g, st);
}
}  // namespace mxq

extern "C" int mxq_fp8_gemm(const void* a, int64_t a_pitch, const float* a_scales, int a_tile, int a_fmt, const void* b,
                            int64_t b_pitch, const float* b_scales, int b_tile, int b_fmt, void* out, int out_dtype,
                            const void* bias, int bias_dtype, int64_t M, int64_t N, int64_t K, void* stream) {
    return mxq::fp8_gemm(a, a_pitch, a_scales, a_tile, a_fmt, b, b_pitch, b_scales, b_tile, b_fmt, out, out_dtype, bias, bias_dtype,
                         M, N, K, false, (cudaStream_t)stream);
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
    // the product may load weights while x is still being quantized: only that kernel lies between them and their last writer
    return mxq::fp8_gemm(workspace, pitch, scales, 0, x_fmt, w, w_pitch, w_scales, w_tile, w_fmt, y, y_dtype, bias, bias_dtype,
                         M, N, K, true, (cudaStream_t)stream);
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
