// Dense products of many rows on the 5th-generation tensor cores (tcgen05.mma, accumulators in tensor memory, TMA tensor copies).
//
// The weights are the M operand, the rows N: an output column is a lane of tensor memory, a row a column of it, so that only as many rows
// are multiplied as there are (in 32).  Pairs of CTAs (cta_group::2, 256 output columns x up to 256 rows), one CTA per SM, walk tiles:
//   warp 0     copies 128 rows of the weights and half of the tile's rows a stage (64 k), of each CTA
//   warp 1     (first CTA) issues the products of the pair
//   warp 2     allocates and frees tensor memory
//   warps 4-11 epilogue: bias, activation, residual or the gated pair, one rounding, while the next pass is multiplied
// A tile is one PASS over K into one of two sets of accumulators.  The gated pair is two passes, gate and up, on the same rows; the
// epilogue keeps act(gate) in registers.  With an fp32 output a pass covers at most 512 k and the epilogue adds passes in fp32 (CHAIN): the
// tensor core truncates as it accumulates, over 4096 k far beyond what fp32 sums are off by.
// Every wait is bounded; one that gives up sets the status word, every role leaves, copies in flight land, tensor memory is freed.
#include <algorithm>

#include "dense.cuh"
#include "tcgen05.cuh"

namespace gf {

__device__ int dense_status_word;

constexpr int DW_STAGES = 6, DW_HALF = 128 * 128, DW_STAGE = 2 * DW_HALF, DW_THREADS = 384, DW_ROWS = 256;
constexpr int DW_CHAIN = 512 / 64;                           // stages of a pass that is one of several
constexpr size_t DW_SMEM = 1024 + (size_t)DW_STAGES * DW_STAGE + 256;
constexpr int DW_REGS_COPY = 40, DW_REGS_EPI = 232;          // launched with 168 x 384: (40 + 2 x 232) x 128
static_assert(DW_REGS_COPY + 2 * DW_REGS_EPI <= 3 * 168, "registers");

struct DenseMaps { CUtensorMap w[2], x; };

struct DenseTiles {
    int bn, across, tiles, stages, pass;                     // rows of a tile, tiles of 256 output columns, all tiles, stages of K, stages of a pass
};

// Values of one lane (output column n, bias b) for 32 rows from r on: what follows the sums, without the store.
template <int MATS>
__device__ __forceinline__ void dense_act32(const DenseArgs &a, float (&v)[32], float b) {
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] += b;
    if (MATS == 2 && a.limit > 0.f) {
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = dense_below(v[i], a.limit);
    }
    switch (a.act) {
        case GLMFLASH_ACT_SILU:
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = silu(v[i]);
            break;
        case GLMFLASH_ACT_GELU:
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = dense_gelu(v[i]);
            break;
        case GLMFLASH_ACT_GELU_TANH:
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = dense_gelu_tanh(v[i]);
            break;
        case GLMFLASH_ACT_RELU:
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = v[i] < 0.f ? 0.f : v[i];
            break;
        default: break;
    }
}
// Walks `count` rows (more than 0) in 32 steps, staying on the last: addresses without a branch between the loads, so that all are on their
// way at once.
template <typename T, typename F>
__device__ __forceinline__ void dense_walk32(T *p, int64_t stride, int count, F f) {
#pragma unroll
    for (int i = 0; i < 32; ++i) {
        f(i, p);
        p += i + 1 < count ? stride : 0;
    }
}
__device__ __forceinline__ void dense_load32(float (&v)[32], const void *p, int64_t at, int64_t stride, int type, int count) {
    if (type == GLMFLASH_F32) dense_walk32(static_cast<const float *>(p) + at, stride, count, [&](int i, const float *q) { v[i] = *q; });
    else if (type == GLMFLASH_F16) dense_walk32(static_cast<const __half *>(p) + at, stride, count, [&](int i, const __half *q) { v[i] = __half2float(*q); });
    else dense_walk32(static_cast<const __nv_bfloat16 *>(p) + at, stride, count, [&](int i, const __nv_bfloat16 *q) { v[i] = __bfloat162float(*q); });
}
__device__ __forceinline__ void dense_store32(const float (&v)[32], void *p, int64_t at, int64_t stride, int type, int count) {
    if (type == GLMFLASH_F32) dense_walk32(static_cast<float *>(p) + at, stride, count, [&](int i, float *q) { if (i < count) *q = v[i]; });
    else if (type == GLMFLASH_F16) dense_walk32(static_cast<__half *>(p) + at, stride, count, [&](int i, __half *q) { if (i < count) *q = __float2half_rn(v[i]); });
    else dense_walk32(static_cast<__nv_bfloat16 *>(p) + at, stride, count, [&](int i, __nv_bfloat16 *q) { if (i < count) *q = __float2bfloat16_rn(v[i]); });
}

template <int MATS, bool CHAIN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(DW_THREADS, 1)
dense_wide_kernel(const __grid_constant__ DenseMaps maps, const DenseArgs a, const DenseTiles d) {
    extern __shared__ unsigned char smem_raw[];
    unsigned char *ring = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint64_t *full = reinterpret_cast<uint64_t *>(ring + (size_t)DW_STAGES * DW_STAGE);   // (first CTA) the copies of both have landed
    uint64_t *done = full + DW_STAGES;                       // products of the stage done, in both CTAs
    uint64_t *acc_full = done + DW_STAGES;                   // [2] a pass is complete, in both
    uint64_t *acc_empty = acc_full + 2;                      // [2] (first CTA) read by the epilogue warps of both
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(acc_empty + 2);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    int *status = &dense_status_word;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = (int)t5_cta_rank(), pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    if (tid == 0) {
        for (int s = 0; s < DW_STAGES; ++s) { mbar_init(full + s, 1); mbar_init(done + s, 1); }
        for (int b = 0; b < 2; ++b) { mbar_init(acc_full + b, 1); mbar_init(acc_empty + b, 16); }
        *abort_flag = 0;
        mbar_fence_init();
    }
    if (warp == 2) t5_alloc<2>(tmem_slot, 512);
    t5_fence_before();
    cluster_sync();                                          // the peer's barriers are initialised as well
    t5_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_wait();
    pdl_launch_dependents();
    const int items = d.tiles > pair ? (d.tiles - pair + pairs - 1) / pairs : 0;
    const uint32_t stages = (uint32_t)items * MATS * d.stages;
    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(DW_REGS_COPY));
        if (warp == 0 && lane == 0) {
            const uint32_t full0 = t5_of_cta(full, 0);       // (the copies of both CTAs count on the first one's barrier)
            T5Ring at;
            uint32_t it = 0;
            bool ok = true;
            for (int tile = pair; ok && tile < d.tiles; tile += pairs) {
                const int n = (tile % d.across) * 256 + rank * 128, r = (tile / d.across) * d.bn + rank * (d.bn >> 1);
                for (int m = 0; m < MATS && ok; ++m)
                    for (int s = 0; s < d.stages; ++s, ++it) {
                        if (it >= DW_STAGES && !t5_wait<200>(done + at.slot, at.parity ^ 1, abort_flag, status, GF_STATUS_TMA_TIMEOUT)) { ok = false; break; }
                        if (rank == 0) mbar_expect_tx(full + at.slot, 2u * (DW_HALF + (uint32_t)(d.bn >> 1) * 128));
                        unsigned char *dst = ring + at.slot * DW_STAGE;
                        t5_load_pair(dst, &maps.w[m], s * 64, n, full0 + 8 * at.slot);
                        t5_load_pair(dst + DW_HALF, &maps.x, s * 64, r, full0 + 8 * at.slot);
                        at.next(DW_STAGES);
                    }
            }
            // after a give-up: copies in flight have landed before the CTA leaves (the second CTA's count elsewhere: it stays that long)
            if (!ok || *abort_flag)
                for (uint32_t k = it > DW_STAGES ? it - DW_STAGES : 0; k < it; ++k) mbar_wait((rank ? done : full) + k % DW_STAGES, (k / DW_STAGES) & 1, nullptr, 1000u);
        } else if (warp == 1 && rank == 0) {
            const uint32_t idesc = t5_idesc(256, d.bn, a.type == GLMFLASH_BF16);
            const uint64_t desc0 = t5_desc(smem_u32(ring));
            T5Ring at;
            uint32_t pc = 0;
            bool ok = true;
            for (int i = 0; i < items * MATS && ok; ++i)
                for (int s0 = 0; s0 < d.stages && ok; s0 += d.pass, ++pc) {
                    const uint32_t b = pc & 1, acc = tmem + b * DW_ROWS;
                    ok = __all_sync(0xffffffffu, t5_wait<0>(acc_empty + b, ((pc >> 1) & 1) ^ 1, abort_flag, status, GF_STATUS_MMA_TIMEOUT));
                    if (!ok) break;
                    t5_fence_after();
                    const int end = min(d.pass, d.stages - s0);
                    for (int s = 0; s < end; ++s) {
                        ok = __all_sync(0xffffffffu, t5_wait<0>(full + at.slot, at.parity, abort_flag, status, GF_STATUS_MMA_TIMEOUT));
                        if (!ok) break;
                        t5_fence_after();
                        const uint64_t da = desc0 + at.slot * (DW_STAGE >> 4), db = da + (DW_HALF >> 4);
                        if (t5_elect()) {
#pragma unroll
                            for (int k = 0; k < 4; ++k) t5_mma<2>(acc, da + 2 * k, db + 2 * k, idesc, k > 0 || s > 0);
                            t5_commit<2>(done + at.slot);
                            if (s == end - 1) t5_commit<2>(acc_full + b);
                        }
                        __syncwarp();
                        at.next(DW_STAGES);
                    }
                }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(DW_REGS_EPI));
        const int q = warp & 3, half = (warp - 4) >> 2, cols = d.bn >> 1;
        const uint32_t lanes = tmem + ((uint32_t)(q * 32) << 16) + half * cols;
        const uint32_t empty0 = t5_of_cta(acc_empty, 0);
        uint32_t pc = 0;
        bool ok = true;
        float keep[4][32];                                   // gated: act(gate) of this lane's rows;  CHAIN: sums
        for (int tile = pair; ok && tile < d.tiles; tile += pairs) {
            const int n = (tile % d.across) * 256 + rank * 128 + q * 32 + lane, r0 = (tile / d.across) * d.bn + half * cols;
            const int live = n < a.N ? min(cols, a.rows - r0) : 0;             // rows of this thread
#pragma unroll
            for (int m = 0; m < MATS; ++m) {
                const float bias = n < a.N && a.bias[m] ? dense_load(a.bias[m], n, a.bias_type) : 0.f;
                const int passes = CHAIN ? (d.stages + d.pass - 1) / d.pass : 1;
                for (int p = 0; p < passes; ++p, ++pc) {
                    const uint32_t b = pc & 1;
                    // (the residual of the first rows is on its way while the pass is multiplied)
                    if (MATS == 1 && !CHAIN && a.residual && live > 0) dense_load32(keep[0], a.residual, r0 * a.rs + n, a.rs, a.residual_type, live);
                    ok = __all_sync(0xffffffffu, t5_wait<200>(acc_full + b, (pc >> 1) & 1, abort_flag, status, GF_STATUS_MMA_TIMEOUT));
                    if (!ok) break;
                    t5_fence_after();
                    if (CHAIN) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            if (32 * j >= cols) continue;
                            float v[32];
                            t5_ld32(lanes + b * DW_ROWS + 32 * j, v);
#pragma unroll
                            for (int i = 0; i < 32; ++i) keep[j][i] = p ? keep[j][i] + v[i] : v[i];
                        }
                        t5_fence_before();
                        __syncwarp();
                        if (lane == 0) t5_arrive_cluster(empty0 + 8 * b);
                        if (p < passes - 1) continue;
                    }
                    // One copy of the code that follows the sums: the four groups of 32 rows take turns in keep[0].
#pragma unroll 1
                    for (int j = 0; j < 4; ++j) {
                        float v[32];
                        __syncwarp();
                        if (CHAIN) {
#pragma unroll
                            for (int i = 0; i < 32; ++i) v[i] = keep[0][i];
                        } else if (32 * j < cols) {
                            t5_ld32(lanes + b * DW_ROWS + 32 * j, v);
                        }
                        if (!CHAIN && 32 * (j + 1) >= cols && 32 * j < cols) {  // the last of them: the accumulators are read
                            t5_fence_before();
                            __syncwarp();
                            if (lane == 0) t5_arrive_cluster(empty0 + 8 * b);
                        }
                        const int count = live - 32 * j;
                        const int64_t row = r0 + 32 * j;
                        if (count > 0) {
                            if (MATS == 1) {
                                float next[32];
                                if (a.residual && CHAIN) dense_load32(next, a.residual, row * a.rs + n, a.rs, a.residual_type, count);
                                if (a.residual && !CHAIN && count > 32) dense_load32(next, a.residual, (row + 32) * a.rs + n, a.rs, a.residual_type, count - 32);
                                dense_act32<1>(a, v, bias);
                                if (a.residual) {
#pragma unroll
                                    for (int i = 0; i < 32; ++i) {
                                        v[i] += CHAIN ? next[i] : keep[0][i];
                                        if (!CHAIN) keep[0][i] = next[i];
                                    }
                                }
                            } else if (m == 0) {
                                dense_act32<2>(a, v, bias);
                            } else {
                                // (CHAIN: act(gate) waits in its places of the fp32 output)
                                float gate[32];
                                if (CHAIN) dense_load32(gate, a.out, row * a.os + n, a.os, GLMFLASH_F32, count);
#pragma unroll
                                for (int i = 0; i < 32; ++i) {
                                    v[i] += bias;
                                    if (a.limit > 0.f) v[i] = dense_within(v[i], a.limit);
                                    v[i] *= CHAIN ? gate[i] : keep[0][i];
                                }
                            }
                            if (MATS == 1 || m == 1 || CHAIN) dense_store32(v, a.out, row * a.os + n, a.os, a.out_type, count);
                        }
                        if (CHAIN || MATS == 2)
#pragma unroll
                            for (int i = 0; i < 32; ++i) {
                                keep[0][i] = keep[1][i];
                                keep[1][i] = keep[2][i];
                                keep[2][i] = keep[3][i];
                                if (MATS == 2 && !CHAIN) keep[3][i] = v[i];
                            }
                    }
                }
                if (!ok) break;
            }
        }
        // the arrivals of the last commits have come in before this CTA ends
        for (uint32_t k = stages > DW_STAGES ? stages - DW_STAGES : 0; k < stages && ok; ++k)
            ok = t5_wait<200>(done + k % DW_STAGES, (k / DW_STAGES) & 1, abort_flag, status, GF_STATUS_MMA_TIMEOUT);
    }
    t5_fence_before();
    // the pair ends together (not the aligned form: single lanes of warps 0 and 1 worked alone)
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
    t5_fence_after();
    if (warp == 2) t5_dealloc<2>(tmem, 512);
}

// [rows][stride] of 16-bit elements, boxes of 64 elements x box_rows
static int dense_map(CUtensorMap *map, const void *base, bool bf, int64_t rows, int K, int64_t stride, int box_rows, const char *what) {
    const uint64_t dims[2] = {(uint64_t)K, (uint64_t)rows}, strides[1] = {(uint64_t)stride * 2};
    const uint32_t box[2] = {64, (uint32_t)box_rows};
    return encode_map(map, bf ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void *>(base), dims, strides, box, what);
}

int dense_wide(cudaStream_t s, const DenseArgs &a, bool pdl) {
    static int sms[64] = {};                               // (threads that come here together set the same)
    int dev = 0;
    GF_CUDA(cudaGetDevice(&dev));
    GF_REQUIRE(dev >= 0 && dev < 64, "device ordinal out of range");
    if (!sms[dev]) {
        int n = 0;
        GF_CUDA(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev));
        GF_CUDA(cudaFuncSetAttribute(dense_wide_kernel<1, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)DW_SMEM));
        GF_CUDA(cudaFuncSetAttribute(dense_wide_kernel<1, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)DW_SMEM));
        GF_CUDA(cudaFuncSetAttribute(dense_wide_kernel<2, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)DW_SMEM));
        GF_CUDA(cudaFuncSetAttribute(dense_wide_kernel<2, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)DW_SMEM));
        sms[dev] = n;
    }
    const int pairs = sms[dev] / 2, mats = a.w[1] ? 2 : 1;
    const bool chain = a.out_type == GLMFLASH_F32 && a.K > DW_CHAIN * 64, bf = a.type == GLMFLASH_BF16;
    DenseTiles d;
    d.across = (a.N + 255) / 256;
    // Rows of a tile: what makes the rounds of tiles over the pairs shortest.  A stage of a round takes 234 ns with 32 rows, 244 with 64, 280 with
    // 128, 312 with 192 (the copies bound it: 42 to 50 bytes a clock and SM) and 386 with 256 (1.61 PFLOP/s: the power limit).
    int64_t best = INT64_MAX;
    for (int bn = 32; bn <= DW_ROWS; bn += 32) {        // (N of a pair's product goes in 32)
        const int64_t tiles = (int64_t)((a.rows + bn - 1) / bn) * d.across, cost = (tiles + pairs - 1) / pairs * std::max(440 + bn, 260 + 2 * bn);
        if (cost <= best && tiles <= INT32_MAX / 2) { best = cost; d.bn = bn; d.tiles = (int)tiles; }
    }
    GF_REQUIRE(best != INT64_MAX, "rows * outputs is too large");
    d.stages = (a.K + 63) / 64;
    d.pass = chain ? DW_CHAIN : d.stages;
    const int64_t passes = (int64_t)d.tiles / pairs * mats * d.stages;
    GF_REQUIRE(passes < INT32_MAX, "product is too large");
    DenseMaps maps;
    if (dense_map(&maps.w[0], a.w[0], bf, a.N, a.K, a.ws[0], 128, "weights")) return -1;
    if (mats == 2 && dense_map(&maps.w[1], a.w[1], bf, a.N, a.K, a.ws[1], 128, "weights")) return -1;
    if (mats == 1) maps.w[1] = maps.w[0];
    if (dense_map(&maps.x, a.x, bf, a.rows, a.K, a.xs, d.bn / 2, "rows")) return -1;
    const dim3 grid((unsigned)(2 * std::min(d.tiles, pairs))), block(DW_THREADS);
    auto kernel = mats == 2 ? (chain ? dense_wide_kernel<2, true> : dense_wide_kernel<2, false>) : (chain ? dense_wide_kernel<1, true> : dense_wide_kernel<1, false>);
    return launch_k(kernel, grid, block, DW_SMEM, s, pdl, maps, a, d);
}

}  // namespace gf

using namespace gf;

extern "C" const int32_t *glmflash_linear_status(void) {
    void *p = nullptr;
    return cudaGetSymbolAddress(&p, dense_status_word) == cudaSuccess ? static_cast<int32_t *>(p) : nullptr;
}
extern "C" int glmflash_linear_clear_status(void *stream) {
    void *p = nullptr;
    GF_CUDA(cudaGetSymbolAddress(&p, dense_status_word));
    GF_CUDA(cudaMemsetAsync(p, 0, sizeof(int), (cudaStream_t)stream));
    return 0;
}
