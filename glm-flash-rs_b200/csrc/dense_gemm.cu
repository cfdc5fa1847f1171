// Dense products of many rows on the 5th-generation tensor cores (tcgen05.mma, accumulators in tensor memory, TMA tensor copies).
//
// The weights are the M operand, the rows N: an output column is a lane of tensor memory, a row a column of it, so that only as many rows
// are multiplied as there are (in 32).  Pairs of CTAs (cta_group::2, 256 output columns x up to 256 rows), one CTA per SM, walk tiles:
//   warps 0, 3 copy 128 rows of the weights and half of the tile's rows a stage (128 k), of each CTA
//   warp 1     (first CTA) issues the products of the pair
//   warp 2     allocates and frees tensor memory
//   warps 4-11 epilogue: bias, activation, residual or the gated pair, one rounding, while the next pass is multiplied
// A tile is one PASS over K into one of two sets of accumulators.  The gated pair is two passes, gate and up, on the same rows; the
// epilogue keeps act(gate) in registers.  With an fp32 output a pass covers at most 512 k and the epilogue adds passes in fp32 (CHAIN): the
// tensor core truncates as it accumulates, over 4096 k far beyond what fp32 sums are off by.  With a 16-bit output a pass covers 8192 k: rows of one sign
// lose 1e-4 over 16384 and 1.7e-3 over 262144 in one pass, a half step of fp16 is 5e-4.
// Stages are 128 k long because a turn of a copying warp (wait, announce, copy) takes 300 to 450 clocks whatever it copies, and each copy beyond the
// first 70 (weights and rows have a warp each): with 64 k and two copies a turn an SM took in 80 GB/s, with one CTA alone as with 148, at any
// depth of the ring.  Where K is a multiple of 64 one copy brings both halves of a stage.
// 8192 x 4096 x 4096 with a residual, calls one behind another: 174 us in the first milliseconds (1.5 GHz and more), 208 to 220 by the GPU once the power limit
// holds it at 1.3 GHz; the tensor pipe is active for 85 % of the time.
// Loops that wait have no way out of them but their end (one that depends on a wait costs 70 to 120 clocks a turn: 180 to 230 in place of 113), and
// whole warps run them, of which an elected lane copies or multiplies.
// Every wait is bounded; one that gives up sets the status word, every role leaves, copies in flight land, tensor memory is freed.
#include <algorithm>
#include <atomic>
#include <initializer_list>

#include "dense.cuh"
#include "tcgen05.cuh"

namespace gf {

__device__ int dense_status_word;

constexpr int DW_K = 128, DW_A = 128 * DW_K * 2;             // k of a stage; bytes of its weights in a CTA
constexpr int DW_DEPTH = 5, DW_RING = 3 * (DW_A + 256 * 128), DW_THREADS = 384, DW_ROWS = 256;
constexpr int DW_CHAIN = 512 / DW_K, DW_CHAIN16 = 8192 / DW_K;   // stages of a pass that is one of several, of an fp32 output and of a 16-bit one
constexpr size_t DW_SMEM = 1024 + DW_RING + 256;
constexpr int DW_REGS_COPY = 40, DW_REGS_EPI = 232;          // launched with 168 x 384: (40 + 2 x 232) x 128
static_assert(DW_REGS_COPY + 2 * DW_REGS_EPI <= 3 * 168, "registers");

struct DenseMaps { CUtensorMap a[2], b[2]; };              // M and N operand of the product, or of the two of a gated pair

// Tiles in the order of M, a pair's next one without a division.
struct DenseTiles {
    int bn, across, tiles, stages, pass;                     // N of a tile, tiles along M (256), all tiles, stages of K, stages of a pass
    int depth, copies;                                       // stages of the ring, copies that bring a stage of an operand
    int step_m, step_n;                                      // from a pair's tile to its next one
};
struct DenseTile {
    int m, n;
    __device__ __forceinline__ void next(const DenseTiles &d) {
        m += d.step_m;
        n += d.step_n;
        if (m >= d.across) { m -= d.across; ++n; }
    }
};

// A stage of `rows` rows: two tiles of 64 k one behind the other.  One copy of a [64][rows][2] box, or two of [64][rows] (K is no multiple of
// 64: the end of a row has to be seen).
template <typename F>
__device__ __forceinline__ void dense_copy(unsigned char *dst, int stage, int rows, int copies, F copy) {
    copy(dst, 2 * stage);
    if (copies == 2) copy(dst + rows * 128, 2 * stage + 1);
}

// Values of one lane (output column n, bias b) for 32 rows from r on: what follows the sums, without the store.
template <int MATS>
__device__ __forceinline__ void dense_act32(const DenseArgs &a, float (&v)[32], float b) {
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] += b;              // (0 where it has been added)
    if (MATS == 2 && a.limit > 0.f) {
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = dense_below(v[i], a.limit);
    }
    dense_act(v, a.act);
}
// (Residual and output pass through L2 without pushing operands out: 8192 x 4096 x 4096 with a residual 221 -> 215 us at the power limit, with the tiles of then.)
// f(i, address of row i) for 32 rows, of which `count` (more than 0) are there: the others stand on the last.  Addresses without a branch between the
// loads, so that all are on their way at once, and each from its own product where the strides allow it (one from another they are a chain of 800
// clocks for 32 rows).
template <typename T, typename F>
__device__ __forceinline__ void dense_walk32(T *p, int64_t stride, int count, F f) {
    if (stride < 1 << 26) {
        const int s = (int)stride;
#pragma unroll
        for (int i = 0; i < 32; ++i) f(i, p + min(i, count - 1) * s);
        return;
    }
#pragma unroll
    for (int i = 0; i < 32; ++i) {
        f(i, p);
        p += i + 1 < count ? stride : 0;
    }
}
__device__ __forceinline__ void dense_load32(float (&v)[32], const void *p, int64_t at, int64_t stride, int type, int count) {
    if (type == GLMFLASH_F32) dense_walk32(static_cast<const float *>(p) + at, stride, count, [&](int i, const float *q) { v[i] = __ldcs(q); });
    else if (type == GLMFLASH_F16) dense_walk32(static_cast<const __half *>(p) + at, stride, count, [&](int i, const __half *q) { v[i] = __half2float(__ushort_as_half(__ldcs(reinterpret_cast<const unsigned short *>(q)))); });
    else dense_walk32(static_cast<const __nv_bfloat16 *>(p) + at, stride, count, [&](int i, const __nv_bfloat16 *q) { v[i] = __bfloat162float(__ushort_as_bfloat16(__ldcs(reinterpret_cast<const unsigned short *>(q)))); });
}
__device__ __forceinline__ void dense_store32(const float (&v)[32], void *p, int64_t at, int64_t stride, int type, int count) {
    if (type == GLMFLASH_F32) dense_walk32(static_cast<float *>(p) + at, stride, count, [&](int i, float *q) { if (i < count) __stcs(q, v[i]); });
    else if (type == GLMFLASH_F16) dense_walk32(static_cast<__half *>(p) + at, stride, count, [&](int i, __half *q) { if (i < count) __stcs(reinterpret_cast<unsigned short *>(q), __half_as_ushort(__float2half_rn(v[i]))); });
    else dense_walk32(static_cast<__nv_bfloat16 *>(p) + at, stride, count, [&](int i, __nv_bfloat16 *q) { if (i < count) __stcs(reinterpret_cast<unsigned short *>(q), __bfloat16_as_ushort(__float2bfloat16_rn(v[i]))); });
}

// The same along a row: 32 neighbouring elements of each lane, 16 bytes at a time where they are aligned and come in that many.
__device__ __forceinline__ void dense_unpack8(float *v, const uint4 &q, int type) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (type == GLMFLASH_F16) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
            v[2 * i] = f.x; v[2 * i + 1] = f.y;
        } else {
            v[2 * i] = __uint_as_float(w[i] << 16); v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
}
__device__ __forceinline__ void dense_load_along(float (&v)[32], const void *p, int64_t at, int type, int count) {
    const int size = type == GLMFLASH_F32 ? 4 : 2;
    const char *q = static_cast<const char *>(p) + at * size;
    if ((uintptr_t)q % 16 || count * size % 16) return dense_load32(v, p, at, 1, type, count);
    if (type == GLMFLASH_F32)
#pragma unroll
        for (int i = 0; i < 8; ++i) *reinterpret_cast<float4 *>(v + 4 * i) = __ldcs(reinterpret_cast<const float4 *>(q) + min(i, count / 4 - 1));
    else
#pragma unroll
        for (int i = 0; i < 4; ++i) dense_unpack8(v + 8 * i, __ldcs(reinterpret_cast<const uint4 *>(q) + min(i, count / 8 - 1)), type);
}
__device__ __forceinline__ void dense_store_along(const float (&v)[32], void *p, int64_t at, int type, int count) {
    const int size = type == GLMFLASH_F32 ? 4 : 2;
    char *q = static_cast<char *>(p) + at * size;
    if ((uintptr_t)q % 16 || count * size % 16) return dense_store32(v, p, at, 1, type, count);
    if (type == GLMFLASH_F32) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (4 * i < count) __stcs(reinterpret_cast<float4 *>(q) + i, make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]));
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float2 f = make_float2(v[8 * i + 2 * k], v[8 * i + 2 * k + 1]);
            if (type == GLMFLASH_F16) {
                const __half2 h = __float22half2_rn(f);
                w[k] = *reinterpret_cast<const uint32_t *>(&h);
            } else {
                const __nv_bfloat162 h = __float22bfloat162_rn(f);
                w[k] = *reinterpret_cast<const uint32_t *>(&h);
            }
        }
        if (8 * i < count) __stcs(reinterpret_cast<uint4 *>(q) + i, make_uint4(w[0], w[1], w[2], w[3]));
    }
}

// ROWS_M: the roles are exchanged, rows of x along M and outputs along N: a lane is a row, a column of tensor memory an output.
template <int MATS, bool CHAIN, bool ROWS_M>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(DW_THREADS, 1)
dense_wide_kernel(const __grid_constant__ DenseMaps maps, const DenseArgs a, const DenseTiles d) {
    extern __shared__ unsigned char smem_raw[];
    unsigned char *ring = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint64_t *full = reinterpret_cast<uint64_t *>(ring + DW_RING);        // (first CTA) the copies of both have landed
    uint64_t *done = full + DW_DEPTH;                        // products of the stage done, in both CTAs
    uint64_t *acc_full = done + DW_DEPTH;                    // [2] a pass is complete, in both
    uint64_t *acc_empty = acc_full + 2;                      // [2] (first CTA) read by the epilogue warps of both
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(acc_empty + 2);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    int *status = &dense_status_word;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = (int)t5_cta_rank(), pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    if (tid < DW_DEPTH) {
        mbar_init(full + tid, 2);
        mbar_init(done + tid, 1);
        mbar_fence_init();
    }
    if (tid == 0) {
        for (int b = 0; b < 2; ++b) { mbar_init(acc_full + b, 1); mbar_init(acc_empty + b, 16); }
        *abort_flag = 0;
        mbar_fence_init();
    }
    if (tid < 2 * MATS) asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)(&maps.a[0] + (tid & 1 ? 2 : 0) + (tid >> 1))) : "memory");
    if (warp == 2) t5_alloc<2>(tmem_slot, 512);
    const int items = (d.tiles - pair + pairs - 1) / pairs;  // (there are no more pairs than tiles)
    const uint32_t stages = (uint32_t)items * MATS * d.stages, depth = d.depth, slot_bytes = DW_A + d.bn * 128;
    DenseTile tile = {pair % d.across, pair / d.across};
    t5_fence_before();
    cluster_sync();                                          // the peer's barriers are initialised as well
    t5_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_wait();
    pdl_launch_dependents();
    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(DW_REGS_COPY));
        if (warp == 0 || warp == 3) {
            const uint32_t full0 = t5_of_cta(full, 0);       // (the copies of both CTAs count on the first one's barrier)
            const bool along_n = warp == 3;
            const int box = along_n ? d.bn >> 1 : 128;
            T5Ring at;
            const bool leader = t5_elect();
            uint32_t turn = 0, it = 0;                       // it: stages that this lane has copied
            bool ok = true;
            for (int i = 0; ok && i < items; ++i, tile.next(d)) {
                const int y = along_n ? tile.n * d.bn + rank * box : tile.m * 256 + rank * 128;
                for (int m = 0; m < MATS; ++m) {
                    const CUtensorMap *map = along_n ? &maps.b[m] : &maps.a[m];
#pragma unroll 1
                    for (int s = 0; s < d.stages; ++s, ++turn) {
                        if (turn >= depth) ok &= t5_wait<200>(done + at.slot, at.parity ^ 1, abort_flag, status, GF_STATUS_TMA_TIMEOUT);
                        if (leader) {
                            if (ok) {
                                if (rank == 0) mbar_expect_tx(full + at.slot, 2 * box * DW_K * 2);
                                const uint32_t bar = full0 + 8 * at.slot;
                                dense_copy(ring + at.slot * slot_bytes + (along_n ? DW_A : 0), s, box, d.copies, [&](unsigned char *to, int k) { t5_load_pair(to, map, d.copies == 1, k, y, bar); });
                                ++it;
                            }
                        }
                        __syncwarp();
                        at.next(depth);
                    }
                }
            }
            // after a give-up: copies in flight have landed before the CTA leaves (the second CTA's count elsewhere: it stays that long)
            if (!ok || *abort_flag)
                for (uint32_t k = it > depth ? it - depth : 0; k < it; ++k) mbar_wait((rank ? done : full) + k % depth, (k / depth) & 1, nullptr, 1000u);
        } else if (warp == 1 && rank == 0) {
            const uint32_t idesc = t5_idesc(256, d.bn, a.type == GLMFLASH_BF16);
            const uint64_t desc0 = t5_desc(smem_u32(ring));
            const uint32_t next = d.bn * 64 >> 4;            // from the first 64 k of the rows to the second
            T5Ring at;
            const bool leader = t5_elect();
            uint32_t pc = 0, left = stages;
            bool ok = true;
            for (int i = 0; i < items * MATS; ++i)
                for (int s0 = 0; s0 < d.stages; s0 += d.pass, ++pc) {
                    const uint32_t b = pc & 1, acc = tmem + b * DW_ROWS;
                    if (pc >= 2) ok &= t5_wait<0>(acc_empty + b, ((pc >> 1) & 1) ^ 1, abort_flag, status, GF_STATUS_MMA_TIMEOUT);
                    t5_fence_after();
                    const int end = min(d.pass, d.stages - s0);
                    for (int s = 0; s < end; ++s, --left) {
                        ok &= t5_wait<0>(full + at.slot, at.parity, abort_flag, status, GF_STATUS_MMA_TIMEOUT);
                        const uint64_t da = desc0 + at.slot * (slot_bytes >> 4), db = da + (DW_A >> 4);
                        if (leader) {
#pragma unroll
                            for (int k = 0; k < DW_K / 16; ++k)
                                t5_mma<2>(acc, da + 2 * (k & 3) + (k >> 2) * (128 * 128 >> 4), db + 2 * (k & 3) + (k >> 2) * next, idesc, k > 0 ? 1u : s > 0);
                            if (left > depth) t5_commit<2>(done + at.slot);        // (somebody waits for it)
                        }
                        at.next(depth);
                        __syncwarp();
                    }
                    if (leader) t5_commit<2>(acc_full + b);
                }
            if (!ok) t5_settle();
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(DW_REGS_EPI));
        const int q = warp & 3, half = (warp - 4) >> 2, cols = d.bn >> 1;
        const uint32_t lanes = tmem + ((uint32_t)(q * 32) << 16) + half * cols;
        const uint32_t empty0 = t5_of_cta(acc_empty, 0);
        // (nobody waits for the last two passes to be read, and an arrival in the other CTA must not come after that one has left)
        const uint32_t all = (uint32_t)items * MATS * (CHAIN ? (d.stages + d.pass - 1) / d.pass : 1);
        constexpr bool EARLY = MATS == 1 && !CHAIN;
        // (a gated pair in passes keeps sums of up to 64 rows and as many act(gate) where the output has no room for those)
        const bool parked = CHAIN && MATS == 2 && a.out_type != GLMFLASH_F32;
        const int turns = parked ? 2 : CHAIN || MATS == 2 ? 4 : (cols + 31) >> 5;
        uint32_t pc = 0;
        bool ok = true;
        float keep[4][32];                                   // gated: act(gate) of this lane's rows;  CHAIN: sums
        for (int i = 0; ok && i < items; ++i, tile.next(d)) {
            // this lane's place along M, the columns' along N, and how many of them there are
            const int own = tile.m * 256 + rank * 128 + q * 32 + lane, c0 = tile.n * d.bn + half * cols;
            const int live = own < (ROWS_M ? a.rows : a.N) ? min(cols, (ROWS_M ? a.N : a.rows) - c0) : 0;
            auto place = [&](int c, int64_t stride) { return ROWS_M ? own * stride + c : c * stride + own; };
            auto load = [&](float (&v)[32], const void *p, int c, int64_t stride, int type, int count) {
                if (ROWS_M) dense_load_along(v, p, place(c, stride), type, count);
                else dense_load32(v, p, place(c, stride), stride, type, count);
            };
#pragma unroll
            for (int m = 0; m < MATS; ++m) {
                const float bias = !ROWS_M && own < a.N && a.bias[m] ? dense_load(a.bias[m], own, a.bias_type) : 0.f;
                const int passes = CHAIN ? (d.stages + d.pass - 1) / d.pass : 1;
                for (int p = 0; p < passes; ++p, ++pc) {
                    const uint32_t b = pc & 1;
                    // (the residual of the first rows is on its way while the pass is multiplied)
                    if (MATS == 1 && !CHAIN && a.residual && live > 0 && (!EARLY || i)) load(keep[0], a.residual, c0, a.rs, a.residual_type, min(live, 32));
                    if (!EARLY) {
                        ok = __all_sync(0xffffffffu, t5_wait<200>(acc_full + b, (pc >> 1) & 1, abort_flag, status, GF_STATUS_MMA_TIMEOUT));
                        if (!ok) break;
                        t5_fence_after();
                    }
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
                        if (lane == 0 && pc + 2 < all) t5_arrive_cluster(empty0 + 8 * b);
                        if (p < passes - 1) continue;
                    }
                    // One copy of the code that follows the sums: the four groups of 32 rows take turns in keep[0].  A pair's first tile has a turn more,
                    // of no rows, while it is multiplied: it brings the instructions in, which took longer than they do, and the first residual
                    // (1000 x 2048 x 1536 10.4 -> 10.1 us; registers do not last for it in a gated pair, nor with passes added in fp32: 21 us for 17).
#pragma unroll 1
                    for (int j = EARLY && !i ? -1 : 0; j < turns; ++j) {
                        float v[32];
                        if (EARLY && j == 0) {
                            ok = __all_sync(0xffffffffu, t5_wait<200>(acc_full + b, (pc >> 1) & 1, abort_flag, status, GF_STATUS_MMA_TIMEOUT));
                            if (!ok) break;
                            t5_fence_after();
                        }
                        __syncwarp();
                        if (CHAIN) {
#pragma unroll
                            for (int i = 0; i < 32; ++i) v[i] = keep[0][i];
                        } else if ((!EARLY || j >= 0) && 32 * j < cols) {
                            t5_ld32(lanes + b * DW_ROWS + 32 * j, v);
                        } else if (EARLY) {
#pragma unroll
                            for (int i = 0; i < 32; ++i) v[i] = 0.f;
                        }
                        if (!CHAIN && (!EARLY || j >= 0) && 32 * (j + 1) >= cols && 32 * j < cols) {  // the last of them: the accumulators are read
                            t5_fence_before();
                            __syncwarp();
                            if (lane == 0 && pc + 2 < all) t5_arrive_cluster(empty0 + 8 * b);
                        }
                        const int here = EARLY ? 32 * max(j, 0) : 32 * j, ahead = 32 * (j + 1), count = min(live - here, 32), c = c0 + here;
                        if (count > 0) {
                            if (ROWS_M && a.bias[m]) {
                                float next[32];
                                dense_load32(next, a.bias[m], c, 1, a.bias_type, count);
#pragma unroll
                                for (int i = 0; i < 32; ++i) v[i] += next[i];
                            }
                            if (MATS == 1) {
                                float next[32];
                                if (a.residual && CHAIN) load(next, a.residual, c, a.rs, a.residual_type, count);
                                if (a.residual && !CHAIN && live > ahead) load(next, a.residual, c0 + ahead, a.rs, a.residual_type, min(live - ahead, 32));
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
                                // (CHAIN: act(gate) waits in its places of the fp32 output, or behind the sums)
                                float gate[32];
                                if (CHAIN && !parked) load(gate, a.out, c, a.os, GLMFLASH_F32, count);
                                else if (CHAIN)
#pragma unroll
                                    for (int i = 0; i < 32; ++i) gate[i] = keep[2][i];
#pragma unroll
                                for (int i = 0; i < 32; ++i) {
                                    v[i] += bias;
                                    if (a.limit > 0.f) v[i] = dense_within(v[i], a.limit);
                                    v[i] *= CHAIN ? gate[i] : keep[0][i];
                                }
                            }
                            if (MATS == 1 || m == 1 || (CHAIN && !parked)) {
                                const int stored = EARLY && j < 0 ? 0 : count;
                                if (ROWS_M) dense_store_along(v, a.out, place(c, a.os), a.out_type, stored);
                                else dense_store32(v, a.out, place(c, a.os), a.os, a.out_type, stored);
                            }
                        }
                        if (CHAIN || MATS == 2)
#pragma unroll
                            for (int i = 0; i < 32; ++i) {
                                keep[0][i] = keep[1][i];
                                keep[1][i] = keep[2][i];
                                keep[2][i] = keep[3][i];
                                if (MATS == 2) keep[3][i] = v[i];
                            }
                    }
                }
                if (!ok) break;
            }
        }
        if (!ok) t5_settle();
    }
    t5_fence_before();
    // the pair ends together (not the aligned form: single lanes worked alone;  relaxed: what was stored to global memory need not have arrived)
    asm volatile("barrier.cluster.arrive.relaxed;\n\tbarrier.cluster.wait;" ::: "memory");
    t5_fence_after();
    if (warp == 2) t5_dealloc<2>(tmem, 512);
}

// ---------------------------------------------------------------------------------------------------------- few tiles
// Too few tiles for a pair each: single CTAs (128 output columns x up to 256 rows) of a CLUSTER that cuts K between them.  Each multiplies its
// part, and sends the sums in fours of rows to the CTA of the cluster that finishes them (distributed shared memory, one way, 16 bytes a
// lane); after a cluster barrier that one adds the parts in ascending order and runs the epilogue.
//   warps 0, 2 copy weights and rows;  warp 1 allocates tensor memory and issues the products;  warps 4-11 epilogue
// us, calls one behind another: 17 x 2048 x 1536 4.1, 45 x 4096 x 4096 7.0, gated 200 x 4096 x 512 8.2 (77 MB through L2 for 10 MB of operands: K cut four
// ways, 32 rows a tile, copies of 112 CTAs).  Sending the parts with stores that count on a barrier of their receiver, in place of the cluster's barrier: 4.0, -, 9.4.
constexpr int DT_THREADS = 384, DT_DEPTH = 8, DT_SMEM = 224 * 1024;

struct DenseThin {
    int t, share, more, chains;                              // rows of a tile (in 16), stages of a CTA, CTAs that have one more, sums of at most 512 k a CTA
    int depth, copies, slots, alias, cols;                   // stages of the ring, copies that bring a stage of an operand, fours of rows a CTA finishes, the parts lie over the ring, tensor memory
};

template <int MATS>
__global__ void __launch_bounds__(DT_THREADS, 1)
dense_thin_kernel(const __grid_constant__ DenseMaps maps, const DenseArgs a, const DenseThin d) {
    extern __shared__ unsigned char smem_raw[];
    unsigned char *ring = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    __shared__ uint64_t full[DT_DEPTH], done[DT_DEPTH], acc_full;
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_word;
    volatile int *abort_flag = &abort_word;
    int *status = &dense_status_word;
    const int tid = threadIdx.x, warp = tid >> 5;
    // (A cluster is a row of the grid.  Divisions at the start and the end of a call of 5 us cost a tenth of it.)
    const uint32_t cn = gridDim.x;
    const int rank = blockIdx.x, n0 = blockIdx.z * 128, r0 = blockIdx.y * d.t;
    const int first = rank * d.share + min(rank, d.more), mine = d.share + (rank < d.more);              // stages of this CTA
    const uint32_t bytes = MATS * DW_A + (uint32_t)d.t * DW_K * 2;
    float4 *parts = reinterpret_cast<float4 *>(ring + (d.alias ? 0 : (size_t)d.depth * bytes));       // [cn][slots][MATS][128]
    if (tid < DT_DEPTH) {
        mbar_init(full + tid, 2);
        mbar_init(done + tid, 1);
        if (tid == 0) {
            mbar_init(&acc_full, 1);
            abort_word = 0;
        }
        mbar_fence_init();
    }
    // (by a warp that has nothing else to do: 2048 x 512 4.95 us instead of 5.12)
    if (tid >= 96 && tid <= 96 + MATS) asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)(tid == 96 ? &maps.b[0] : &maps.a[tid - 97])) : "memory");
    __syncthreads();
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");     // (waited for in front of the first store to a peer)
    bool ok = true;
    if (warp == 0 || warp == 2) {                            // (they do not wait for the tensor memory)
        pdl_wait();
        T5Ring at;
        const bool leader = t5_elect();
        int copied = 0;                                      // stages that this lane has copied
#pragma unroll 1
        for (int it = 0; it < mine; ++it) {
            if (it >= d.depth) ok &= t5_wait<200>(done + at.slot, at.parity ^ 1, abort_flag, status, GF_STATUS_TMA_TIMEOUT);
            if (leader) {
                if (ok) {
                    unsigned char *dst = ring + (size_t)at.slot * bytes;
                    mbar_expect_tx(full + at.slot, warp ? d.t * DW_K * 2 : MATS * DW_A);
                    if (warp == 0)
                        for (int m = 0; m < MATS; ++m)
                            dense_copy(dst + m * DW_A, first + it, 128, d.copies, [&](unsigned char *to, int k) { t5_load(to, &maps.a[m], d.copies == 1, k, n0, full + at.slot); });
                    else
                        dense_copy(dst + MATS * DW_A, first + it, d.t, d.copies, [&](unsigned char *to, int k) { t5_load(to, &maps.b[0], d.copies == 1, k, r0, full + at.slot); });
                    ++copied;
                }
            }
            __syncwarp();
            at.next(d.depth);
        }
        // after a give-up: copies in flight have landed before the CTA leaves
        if (!ok || *abort_flag)
            for (int k = max(copied - d.depth, 0); k < copied; ++k) mbar_wait(full + k % d.depth, (k / d.depth) & 1, nullptr, 1000u);
    } else if (warp == 1) {
        // (The next kernel of the stream may start only now: one that took the SM's tensor memory first would wait for this one, which waits for it.)
        t5_alloc<1>(&tmem_slot, d.cols);
        pdl_launch_dependents();
        pdl_wait();
        t5_fence_before();
        asm volatile("barrier.sync 1, 288;" ::: "memory");   // the epilogue warps may read where it is
        const uint32_t tmem = tmem_slot;
        const uint32_t idesc = t5_idesc(128, d.t, a.type == GLMFLASH_BF16);
        const uint64_t desc0 = t5_desc(smem_u32(ring));
        const uint32_t next = d.t * 128 >> 4;
        const int chain = d.chains > 1 ? (mine + d.chains - 1) / d.chains : mine;
        int in_chain = 0;
        const bool leader = t5_elect();
        uint32_t acc = tmem;
        T5Ring at;
        for (int it = 0; it < mine; ++it) {
            ok &= t5_wait<0>(full + at.slot, at.parity, abort_flag, status, GF_STATUS_MMA_TIMEOUT);       // (a vote a stage costs 90 clocks of each)
            const uint64_t da = desc0 + at.slot * (bytes >> 4), db = da + (MATS * DW_A >> 4);
            if (in_chain == chain) {                         // the next sum
                in_chain = 0;
                acc += d.t;
            }
            // (A stage is always multiplied whole, zeros behind K and all: a branch around each product made each take 200 clocks.)
            if (leader) {
#pragma unroll
                for (int m = 0; m < MATS; ++m)
#pragma unroll
                    for (int k = 0; k < DW_K / 16; ++k)
                        t5_mma<1>(acc + m * d.chains * d.t, da + m * (DW_A >> 4) + 2 * (k & 3) + (k >> 2) * (128 * 128 >> 4), db + 2 * (k & 3) + (k >> 2) * next, idesc,
                                  k > 0 ? 1u : in_chain > 0);
                if (it + d.depth < mine) t5_commit<1>(done + at.slot);             // (somebody waits for it)
            }
            ++in_chain;
            at.next(d.depth);
            __syncwarp();
        }
        if (leader) t5_commit<1>(&acc_full);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) t5_settle();
    } else if (warp >= 4) {
        pdl_wait();
        asm volatile("barrier.sync 1, 288;" ::: "memory");
    }
    __syncwarp();
    // The four rows `four` are finished by CTA four % cn, as its slot four / cn (counted along: a division takes 40 instructions).
    const int live = min(d.t, a.rows - r0), fours = (live + 3) >> 2, q = warp & 3, half = (warp - 4) >> 2, col = (tid - 128) & 127, n = n0 + col;
    const int groups = (live + 31) >> 5, from = half ? (groups + 1) >> 1 : 0, to = half ? groups : (groups + 1) >> 1;
    uint32_t slot = 8 * from / cn, owner = 8 * from % cn;
    float b[2] = {0.f, 0.f};
    if (warp >= 4) {
        dense_biases<MATS>(a, n, b);
        ok = __all_sync(0xffffffffu, t5_wait<100>(&acc_full, 0, abort_flag, status, GF_STATUS_MMA_TIMEOUT));
        t5_fence_after();
    }
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (d.alias) cluster_sync();                             // every CTA has multiplied: the ring is free
    if (warp >= 4 && ok) {
        int used = 1;                                        // sums that stages fell to
        if (d.chains > 1) {
            const int chain = (mine + d.chains - 1) / d.chains;
            used = (mine + chain - 1) / chain;
        }
        const uint32_t lanes = tmem_slot + ((uint32_t)(q * 32) << 16);
#pragma unroll 1
        for (int j = from; j < to; ++j) {
            float v[MATS][32];
#pragma unroll
            for (int m = 0; m < MATS; ++m) {
                const uint32_t at = lanes + m * d.chains * d.t + 32 * j;
                t5_ld32(at, v[m]);
#pragma unroll 1
                for (int c = 1; c < used; ++c) {
                    float w[32];
                    t5_ld32(at + c * d.t, w);
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[m][i] += w[i];
                }
            }
            if (cn == 1) {                                   // nothing to add
                const int64_t r = r0 + 32 * j;
                const int count = n < a.N ? min(32, live - 32 * j) : 0;
                if (count > 0) {
                    float res[32];
                    if (MATS == 1 && a.residual) dense_load32(res, a.residual, r * a.rs + n, a.rs, a.residual_type, count);
                    dense_act32<MATS>(a, v[0], b[0]);
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        if (MATS == 1 && a.residual) v[0][i] += res[i];
                        if (MATS == 2) {
                            float u = v[MATS - 1][i] + b[1];
                            if (a.limit > 0.f) u = dense_within(u, a.limit);
                            v[0][i] *= u;
                        }
                    }
                    dense_store32(v[0], a.out, r * a.os + n, a.os, a.out_type, count);
                }
                __syncwarp();
                continue;
            }
            const uint32_t here = smem_u32(parts + rank * d.slots * MATS * 128 + col);
#pragma unroll
            for (int g = 0; g < 8; ++g) {
                if (8 * j + g < fours) {
                    uint32_t peer;
                    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(peer) : "r"(here + slot * (MATS * 2048)), "r"(owner));
#pragma unroll
                    for (int m = 0; m < MATS; ++m)
                        asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(peer + m * 2048), "f"(v[m][4 * g]), "f"(v[m][4 * g + 1]),
                                     "f"(v[m][4 * g + 2]), "f"(v[m][4 * g + 3]) : "memory");
                }
                if (++owner == cn) { owner = 0; ++slot; }
            }
        }
    }
    t5_fence_before();
    const bool sound = !*abort_flag;
    __syncwarp();
    cluster_sync();                                          // the parts of all CTAs have come in
    t5_fence_after();
    if (warp == 1) t5_dealloc<1>(tmem_slot, d.cols);
    if (warp < 4 || cn == 1 || !sound || n >= a.N) return;
#pragma unroll 1
    for (int s = half; s * (int)cn + rank < fours; s += 2) {
        float v[MATS][4];
        const float4 *p = parts + s * MATS * 128 + col;
#pragma unroll
        for (int m = 0; m < MATS; ++m) *reinterpret_cast<float4 *>(v[m]) = p[m * 128];
#pragma unroll 1
        for (int c = 1; c < (int)cn; ++c) {
            p += d.slots * MATS * 128;
#pragma unroll
            for (int m = 0; m < MATS; ++m) {
                const float4 w = p[m * 128];
                v[m][0] += w.x; v[m][1] += w.y; v[m][2] += w.z; v[m][3] += w.w;
            }
        }
        const int r = (s * (int)cn + rank) * 4;
        dense_finish<MATS>(a, [&](int i) { return r0 + r + i; }, r0 + live, n, v[0], v[MATS - 1], b);
    }
}

// [rows][stride] of 16-bit elements: copies of `box` rows x 64 elements, or x 128 as two blocks of 64 (copies == 1)
static int dense_map(CUtensorMap *map, const void *base, bool bf, int64_t rows, int K, int64_t stride, int box, int copies, const char *what) {
    const auto type = bf ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    const uint32_t boxes[3] = {64, (uint32_t)box, 2};
    const uint64_t blocks[3] = {64, (uint64_t)rows, (uint64_t)K / 64}, dims[2] = {(uint64_t)K, (uint64_t)rows}, strides[2] = {(uint64_t)stride * 2, 128};
    return encode_map(map, type, copies == 1 ? 3 : 2, const_cast<void *>(base), copies == 1 ? blocks : dims, strides, boxes, what);
}

// What a device holds: SMs, and clusters of each size (one CTA an SM; they do not span its clusters of SMs).
struct DenseDevice { int sms, clusters[9]; };
static int dense_device(const DenseDevice **out) {
    static DenseDevice known[64] = {};                       // (threads that come here together set the same)
    static std::atomic<bool> ready[64] = {};
    int dev = 0;
    GF_CUDA(cudaGetDevice(&dev));
    GF_REQUIRE(dev >= 0 && dev < 64, "device ordinal out of range");
    if (!ready[dev].load(std::memory_order_acquire)) {
        for (auto k : {dense_wide_kernel<1, false, false>, dense_wide_kernel<1, true, false>, dense_wide_kernel<2, false, false>, dense_wide_kernel<2, true, false>,
                       dense_wide_kernel<1, false, true>, dense_wide_kernel<1, true, true>, dense_wide_kernel<2, false, true>, dense_wide_kernel<2, true, true>})
            GF_CUDA(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)DW_SMEM));
        for (auto k : {dense_thin_kernel<1>, dense_thin_kernel<2>}) GF_CUDA(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, DT_SMEM));
        DenseDevice d = {};
        GF_CUDA(cudaDeviceGetAttribute(&d.sms, cudaDevAttrMultiProcessorCount, dev));
        for (int cn = 1; cn <= 8; ++cn) {
            cudaLaunchConfig_t cfg = {};
            cudaLaunchAttribute at[1];
            at[0].id = cudaLaunchAttributeClusterDimension;
            at[0].val.clusterDim.x = (unsigned)cn;
            at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
            cfg.gridDim = dim3((unsigned)(cn * d.sms));
            cfg.blockDim = dim3(DT_THREADS);
            cfg.dynamicSmemBytes = DT_SMEM;
            cfg.attrs = at;
            cfg.numAttrs = 1;
            GF_CUDA(cudaOccupancyMaxActiveClusters(&d.clusters[cn], dense_thin_kernel<1>, &cfg));
        }
        for (int cn = 1; cn <= 8; ++cn) known[dev].clusters[cn] = d.clusters[cn];
        known[dev].sms = d.sms;
        ready[dev].store(true, std::memory_order_release);
    }
    *out = &known[dev];
    return 0;
}

// a and b of the maps: the weights with boxes of 128 and x with boxes of n_box rows, or the roles exchanged
static int dense_maps(DenseMaps *maps, const DenseArgs &a, bool rows_m, int n_box, int copies) {
    const bool bf = a.type == GLMFLASH_BF16;
    CUtensorMap *w = rows_m ? maps->b : maps->a, *x = rows_m ? maps->a : maps->b;
    const int w_box = rows_m ? n_box : 128, x_box = rows_m ? 128 : n_box;
    if (dense_map(&w[0], a.w[0], bf, a.N, a.K, a.ws[0], w_box, copies, "weights") || dense_map(&x[0], a.x, bf, a.rows, a.K, a.xs, x_box, copies, "rows")) return -1;
    if (a.w[1] && dense_map(&w[1], a.w[1], bf, a.N, a.K, a.ws[1], w_box, copies, "weights")) return -1;
    if (!a.w[1]) w[1] = w[0];
    x[1] = x[0];
    return 0;
}

int dense_gemm(cudaStream_t s, const DenseArgs &a, bool pdl) {
    const DenseDevice *device;
    if (dense_device(&device)) return -1;
    const int pairs = device->sms / 2, mats = a.w[1] ? 2 : 1, stages = (a.K + DW_K - 1) / DW_K, copies = a.K % 64 ? 2 : 1;
    const int pass = a.out_type == GLMFLASH_F32 ? DW_CHAIN : DW_CHAIN16;
    const bool chain = stages > pass, parked = chain && mats == 2 && a.out_type != GLMFLASH_F32;
    // ns of either kernel with any tiles, fitted to 3520 times (17 to 4096 rows, K 504 to 8192, 288 to 8192 outputs): what this takes is on average 2 %
    // behind the best of them.  One term is not the fit's: 2.4 clocks and not 2.64 for each of N, so that the larger of two tiles that come out alike is taken, which
    // at the power limit is the faster one (8192 x 4096 x 4096 with N of 256, 224, 192 on one GPU: 208, 214, 222 us).
    // Wide: N of a tile and the operand along M.  Rounds of tiles over the pairs: a stage takes its copies' turns, 4 clocks and more for each of N on
    // the tensor cores, or its bytes once all pairs copy;  the epilogue (whole rows of outputs a lane, exchanged, cost as little only if they can
    // be stored in 16 bytes) hides behind the next tile's products.
    const int size = a.out_type == GLMFLASH_F32 ? 4 : 2;
    const bool vectors = ((uintptr_t)a.out | a.os * size | (int64_t)a.N * size) % 16 == 0;
    const double halves = copies == 2 ? 1. : 0.;             // (two copies a stage)
    DenseTiles d = {};
    bool rows_m = false;
    d.stages = stages;
    d.pass = chain ? pass : stages;
    double wide = 1e30;
    for (int exchanged = 0; exchanged < 2; ++exchanged) {
        const int across = ((exchanged ? a.rows : a.N) + 255) / 256, along = exchanged ? a.N : a.rows;
        for (int bn = 32; bn <= (parked ? DW_ROWS / 2 : DW_ROWS); bn += 32) {         // (N of a pair's product goes in 32)
            const int64_t tiles = (int64_t)((along + bn - 1) / bn) * across;
            const int64_t rounds = (tiles + pairs - 1) / pairs;
            const double busy = std::min(1., (double)tiles / pairs);
            const double stage = std::max({256. + 231. * halves, 60. + 2.4 * bn, busy * (191. + 1.29 * bn) + 231. * halves});
            const double body = mats * (stages * stage + (chain ? 350. * stages / pass : 0.)), end = 939. + bn * (!exchanged ? 10.3 : vectors ? 13.3 : 60.);
            const double ns = 2120. + body + end + (rounds - 1) * std::max(body, end);
            if ((exchanged ? ns < wide : ns <= wide) && tiles <= INT32_MAX / 2) { wide = ns; rows_m = exchanged; d.bn = bn; d.across = across; d.tiles = (int)tiles; }
        }
    }
    GF_REQUIRE(wide < 1e30 && (int64_t)(d.tiles / pairs + 1) * mats * stages < INT32_MAX, "the product is too large");
    // Thin: rows of a tile and CTAs that cut K.  (Operands beyond what L2 holds at hand: its copies, twice those of pairs, wait for them. 4096 rows, 8192 x
    // 1024: 74 us, pairs 50.)
    const double beyond = ((int64_t)a.rows + (int64_t)mats * a.N) * a.K > 24 << 20 ? 0.75 : 0.;
    DenseThin h = {};
    int cluster = 0, row_split = 0;
    double thin = 1e30;
    const int across = (a.N + 127) / 128;
    for (int tiles = 1; tiles <= 64; ++tiles) {
        const int t = ((a.rows + tiles - 1) / tiles + 15) / 16 * 16, row_tiles = (a.rows + t - 1) / t;
        if (t > 256 || row_tiles < tiles) continue;
        for (int cn = 1; cn <= 8 && cn <= stages; ++cn) {
            if ((int64_t)across * row_tiles > device->clusters[cn]) continue;
            const int most = (stages + cn - 1) / cn, chains = chain ? (most + pass - 1) / pass : 1, bytes = mats * DW_A + t * DW_K * 2;
            const int slots = (t / 4 + cn - 1) / cn, parts = cn == 1 ? 0 : cn * slots * mats * 2048, need = mats * chains * t + (t % 32 ? 16 : 0);
            if (need > 512 || parts > DT_SMEM - 1024) continue;
            const int room = DT_SMEM - 1024 - parts, apart = std::min(room / bytes, most);
            const bool alias = apart < std::min(3, most);
            const int depth = std::min({alias ? (DT_SMEM - 1024) / bytes : apart, most, DT_DEPTH});
            if (depth < std::min(2, most)) continue;
            const double mma = mats * 8 * std::max({41., 33. + 0.25 * t, 0.5 * t}) / 1.9 + 130.;
            const double work = std::max({mma, bytes / 150., bytes * (double)(across * row_tiles * cn) / 9000.});
            const double stage = std::max((cn == 1 ? 243. + 0.317 * work : 168. + 0.278 * work) + 185. * halves, beyond * work);
            const double ns = cn == 1 ? 1257. + most * stage + 24.8 * mats * t : 2150. + most * stage + slots * mats * (78. + 114. * cn);
            if (ns < thin) {
                thin = ns;
                cluster = cn;
                row_split = row_tiles;
                h = {t, stages / cn, stages % cn, chains, depth, copies, slots, alias, need <= 32 ? 32 : need <= 64 ? 64 : need <= 128 ? 128 : need <= 256 ? 256 : 512};
            }
        }
    }
    DenseMaps maps;
    if (thin < wide) {
        if (dense_maps(&maps, a, false, h.t, copies)) return -1;
        const int bytes = mats * DW_A + h.t * DW_K * 2, parts = cluster == 1 ? 0 : cluster * h.slots * mats * 2048;
        // At least the share of the shared memory that it takes of the tensor memory: CTAs that fit on an SM side by side (of two streams) then never
        // wait for each other's tensor memory, which CTAs of two clusters could do crosswise, and for good.
        const size_t smem = std::max<size_t>(1024 + (h.alias ? std::max(h.depth * bytes, parts) : h.depth * bytes + parts), (size_t)DT_SMEM * h.cols / 512);
        return launch_kc(mats == 2 ? dense_thin_kernel<2> : dense_thin_kernel<1>, dim3((unsigned)cluster, (unsigned)row_split, (unsigned)across), dim3(DT_THREADS),
                         dim3((unsigned)cluster), smem, s, pdl, maps, a, h);
    }
    d.copies = copies;
    const int walking = std::min(d.tiles, pairs);
    d.step_m = walking % d.across;
    d.step_n = walking / d.across;
    d.depth = std::min(DW_RING / (DW_A + d.bn * 128), DW_DEPTH);
    if (dense_maps(&maps, a, rows_m, d.bn / 2, copies)) return -1;
    auto kernel = rows_m ? (mats == 2 ? (chain ? dense_wide_kernel<2, true, true> : dense_wide_kernel<2, false, true>)
                                      : (chain ? dense_wide_kernel<1, true, true> : dense_wide_kernel<1, false, true>))
                         : (mats == 2 ? (chain ? dense_wide_kernel<2, true, false> : dense_wide_kernel<2, false, false>)
                                      : (chain ? dense_wide_kernel<1, true, false> : dense_wide_kernel<1, false, false>));
    return launch_k(kernel, dim3((unsigned)(2 * walking)), dim3(DW_THREADS), DW_SMEM, s, pdl, maps, a, d);
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
