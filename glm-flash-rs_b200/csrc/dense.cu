// Dense products beside the quantised ones: out = act(x . w^T + bias) + residual and the gated pair
// out = act(min(x . wg^T + bg, limit)) * clamp(x . wu^T + bu, -limit, limit), fp16 or bf16 operands, fp32 sums, one rounding at the end.
// The projections around the expert path that a checkpoint keeps dense (the shared expert of an upstream bank, a vocabulary head).
#include "dense.cuh"
#include "select.cuh"

namespace gf {

template <bool BF>
__device__ __forceinline__ void dense_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if (BF)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Eight elements of a row from k on, zeros behind K: what lies there between the rows of a wider buffer counts for nothing.
__device__ __forceinline__ uint4 dense_piece(const uint16_t *row, int k, int K) {
    if (k + 8 <= K) return *reinterpret_cast<const uint4 *>(row + k);
    uint32_t v[4] = {0u, 0u, 0u, 0u};
    for (int i = 0; k + i < K; ++i) v[i >> 1] |= (uint32_t)row[k + i] << (i & 1) * 16;
    return make_uint4(v[0], v[1], v[2], v[3]);
}

__device__ __forceinline__ uint4 dense_ldg(const void *p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

// Up to 8 RT rows: bound by the latency of one trip to the weights.  A CTA has 16 output columns, its 16 warps cut K into steps of 32 and ask for
// several steps each before the first product.  The weights are the 16-row operand of mma.m16n8k16, the rows the 8-column
// one.  The k slots of a fragment may be any as long as both operands agree: a lane loads 16 contiguous bytes of a row (k = 8 t .. 8 t + 7 of a step) and
// uses them as the fragments of two instructions.
constexpr int DN_N = 16, DN_WARPS = 16, DN_AHEAD = 4;
// start() once the kernel in front has ended, finish(row, column, sums) for what this thread has of them.
template <bool BF, int MATS, int RT, typename S, typename F>
__device__ __forceinline__ void dense_columns(const DenseArgs &a, int n0, S start, F finish, float (&part)[DN_WARPS][MATS][8 * RT][DN_N + 1]) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3, whole = a.K >> 5;
    const uint16_t *w[MATS][2];
#pragma unroll
    for (int m = 0; m < MATS; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) w[m][h] = static_cast<const uint16_t *>(a.w[m]) + min(n0 + 8 * h + g, a.N - 1) * a.ws[m] + 8 * t;   // (columns behind the last: the last's)
#pragma unroll
    for (int m = 0; m < MATS; ++m)                           // (a hint: the lines are on their way to L2 while the kernel in front ends)
#pragma unroll
        for (int i = 0; i < DN_AHEAD; ++i)
            if (warp + DN_WARPS * i < whole) {
                asm volatile("prefetch.global.L2 [%0];" ::"l"(w[m][0] + (warp + DN_WARPS * i) * 32));
                asm volatile("prefetch.global.L2 [%0];" ::"l"(w[m][1] + (warp + DN_WARPS * i) * 32));
            }
    pdl_wait();
    pdl_launch_dependents();
    start();
    const uint16_t *x = static_cast<const uint16_t *>(a.x) + g * a.xs + 8 * t;
    float acc[MATS][RT][4] = {};
    const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
    auto multiply = [&](const uint4 (&wv)[MATS][2], const uint4 (&xv)[RT]) {
#pragma unroll
        for (int m = 0; m < MATS; ++m)
#pragma unroll
            for (int i = 0; i < RT; ++i) {
                dense_mma<BF>(acc[m][i], wv[m][0].x, wv[m][1].x, wv[m][0].y, wv[m][1].y, xv[i].x, xv[i].y);
                dense_mma<BF>(acc[m][i], wv[m][0].z, wv[m][1].z, wv[m][0].w, wv[m][1].w, xv[i].z, xv[i].w);
            }
    };
#pragma unroll 1
    for (int s0 = warp; s0 < whole; s0 += DN_WARPS * DN_AHEAD) {
        uint4 wv[DN_AHEAD][MATS][2], xv[DN_AHEAD][RT];
#pragma unroll
        for (int i = 0; i < DN_AHEAD; ++i) {
            const int s = s0 + DN_WARPS * i;
            const bool here = s < whole;
#pragma unroll
            for (int m = 0; m < MATS; ++m)
#pragma unroll
                for (int h = 0; h < 2; ++h) wv[i][m][h] = here ? dense_ldg(w[m][h] + s * 32) : zero;
#pragma unroll
            for (int j = 0; j < RT; ++j) xv[i][j] = here && 8 * j + g < a.rows ? dense_ldg(x + 8 * j * a.xs + s * 32) : zero;
        }
#pragma unroll
        for (int i = 0; i < DN_AHEAD; ++i) multiply(wv[i], xv[i]);
    }
    if ((a.K & 31) && warp == whole % DN_WARPS) {            // the ragged end of K
        uint4 wv[MATS][2], xv[RT];
        const int k = whole * 32 + 8 * t;
#pragma unroll
        for (int m = 0; m < MATS; ++m)
#pragma unroll
            for (int h = 0; h < 2; ++h) wv[m][h] = k < a.K ? dense_piece(w[m][h] - 8 * t, k, a.K) : zero;
#pragma unroll
        for (int j = 0; j < RT; ++j) xv[j] = 8 * j + g < a.rows && k < a.K ? dense_piece(x + 8 * j * a.xs - 8 * t, k, a.K) : zero;
        multiply(wv, xv);
    }
#pragma unroll
    for (int m = 0; m < MATS; ++m)
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            part[warp][m][8 * i + 2 * t][g] = acc[m][i][0];
            part[warp][m][8 * i + 2 * t + 1][g] = acc[m][i][1];
            part[warp][m][8 * i + 2 * t][g + 8] = acc[m][i][2];
            part[warp][m][8 * i + 2 * t + 1][g + 8] = acc[m][i][3];
        }
    __syncthreads();
    const int r = tid / DN_N, n = tid % DN_N;
    if (tid >= 8 * RT * DN_N || r >= a.rows || n0 + n >= a.N) return;
    float v[MATS][1];
#pragma unroll
    for (int m = 0; m < MATS; ++m) {
        v[m][0] = 0.f;
#pragma unroll
        for (int k = 0; k < DN_WARPS; ++k) v[m][0] += part[k][m][r][n];
    }
    finish(r, n0 + n, v);
}
template <bool BF, int MATS, int RT>
__global__ void __launch_bounds__(DN_WARPS * 32, MATS * RT == 1 ? 2 : 1) dense_kernel(const DenseArgs a) {
    __shared__ float part[DN_WARPS][MATS][8 * RT][DN_N + 1];
    dense_columns<BF, MATS, RT>(a, blockIdx.x * DN_N, [] {}, [&](int r, int n, float (&v)[MATS][1]) {
        float b[2];
        dense_biases<MATS>(a, n, b);
        dense_finish<MATS>(a, [&](int) { return r; }, a.rows, n, v[0], v[MATS - 1], b);
    }, part);
}

// The router of up to 16 rows in one launch: a cluster of up to eight CTAs has the columns between them and sends each logit to the shared memory of the
// CTA whose warp selects that row.  Two launches wait for the first one's stores and end, and cost the host
// 2 us more.  us in a graph, 2048 x 64, 1, 8 and 16 rows: 4.3, 4.7, 5.3 instead of 5.0, 5.4, 6.0; 4096 x 128, 1 row: 5.2 instead of 6.2.  With two blocks of
// columns a CTA (2048 x 256, 1 row) the one launch takes 7.6, two 5.4.
template <int RT>
__global__ void __launch_bounds__(DN_WARPS * 32, 1) dense_route_kernel(const DenseArgs a, const float *bias, int topk, SelRule rule, int *picks, float *weights) {
    extern __shared__ double route_values[];                 // of each of this CTA's rows: keys, biases, logits
    __shared__ float part[DN_WARPS][1][8 * RT][DN_N + 1];
    __shared__ int2 spot[DN_WARPS][32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, cn = gridDim.x, r = blockIdx.x + warp * cn, wide = (a.N + 31) / 32 * 32;
    float *keys = reinterpret_cast<float *>(route_values) + warp * 3 * wide;
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");     // (waited for in front of the first store to a peer)
    int row = -1, column = 0;
    float logit = 0.f;
    auto fetch = [&] {
        if (r >= a.rows) return;
        if (bias) sel_fetch(keys + wide, bias, a.N, lane);
        sel_pad(keys, a.N, bias != nullptr, lane);
    };
    dense_columns<true, 1, RT>(a, blockIdx.x * DN_N, fetch, [&](int r, int n, float (&v)[1][1]) { row = r; column = n; logit = v[0][0]; }, part);
    __syncwarp();
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (row >= 0) {
        float *to = const_cast<float *>(cluster_map(reinterpret_cast<float *>(route_values) + row / cn * 3 * wide + column, row % cn));
        to[0] = to[2 * wide] = logit;
    }
    __syncwarp();
    cluster_sync();
    if (row >= 0) static_cast<float *>(a.out)[row * a.os + column] = logit;
    if (r < a.rows) select_row<true>(keys + 2 * wide, bias, a.N, topk, rule, keys, spot[warp], picks + r * (topk + 1), weights + r * (topk + 1), lane);
}

// Which calls of up to 16 rows it takes: those whose CTAs run at once (two an SM for one matrix and up to 8 rows), with few trips a warp.  us, this
// kernel | the tensor-memory ones, inner x outer, 1 and 8 rows: 512 x 512 2.1 2.1 | 3.3 3.1; 2048 x 2048 3.1 3.5 | 4.3 4.3; 2048 x 4096 4.3 4.9
// | 5.2 5.2; 4096 x 4096 6.3 7.8 | 6.6 6.4; 8192 x 1024 6.5 7.0 | 5.6 5.8; 2048 x 8192 8.0 9.1 | 6.6 6.2.  9 and 16 rows: 2048 x 2048 3.4 4.2 |
// 4.3 4.4; 4096 x 2048 5.6 5.9 | 5.4 5.4; 2048 x 4096 6.2 7.0 | 5.2 5.1.  The gated pair, 1, 8, 9, 16 rows: 2048 x 2048 4.2 4.5 4.9 5.8 | 5.8 5.6
// 6.0 5.8; 4096 x 2048 5.8 6.2 7.0 7.5 | 7.7 7.5 8.0 7.8; 8192 x 1024 8.1 9.0 10.1 11.0 | 8.5 8.3 8.8 8.6; 2048 x 4096 7.9 8.6 9.2 10.1 | 7.2 6.8 7.2 6.8.
static bool dense_small(const DenseArgs &a) {
    if (a.rows > 16 || a.K > 4096 || a.N > 148 * 2 * DN_N) return false;
    if (a.w[1]) return a.N <= 148 * DN_N;
    return a.rows <= 8 ? (int64_t)a.K * a.N <= 1 << 23 : a.K <= 2048 && a.N <= 148 * DN_N;
}

template <bool BF, int MATS>
static int launch_dense(cudaStream_t s, const DenseArgs &a, bool pdl) {
    const dim3 grid((unsigned)((a.N + DN_N - 1) / DN_N)), block(DN_WARPS * 32);
    return a.rows > 8 ? launch_k(dense_kernel<BF, MATS, 2>, grid, block, 0, s, pdl, a) : launch_k(dense_kernel<BF, MATS, 1>, grid, block, 0, s, pdl, a);
}

bool dense_route_fits(const DenseArgs &a) { return dense_small(a) && a.N <= 8 * DN_N; }
int dense_route(cudaStream_t s, const DenseArgs &a, const float *bias, int topk, const SelRule &rule, int *picks, float *weights, bool pdl) {
    const int cn = std::min((a.N + DN_N - 1) / DN_N, 8);
    const size_t smem = (size_t)((a.rows + cn - 1) / cn) * ((a.N + 31) / 32 * 32) * 3 * sizeof(float);
    return launch_kc(a.rows > 8 ? dense_route_kernel<2> : dense_route_kernel<1>, dim3((unsigned)cn), dim3(DN_WARPS * 32), dim3((unsigned)cn), smem, s, pdl, a, bias, topk, rule,
                     picks, weights);
}

}  // namespace gf

using namespace gf;

extern "C" size_t glmflash_linear_args_bytes(void) { return sizeof(glmflash_linear_args); }

extern "C" int glmflash_linear(void *stream, const glmflash_linear_args *p, size_t bytes) {
    GF_REQUIRE(p != nullptr, "null argument");
    GF_REQUIRE(bytes == sizeof(glmflash_linear_args), "linear argument struct size mismatch");
    GF_REQUIRE(p->x && p->w && p->out, "null argument");
    const int32_t side = 1 << 30;
    GF_REQUIRE(p->rows > 0 && p->inner > 0 && p->outer > 0 && p->rows <= side && p->inner <= side && p->outer <= side,
               "rows, inner and outer must be in 1..2^30");
    GF_REQUIRE(p->type == GLMFLASH_F16 || p->type == GLMFLASH_BF16, "x and the weights must be fp16 or bf16");
    GF_REQUIRE(p->bias_type == GLMFLASH_F32 || p->bias_type == p->type, "a bias must be fp32 or of x's type");
    GF_REQUIRE(p->residual_type == GLMFLASH_F32 || p->residual_type == p->type, "the residual must be fp32 or of x's type");
    GF_REQUIRE(p->out_type == GLMFLASH_F32 || p->out_type == p->type, "the output must be fp32 or of x's type");
    GF_REQUIRE(p->act >= GLMFLASH_ACT_NONE && p->act <= GLMFLASH_ACT_RELU, "unknown activation");
    GF_REQUIRE(p->limit >= 0.f && p->limit - p->limit == 0.f, "limit must be finite and not negative (0: none)");
    const bool gated = p->w_up != nullptr;
    GF_REQUIRE(gated || (!p->bias_up && p->limit == 0.f), "bias_up and limit belong to the gated form (w_up)");
    GF_REQUIRE(!gated || !p->residual, "the gated form takes no residual");
    GF_REQUIRE(!p->reserved[0] && !p->reserved[1], "reserved fields must be 0");
    GF_REQUIRE(p->x_stride >= p->inner && p->w_stride >= p->inner && (!gated || p->w_up_stride >= p->inner), "strides of x and the weights must be >= inner");
    GF_REQUIRE(p->out_stride >= p->outer && (!p->residual || p->residual_stride >= p->outer), "strides of output and residual must be >= outer");
    GF_REQUIRE((p->x_stride | p->w_stride | (gated ? p->w_up_stride : 0)) % 8 == 0, "strides of x and the weights must be multiples of 8");
    GF_REQUIRE(((uintptr_t)p->x | (uintptr_t)p->w | (uintptr_t)p->w_up) % 16 == 0, "x and the weights must be 16-byte aligned");
    const int64_t most = (int64_t)1 << 38;                        // (strides in bytes below 2^40)
    GF_REQUIRE(p->x_stride < most && p->w_stride < most && (!gated || p->w_up_stride < most) && p->out_stride < most &&
                   (!p->residual || p->residual_stride < most), "stride too large");
    auto aligned = [](const void *q, int type) { return (uintptr_t)q % (type == GLMFLASH_F32 ? 4 : 2) == 0; };
    GF_REQUIRE(aligned(p->bias, p->bias_type) && aligned(p->bias_up, p->bias_type) && aligned(p->residual, p->residual_type) && aligned(p->out, p->out_type),
               "bias, residual and output must be aligned to their elements");
    DenseArgs a = {p->x, {p->w, p->w_up}, {p->bias, p->bias_up}, p->residual, p->out, p->x_stride, {p->w_stride, p->w_up_stride}, p->residual_stride,
                   p->out_stride, p->rows, p->inner, p->outer, p->type, p->bias_type, p->residual_type, p->out_type, p->act, p->limit};
    const bool bf = p->type == GLMFLASH_BF16, pdl = p->pdl != 0;
    cudaStream_t s = (cudaStream_t)stream;
    if (!dense_small(a)) return dense_gemm(s, a, pdl);
    if (gated) return bf ? launch_dense<true, 2>(s, a, pdl) : launch_dense<false, 2>(s, a, pdl);
    return bf ? launch_dense<true, 1>(s, a, pdl) : launch_dense<false, 1>(s, a, pdl);
}
