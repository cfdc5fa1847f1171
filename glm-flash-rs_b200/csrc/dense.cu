// Dense products beside the quantised ones: out = act(x . w^T + bias) + residual and the gated pair
// out = act(min(x . wg^T + bg, limit)) * clamp(x . wu^T + bu, -limit, limit), fp16 or bf16 operands, fp32 sums, one rounding at the end.
// The projections around the expert path that a checkpoint keeps dense (the shared expert of an upstream bank, a vocabulary head).
#include "dense.cuh"

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

// A CTA has 16 output columns of 8 RT rows; its 8 warps cut K.  The weights are the 16-row operand of mma.m16n8k16, the rows the 8-column
// one.  The k slots of a fragment may be any as long as both operands agree: a lane loads 16 contiguous bytes of a row (k = 8 t .. 8 t + 7
// of a 32-k step) and uses them as the fragments of two instructions.
constexpr int DN_N = 16, DN_WARPS = 8;
template <bool BF, int MATS, int RT>
__global__ void __launch_bounds__(DN_WARPS * 32) dense_kernel(const DenseArgs a, int row_tiles) {
    __shared__ float part[DN_WARPS][MATS][8 * RT][DN_N + 1];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    pdl_wait();
    pdl_launch_dependents();
    const int n0 = (int)(blockIdx.x / row_tiles) * DN_N, r0 = (int)(blockIdx.x % row_tiles) * 8 * RT;
    float acc[MATS][RT][4] = {};
    const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
    for (int s = warp; s * 32 < a.K; s += DN_WARPS) {
        const int k = s * 32 + 8 * t;
        uint4 xv[RT];
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            const int r = r0 + 8 * i + g;
            xv[i] = r < a.rows && k < a.K ? dense_piece(static_cast<const uint16_t *>(a.x) + r * a.xs, k, a.K) : zero;
        }
#pragma unroll
        for (int m = 0; m < MATS; ++m) {
            uint4 wv[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int n = n0 + 8 * h + g;
                wv[h] = n < a.N && k < a.K ? dense_piece(static_cast<const uint16_t *>(a.w[m]) + n * a.ws[m], k, a.K) : zero;
            }
#pragma unroll
            for (int i = 0; i < RT; ++i) {
                dense_mma<BF>(acc[m][i], wv[0].x, wv[1].x, wv[0].y, wv[1].y, xv[i].x, xv[i].y);
                dense_mma<BF>(acc[m][i], wv[0].z, wv[1].z, wv[0].w, wv[1].w, xv[i].z, xv[i].w);
            }
        }
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
    if (tid >= 8 * RT * DN_N) return;
    const int r = tid / DN_N, n = tid % DN_N;
    if (r0 + r >= a.rows || n0 + n >= a.N) return;
    float v[MATS][1], b[2];
    dense_biases<MATS>(a, n0 + n, b);
#pragma unroll
    for (int m = 0; m < MATS; ++m) {
        v[m][0] = 0.f;
#pragma unroll
        for (int w = 0; w < DN_WARPS; ++w) v[m][0] += part[w][m][r][n];
    }
    dense_finish<MATS>(a, r0 + r, n0 + n, 1, v[0], v[MATS - 1], b);
}

template <bool BF, int MATS>
static int launch_dense(cudaStream_t s, const DenseArgs &a, bool pdl) {
    const int rt = a.rows > 8 ? 2 : 1;
    const int64_t row_tiles = (a.rows + 8 * rt - 1) / (8 * rt), tiles = row_tiles * ((a.N + DN_N - 1) / DN_N);
    GF_REQUIRE(tiles <= INT32_MAX, "rows * outputs is too large");
    const dim3 grid((unsigned)tiles), block(DN_WARPS * 32);
    return rt == 2 ? launch_k(dense_kernel<BF, MATS, 2>, grid, block, 0, s, pdl, a, (int)row_tiles)
                   : launch_k(dense_kernel<BF, MATS, 1>, grid, block, 0, s, pdl, a, (int)row_tiles);
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
    if (p->rows > 16) return dense_gemm(s, a, pdl);
    if (gated) return bf ? launch_dense<true, 2>(s, a, pdl) : launch_dense<false, 2>(s, a, pdl);
    return bf ? launch_dense<true, 1>(s, a, pdl) : launch_dense<false, 1>(s, a, pdl);
}
