// What the kernels of the dense products share: arguments and epilogue.
#pragma once
#include "common.cuh"

namespace gf {

struct DenseArgs {
    const void *x, *w[2], *bias[2], *residual;
    void *out;
    int64_t xs, ws[2], rs, os;
    int rows, K, N, type, bias_type, residual_type, out_type, act;
    float limit;                                         // 0: none
};

__device__ __forceinline__ float dense_load(const void *p, int64_t i, int type) {
    if (type == GLMFLASH_F32) return static_cast<const float *>(p)[i];
    return type == GLMFLASH_F16 ? __half2float(static_cast<const __half *>(p)[i]) : __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
}
// v / (1 + exp(-x)) with the fast exponential (2 + 1.2 |x| units in the last place, which x (1 - s) s keeps below one of v) and quotient (2 units; 0
// for denominators beyond 2^126): off by less than 8 half steps of v.  The full ones took the epilogue of a gated tile nearly as long as its
// pass on the tensor cores.
__device__ __forceinline__ float dense_logistic(float v, float x) { return __fdividef(v, 1.f + __expf(-x)); }
__device__ __forceinline__ float dense_silu(float v) { return dense_logistic(v, v); }
// v times the normal distribution function of v.  Its tail below -s is exp(-s^2 / 2) t q(t) with t = 1 / (1 + 0.35 s): the smooth factor of the exponential by a
// polynomial of least relative error (3.2e-8 for s up to 15, fitted to it in 64 bits), so that small results keep their relative accuracy, 12 + 4 s^2 half steps,
// where 1 + erf cancels (4e-3 of the value lost at -4, all of it at -6).  It is shorter than erf and erfc, too: 4096 x 512 x 4096 31.5 us, 34.4 and 54.4 by those.
__device__ __forceinline__ float dense_gelu(float v) {
    const float s = fabsf(v);
    float t;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(fmaf(0.35f, s, 1.f)));
    float q = -0.029163932f;
    q = fmaf(q, t, 0.14406084f);
    q = fmaf(q, t, -0.25590196f);
    q = fmaf(q, t, 0.15939303f);
    q = fmaf(q, t, -0.023263901f);
    q = fmaf(q, t, 0.10557483f);
    q = fmaf(q, t, 0.11981549f);
    q = fmaf(q, t, 0.13986434f);
    q = fmaf(q, t, 0.13962126f);
    const float below = q * t * __expf(-0.5f * s * s);
    return v * (v < 0.f ? below : 1.f - below);            // (-inf: NaN, as -inf times 0)
}
// (1 + tanh z) / 2 is the logistic function of 2 z
__device__ __forceinline__ float dense_gelu_tanh(float v) { return dense_logistic(v, 1.59576912160573071f * (v + 0.044715f * v * v * v)); }
// clamps that let NaN through (fminf and fmaxf would drop it)
__device__ __forceinline__ float dense_below(float v, float limit) { return v > limit ? limit : v; }
__device__ __forceinline__ float dense_within(float v, float limit) { return v > limit ? limit : v < -limit ? -limit : v; }

// What follows the sums of output column n of several rows (row(i), of which those are there that are less than `rows`; row(0) is): bias (b),
// activation and residual, or the gated pair.  Chosen by comparisons around all rows: a jump table in front of every value cost 400 clocks each.
template <int ROWS, typename F>
__device__ __forceinline__ void dense_each(F f) {
#pragma unroll
    for (int i = 0; i < ROWS; ++i) f(i);
}
template <int ROWS>
__device__ __forceinline__ void dense_act(float (&v)[ROWS], int act) {
    if (act == GLMFLASH_ACT_NONE) return;
    if (act == GLMFLASH_ACT_SILU) dense_each<ROWS>([&](int i) { v[i] = dense_silu(v[i]); });
    else if (act == GLMFLASH_ACT_GELU) dense_each<ROWS>([&](int i) { v[i] = dense_gelu(v[i]); });
    else if (act == GLMFLASH_ACT_GELU_TANH) dense_each<ROWS>([&](int i) { v[i] = dense_gelu_tanh(v[i]); });
    else dense_each<ROWS>([&](int i) { v[i] = v[i] < 0.f ? 0.f : v[i]; });                                 // (NaN stays)
}
template <int MATS, int ROWS, typename R>
__device__ __forceinline__ void dense_finish(const DenseArgs &a, R row, int rows, int n, float (&g)[ROWS], float (&u)[ROWS], const float (&b)[2]) {
    float res[ROWS];
    if (MATS == 1 && a.residual) {                       // (rows that are not there read the first once more: no branch between the loads)
        auto at = [&](int i) { return (int64_t)(row(i) < rows ? row(i) : row(0)) * a.rs + n; };
        if (a.residual_type == GLMFLASH_F32) dense_each<ROWS>([&](int i) { res[i] = static_cast<const float *>(a.residual)[at(i)]; });
        else if (a.residual_type == GLMFLASH_F16) dense_each<ROWS>([&](int i) { res[i] = __half2float(static_cast<const __half *>(a.residual)[at(i)]); });
        else dense_each<ROWS>([&](int i) { res[i] = __bfloat162float(static_cast<const __nv_bfloat16 *>(a.residual)[at(i)]); });
    }
    dense_each<ROWS>([&](int i) { g[i] += b[0]; });
    if (MATS == 2) {
        dense_each<ROWS>([&](int i) { u[i] += b[1]; });
        if (a.limit > 0.f) dense_each<ROWS>([&](int i) { g[i] = dense_below(g[i], a.limit); u[i] = dense_within(u[i], a.limit); });
    }
    dense_act(g, a.act);
    if (MATS == 2) dense_each<ROWS>([&](int i) { g[i] *= u[i]; });
    else if (a.residual) dense_each<ROWS>([&](int i) { g[i] += res[i]; });
    auto at = [&](int i) { return (int64_t)row(i) * a.os + n; };
    if (a.out_type == GLMFLASH_F32) dense_each<ROWS>([&](int i) { if (row(i) < rows) static_cast<float *>(a.out)[at(i)] = g[i]; });
    else if (a.out_type == GLMFLASH_F16) dense_each<ROWS>([&](int i) { if (row(i) < rows) static_cast<__half *>(a.out)[at(i)] = __float2half_rn(g[i]); });
    else dense_each<ROWS>([&](int i) { if (row(i) < rows) static_cast<__nv_bfloat16 *>(a.out)[at(i)] = __float2bfloat16_rn(g[i]); });
}
template <int MATS>
__device__ __forceinline__ void dense_biases(const DenseArgs &a, int n, float (&b)[2]) {
#pragma unroll
    for (int m = 0; m < 2; ++m) b[m] = m < MATS && a.bias[m] && n < a.N ? dense_load(a.bias[m], n, a.bias_type) : 0.f;
}

int dense_gemm(cudaStream_t s, const DenseArgs &a, bool pdl);
// Router product (bf16, fp32 output) and selection in one launch, where they fit a cluster
struct SelRule;
bool dense_route_fits(const DenseArgs &a);
int dense_route(cudaStream_t s, const DenseArgs &a, const float *bias, int topk, const SelRule &rule, int *picks, float *weights, bool pdl);

}  // namespace gf
