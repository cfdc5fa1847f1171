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
__device__ __forceinline__ void dense_store(void *p, int64_t i, int type, float v) {
    if (type == GLMFLASH_F32) static_cast<float *>(p)[i] = v;
    else if (type == GLMFLASH_F16) static_cast<__half *>(p)[i] = __float2half_rn(v);
    else static_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(v);
}
__device__ __forceinline__ float dense_gelu(float v) { return 0.5f * v * (1.f + erff(v * 0.70710678118654752f)); }
__device__ __forceinline__ float dense_gelu_tanh(float v) { return 0.5f * v * (1.f + tanhf(0.79788456080286536f * (v + 0.044715f * v * v * v))); }
__device__ __forceinline__ float dense_act(float v, int act) {
    switch (act) {
        case GLMFLASH_ACT_SILU: return silu(v);
        case GLMFLASH_ACT_GELU: return dense_gelu(v);
        case GLMFLASH_ACT_GELU_TANH: return dense_gelu_tanh(v);
        case GLMFLASH_ACT_RELU: return v < 0.f ? 0.f : v;                            // (NaN stays)
        default: return v;
    }
}
// clamps that let NaN through (fminf and fmaxf would drop it)
__device__ __forceinline__ float dense_below(float v, float limit) { return v > limit ? limit : v; }
__device__ __forceinline__ float dense_within(float v, float limit) { return v > limit ? limit : v < -limit ? -limit : v; }

// What follows the sums of output column n of row r.
template <int MATS>
__device__ __forceinline__ void dense_finish(const DenseArgs &a, int r, int n, float g, float u) {
    if (a.bias[0]) g += dense_load(a.bias[0], n, a.bias_type);
    if (MATS == 2) {
        if (a.bias[1]) u += dense_load(a.bias[1], n, a.bias_type);
        if (a.limit > 0.f) { g = dense_below(g, a.limit); u = dense_within(u, a.limit); }
        g = dense_act(g, a.act) * u;
    } else {
        g = dense_act(g, a.act);
        if (a.residual) g += dense_load(a.residual, r * a.rs + n, a.residual_type);
    }
    dense_store(a.out, r * a.os + n, a.out_type, g);
}

int dense_wide(cudaStream_t s, const DenseArgs &a, bool pdl);

}  // namespace gf
