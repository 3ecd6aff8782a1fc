// ops_epilogue.cuh — the per-element ends of a matrix product (ops.cuh), shared
// by the kernels that compute one.
#pragma once
#include "ops.cuh"

namespace msplat {
namespace ops {

__device__ __forceinline__ bool labelled(const Product& p, int64_t row) {
    const int32_t t = __ldg(p.targets + row);
    return t >= 0 && t < p.labels;
}

// bias, activation, residual (kEpiLinear) of one element
template <typename TI, typename TO>
__device__ __forceinline__ void epi_linear(const Product& p, float alpha, bool zero, int64_t i, int64_t j, float acc) {
    float z = acc * alpha;
    if (p.bias) z += to_f32(static_cast<const TI*>(p.bias)[j]);
    if (zero) z = 0.f;
    if (p.preact) static_cast<TO*>(p.preact)[i * p.ldz + j] = from_f32<TO>(z);
    float y = activate(z, p.act);
    if (p.residual) y += to_f32(static_cast<const TO*>(p.residual)[i * p.ldr + j]);
    static_cast<TO*>(p.out)[i * p.ldo + j] = from_f32<TO>(y);
}

// softmax minus one-hot, scaled, of a logit in log2 units. The logit must be
// the same bits as the statistics saw (a product with rounding, not part of a
// fused multiply-add): at large logits one bit of it is a large difference.
__device__ __forceinline__ float epi_grad(float l2, float lse, bool is_label, float g_scale) {
    return (exp2f(l2 - lse) - (is_label ? 1.f : 0.f)) * g_scale;
}

}  // namespace ops
}  // namespace msplat
