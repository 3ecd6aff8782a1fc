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

// softmax minus one-hot, scaled, of a logit in log2 units. The logit must be
// the same bits as the statistics saw (a product with rounding, not part of a
// fused multiply-add): at large logits one bit of it is a large difference.
__device__ __forceinline__ float epi_grad(float l2, float lse, bool is_label, float g_scale) {
    return (exp2f(l2 - lse) - (is_label ? 1.f : 0.f)) * g_scale;
}

}  // namespace ops
}  // namespace msplat
