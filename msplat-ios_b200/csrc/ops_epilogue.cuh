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

// 2^x with the special function unit alone (2 units in the last place; results
// below 2^-126 are 0). The logits of the statistics and of the gradient must be
// the same bits when they get here (a product with rounding, not part of a
// fused multiply-add): at large logits one bit of them is a large difference.
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

}  // namespace ops
}  // namespace msplat
