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

}  // namespace ops
}  // namespace msplat
