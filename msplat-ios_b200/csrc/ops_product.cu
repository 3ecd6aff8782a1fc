// ops_product.cu — which kernel a matrix product takes.
#include "ops.cuh"

namespace msplat {
namespace ops {

int64_t stats_blocks(const Product& p) { return can_product_tc16(p) ? stats_blocks_tc16(p) : stats_blocks_tcv(p); }

void launch_product(const Product& p, cudaStream_t s) {
    if (can_product_gemv(p)) return launch_product_gemv(p, s);
    if (can_product_few(p)) return launch_product_few(p, s);
    if (can_product_tc16(p)) return launch_product_tc16(p, s);
    launch_product_tcv(p, s);
}

}  // namespace ops
}  // namespace msplat
