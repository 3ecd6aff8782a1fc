// ops_simt.cu — matrix products of any type, stride and alignment on the FP32
// pipes: 64 x 64 tiles staged in shared memory, 4 x 4 results per thread.
#include "ops_epilogue.cuh"

namespace msplat {
namespace ops {
namespace {

constexpr int kTileM = 64, kTileN = 64, kTileR = 16;

template <typename T>
__device__ __forceinline__ void load_tile(float (*s)[kTileM + 4], const T* g, int64_t ld, bool mn, int64_t i0,
                                          int64_t n_i, int64_t r0, int64_t r_end, const Product* masked) {
    for (int e = threadIdx.x; e < kTileM * kTileR; e += 256) {
        const int i = mn ? e % kTileM : e / kTileR, r = mn ? e / kTileM : e % kTileR;
        const int64_t gi = i0 + i, gr = r0 + r;
        float v = 0.f;
        if (gi < n_i && gr < r_end && (!masked || labelled(*masked, gr))) v = to_f32(mn ? g[gr * ld + gi] : g[gi * ld + gr]);
        s[r][i] = v;
    }
}

template <typename T, int EPI>
__global__ void __launch_bounds__(256) k_product_simt(const __grid_constant__ Product p, int tiles_n) {
    __shared__ float sa[kTileR][kTileM + 4], sb[kTileR][kTileN + 4];
    const int64_t i0 = (int64_t)(blockIdx.x / tiles_n) * kTileM, j0 = (int64_t)(blockIdx.x % tiles_n) * kTileN;
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    int64_t r_begin = 0, r_end = p.R;
    if (EPI == kEpiSlab) {
        r_begin = blockIdx.y * p.split_len;
        r_end = min(p.R, r_begin + p.split_len);
    }
    float acc[4][4] = {};
    for (int64_t r0 = r_begin; r0 < r_end; r0 += kTileR) {
        load_tile<T>(sa, static_cast<const T*>(p.A), p.lda, p.a_mn, i0, p.M, r0, r_end, nullptr);
        load_tile<T>(sb, static_cast<const T*>(p.B), p.ldb, p.b_mn, j0, p.N, r0, r_end,
                     p.label_reduces ? &p : nullptr);
        __syncthreads();
#pragma unroll
        for (int r = 0; r < kTileR; ++r) {
            float a[4], b[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                a[q] = sa[r][ty * 4 + q];
                b[q] = sb[r][tx * 4 + q];
            }
#pragma unroll
            for (int y = 0; y < 4; ++y)
#pragma unroll
                for (int x = 0; x < 4; ++x) acc[y][x] = fmaf(a[y], b[x], acc[y][x]);
        }
        __syncthreads();
    }
    if (EPI == kEpiLinear) {
        const float alpha = p.alpha * (p.alpha_dev ? *p.alpha_dev : 1.f);
#pragma unroll
        for (int y = 0; y < 4; ++y) {
            const int64_t i = i0 + ty * 4 + y;
            if (i >= p.M) continue;
            const bool zero = p.targets && !p.label_reduces && !labelled(p, i);
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const int64_t j = j0 + tx * 4 + x;
                if (j >= p.N) continue;
                if (p.out_dtype == MSPLAT_DTYPE_F32)
                    epi_linear<T, float>(p, alpha, zero, i, j, acc[y][x]);
                else
                    epi_linear<T, T>(p, alpha, zero, i, j, acc[y][x]);
            }
        }
    } else if (EPI == kEpiSlab) {
        float* slab = p.slab + (int64_t)blockIdx.y * p.M * p.N;
#pragma unroll
        for (int y = 0; y < 4; ++y)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const int64_t i = i0 + ty * 4 + y, j = j0 + tx * 4 + x;
                if (i < p.M && j < p.N) {
                    float* o = slab + i * p.N + j;
                    *o = p.accumulate ? *o + acc[y][x] : acc[y][x];
                }
            }
    } else {
        const float to2 = p.logit_scale * kLog2e;
#pragma unroll
        for (int y = 0; y < 4; ++y) {
            const int64_t i = i0 + ty * 4 + y;
            const bool in = i < p.M;
            const int32_t t = in ? __ldg(p.targets + i) : -1;
            if (EPI == kEpiStats) {
                float top = -INFINITY, sum = 0.f;
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const int64_t j = j0 + tx * 4 + x;
                    acc[y][x] = __fmul_rn(acc[y][x], to2);
                    if (j >= p.N) continue;
                    top = fmaxf(top, acc[y][x]);
                    if (p.col0 + j == t) p.label_logit[i] = acc[y][x];
                }
                for (int o = 8; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
                const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
                for (int x = 0; x < 4; ++x)
                    if (j0 + tx * 4 + x < p.N) sum += exp2f(acc[y][x] - ref);
                for (int o = 8; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
                if (in && tx == 0)
                    p.stats[(p.stats_block0 + blockIdx.x % tiles_n) * p.stats_ld + i] = make_float2(top, sum);
            } else if (in) {
                const bool zero = !labelled(p, i);
                const float lse = p.lse[i];
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const int64_t j = j0 + tx * 4 + x;
                    if (j >= p.N) continue;
                    const float g = zero ? 0.f : epi_grad(__fmul_rn(acc[y][x], to2), lse, p.col0 + j == t, p.g_scale);
                    static_cast<T*>(p.out)[i * p.ldo + j] = from_f32<T>(g);
                }
            }
        }
    }
}

template <typename T>
void typed(const Product& p, cudaStream_t s) {
    const int64_t tm = ceil_div(p.M, kTileM), tn = ceil_div(p.N, kTileN);
    if (tm * tn > 0x7fffffff) throw Error(MSPLAT_ERR_CAPACITY, "too many tiles");
    const dim3 grid((unsigned)(tm * tn), p.epi == kEpiSlab ? p.splits : 1);
    note_launches(1);
    switch (p.epi) {
        case kEpiLinear: k_product_simt<T, kEpiLinear><<<grid, 256, 0, s>>>(p, (int)tn); break;
        case kEpiSlab: k_product_simt<T, kEpiSlab><<<grid, 256, 0, s>>>(p, (int)tn); break;
        case kEpiStats: k_product_simt<T, kEpiStats><<<grid, 256, 0, s>>>(p, (int)tn); break;
        default: k_product_simt<T, kEpiGrad><<<grid, 256, 0, s>>>(p, (int)tn); break;
    }
    OPS_CK(cudaGetLastError());
}

}  // namespace

void launch_product_simt(const Product& p, cudaStream_t s) {
    if (p.dtype == MSPLAT_DTYPE_F32)
        typed<float>(p, s);
    else if (p.dtype == MSPLAT_DTYPE_F16)
        typed<__half>(p, s);
    else
        typed<__nv_bfloat16>(p, s);
}

int64_t stats_blocks(const Product& p) {
    if (!can_product_tc16(p)) return ceil_div(p.N, kTileN);
    return 2 * ceil_div(p.N, p.N > 128 ? 256 : p.N > 64 ? 128 : 64);  // halves of a tile
}
void launch_product(const Product& p, cudaStream_t s) {
    if (can_product_tc16(p)) return launch_product_tc16(p, s);
    launch_product_simt(p, s);
}

}  // namespace ops
}  // namespace msplat
