// ops.cuh — what the kernels behind include/msplat_ops.h share: element types,
// the description of one matrix product with its epilogue, and the launchers.
#pragma once
#include <algorithm>
#include <atomic>
#include <cstdint>
#include <stdexcept>
#include <string>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "msplat_backend.h"
#include "msplat_ops.h"
#include "kernels.cuh"

namespace msplat {
namespace ops {

struct Error : std::runtime_error {
    int code;
    Error(int c, const std::string& m) : std::runtime_error(m), code(c) {}
};

#define OPS_CK(call)                                                                                \
    do {                                                                                            \
        cudaError_t e_ = (call);                                                                    \
        if (e_ != cudaSuccess)                                                                      \
            throw ::msplat::ops::Error(MSPLAT_ERR_CUDA, std::string(#call) + ": " + cudaGetErrorString(e_)); \
    } while (0)

__host__ __device__ inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
__host__ __device__ inline int64_t round_up(int64_t a, int64_t b) { return ceil_div(a, b) * b; }
inline int dtype_size(int dtype) { return dtype == MSPLAT_DTYPE_F32 ? 4 : 2; }
constexpr int kSMs = 148;

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// 2^x with the special function unit alone (2 units in the last place; results
// below 2^-126 are 0).
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// 1 / x with the special function unit alone (1 unit in the last place).
__device__ __forceinline__ float recip_fast(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The Gaussian distribution function through the error function's
// approximation 7.1.26 of Abramowitz and Stegun, Handbook of Mathematical
// Functions: erfc(x) = t (a1 + t (a2 + ...)) exp(-x^2), t = 1 / (1 + p x), off by
// at most 1.5e-7; a reciprocal and an exponential in place of erff's longer
// polynomials. *density: exp(-z^2 / 2).
__device__ __forceinline__ float normal_cdf(float z, float* density) {
    const float x = fabsf(z) * 0.70710678118654752f;
    const float t = recip_fast(fmaf(0.3275911f, x, 1.f));
    const float e = exp2_fast(-kLog2e * x * x);
    float q = fmaf(1.061405429f, t, -1.453152027f);
    q = fmaf(q, t, 1.421413741f);
    q = fmaf(q, t, -0.284496736f);
    q = fmaf(q, t, 0.254829592f);
    q = 0.5f * q * t * e;  // half of erfc(x)
    *density = e;
    return z < 0.f ? q : 1.f - q;
}
__device__ __forceinline__ float logistic(float z) { return recip_fast(1.f + exp2_fast(-kLog2e * z)); }

__device__ __forceinline__ float act_relu(float z) { return z < 0.f ? 0.f : z; }
__device__ __forceinline__ float act_gelu(float z) {
    float e;
    return z * normal_cdf(z, &e);
}
__device__ __forceinline__ float act_silu(float z) { return z * logistic(z); }
__device__ __forceinline__ float act_sigmoid(float z) { return logistic(z); }
// act'(z)
template <int ACT>
__device__ __forceinline__ float act_slope(float z) {
    if (ACT == MSPLAT_ACT_RELU) return z > 0.f ? 1.f : 0.f;
    if (ACT == MSPLAT_ACT_GELU) {
        float e;
        const float c = normal_cdf(z, &e);
        return fmaf(z * 0.3989422804014327f, e, c);
    }
    if (ACT == MSPLAT_ACT_SILU) {
        const float q = logistic(z);
        return q * fmaf(z, 1.f - q, 1.f);
    }
    if (ACT == MSPLAT_ACT_SIGMOID) {
        const float q = logistic(z);
        return q * (1.f - q);
    }
    return 1.f;
}

// Lets a kernel use `bytes` of dynamic shared memory, once per kernel and device.
template <auto KERNEL>
void allow_shared(int bytes) {
    static std::atomic<uint64_t> done{0};
    int dev = 0;
    OPS_CK(cudaGetDevice(&dev));
    const uint64_t bit = 1ull << (dev & 63);
    if (done.load(std::memory_order_acquire) & bit) return;
    OPS_CK(cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    done.fetch_or(bit, std::memory_order_release);
}

// What a matrix product does with its result.
enum EpiKind {
    kEpiLinear = 0,  // bias, activation, residual; element type T or float
    kEpiSlab = 1,    // float partial sums: slab[split][row][col] = or += result, slab_ld(N) floats per row
    kEpiStats = 2,   // per row and column block: max and sum of exp of the logits; the label's logit
    kEpiGrad = 3,    // (softmax - one-hot), times g_scale, in T
};

__host__ __device__ inline int64_t slab_ld(int64_t n) { return round_up(n, 4); }

// C[i, j] = sum_r A(i, r) B(j, r), i < M, j < N, r < R.
// A(i, r) = a_mn ? A[r * lda + i] : A[i * lda + r], B(j, r) likewise.
struct Product {
    int64_t M, N, R;
    const void* A;
    const void* B;
    int64_t lda, ldb;
    bool a_mn, b_mn;
    int dtype;
    int epi;
    // kEpiLinear
    const void* bias;
    int act;
    const void* residual;
    int64_t ldr;
    void* preact;
    int64_t ldz;
    void* out;          // kEpiLinear, kEpiGrad
    int64_t ldo;
    int out_dtype;
    float alpha;              // times the product (kEpiLinear)
    const float* alpha_dev;   // times this, when not null
    // kEpiSlab: R is cut into `splits` pieces of `split_len`
    float* slab;
    int splits;
    int64_t split_len;
    int accumulate;
    // labels (kEpiStats, kEpiGrad; kEpiLinear: rows without one become zeros)
    const int32_t* targets;
    int64_t labels;     // number of labels
    int64_t col0;       // label of column 0 of this piece
    float logit_scale;
    float g_scale;
    float2* stats;            // [column blocks][stats_ld]
    int64_t stats_ld;
    float* label_logit;       // [M]
    const float* lse;         // [M], in units of log2
};

// Column blocks that a kEpiStats product leaves statistics of; at most
// stats_blocks_most(N) for any type and alignment.
int64_t stats_blocks(const Product& p);
inline int64_t stats_blocks_most(int64_t n) { return 2 * ceil_div(n, 64); }

void launch_product(const Product& p, cudaStream_t s);
// 16-bit matrices that TMA can address (ops_tc16.cu); everything else (ops_tcv.cu).
bool can_product_tc16(const Product& p);
int64_t stats_blocks_tc16(const Product& p);
void launch_product_tc16(const Product& p, cudaStream_t s);
bool gave_up_tc16(cudaStream_t s);
void launch_product_tcv(const Product& p, cudaStream_t s);
// layers of a few rows (ops_gemv.cu)
bool can_product_gemv(const Product& p);
void launch_product_gemv(const Product& p, cudaStream_t s);
// layers with few outputs and many rows (ops_few.cu)
bool can_product_few(const Product& p);
void launch_product_few(const Product& p, cudaStream_t s);
int64_t stats_blocks_tcv(const Product& p);
bool gave_up_tcv(cudaStream_t s);

// Many rows against a small matrix in one pass (ops_rows.cu): v x d w, at most
// 128 x 64. slab: [rows_blocks(m)][v][slab_ld(d)] partial sums of dw, sums:
// [rows_blocks(m)][v] of g; each may be null, and dx.
bool fits_rows(int64_t m, int64_t v, int64_t d);
int rows_blocks(int64_t m);
bool gave_up_rows(cudaStream_t s);
void launch_rows_labels(int64_t m, int64_t v, int64_t d, const void* x, int64_t ldx, const void* w, int64_t ldw,
                        const int32_t* targets, float logit_scale, float g_scale, const float* alpha, float* row_loss,
                        double* partial, void* dx, int64_t lddx, float* slab, int dtype, cudaStream_t s);
void launch_rows_layer(int64_t m, int64_t n, int64_t k, const void* x, int64_t ldx, const void* w, int64_t ldw,
                       const void* z, int64_t ldz, int act, const void* dy, int64_t lddy, void* dx, int64_t lddx,
                       float* slab, float* sums, int dtype, cudaStream_t s);
// partial[block] = (0, labelled rows of the block's share)
void launch_count_labels(int64_t m, const int32_t* targets, int64_t labels, double* partial, int blocks,
                         cudaStream_t s);

// dz = dy act'(z) (dz may be null) and the column sums of dz in pieces of
// rows: partial[piece][n]. Returns the number of pieces.
int dz_pieces(int64_t m, int64_t n);
void launch_dz(int64_t m, int64_t n, const void* z, int64_t ldz, int act, const void* dy, int64_t lddy, void* dz,
               int64_t lddz, float* partial, int dtype, cudaStream_t s);
// out[i, j] = alpha * sum_p slab[p][i][j]; slab rows of ld floats
void launch_slab_sum(int64_t rows, int64_t cols, const float* slab, int64_t ld, int pieces, void* out, int64_t ldo, float alpha,
                     const float* alpha_dev, const int32_t* targets, int64_t labels, int dtype, cudaStream_t s);
// Joins the column blocks' statistics of m rows into lse (log2 units) and
// row_loss; partial[block] = (sum of the labelled rows' losses, their number).
struct JoinArgs {
    int64_t m, blocks;
    const float2* stats;
    int64_t stats_ld;
    const float* label_logit;
    const int32_t* targets;
    int64_t labels;
    float* lse;
    float* row_loss;
    double* partial;      // [join_blocks(m)][2]
};
int join_blocks(int64_t m);
// The rows of x with a label, zeros in place of the others: what the products
// read, so that an unlabelled row's NaN or infinity reaches nothing (in dw even
// a zero gradient times it would). Without targets, all of x (into rows that
// TMA can address).
void launch_labelled_rows(int64_t m, int64_t d, const void* x, int64_t ldx, const int32_t* targets, int64_t labels,
                          void* out, int64_t ldo, int dtype, cudaStream_t s);
void launch_join(const JoinArgs& a, cudaStream_t s);
// loss = weight * mean, *alpha = factor / number of labelled rows (both 0
// without any), from all the partial sums.
void launch_loss_total(const double* partial, int blocks, float weight, float factor, float* loss, float* alpha,
                       cudaStream_t s);

void launch_dropout(int64_t rows, int64_t cols, const void* x, int64_t ldx, const void* residual, int64_t ldr, void* y,
                    int64_t ldy, uint32_t below, float scale, uint64_t seed, uint64_t offset,
                    const uint64_t* offset_dev, int dtype, cudaStream_t s);

}  // namespace ops
}  // namespace msplat
