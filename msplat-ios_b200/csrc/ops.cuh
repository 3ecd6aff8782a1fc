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

constexpr float kLog2e = 1.4426950408889634f, kLog2eRest = 1.925963e-8f;  // log2(e) is the sum
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

// The activations, two values at a time, for results of 32 (FULL) or 16 bits.
//
// e^-z and e^(-z^2/2) are powers of 2 whose exponent is rounded: 2^-24 of an
// exponent of 100 is 4e-6 of the power, far below half a step of 16 bits (2^-11) but
// 70 steps of 32. FULL adds the rounded-off rest: 2^(b - r) = 2^b (1 - r ln 2).
//
// The Gaussian distribution function: with x = |z| / sqrt(2), t = 1 / (1 + p x) maps
// 0 .. infinity to 1 .. 0, and erfc(x) e^(x^2) / t is a smooth function of t; its
// minimax polynomials in the relative error (Remez exchange for x up to 9.4; e^(-x^2)
// is below 2^-126 from 9.35 on), here of half of it, keep the bits of the negative
// tail: off by 7e-9 (p = 0.4, ten coefficients, FULL; 4e-7 with t's rounding) or
// 1.2e-6 (p = 0.5, seven).
//
// FULL is written with the instructions for pairs, which halve its issue slots: one
// value at a time took 1M x 32 -> 64 with GELU from 171 to 212 us, pairs to 179.
constexpr float kHalfLog2e = 0.72134752f, kHalfLog2eRest = 9.62981e-9f;  // log2(e) / 2 is the sum

__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
__device__ __forceinline__ float2 exp2_rest(float2 b, float2 r) {
    const float2 e = make_float2(exp2_fast(b.x), exp2_fast(b.y));
    return __ffma2_rn(__fmul2_rn(e, r), both(-kLn2), e);
}
// The smaller and the larger of two, NaN for NaN.
__device__ __forceinline__ float least(float a, float b) {
    float x;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(x) : "f"(a), "f"(b));
    return x;
}
__device__ __forceinline__ float most(float a, float b) {
    float x;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(x) : "f"(a), "f"(b));
    return x;
}
__device__ __forceinline__ float size14(float z) { return least(fabsf(z), 14.f); }
// x = size14(z): the distribution function of -x as tail * density
__device__ __forceinline__ float2 normal_tail(float2 x, float2* density) {
    const float2 u = __ffma2_rn(x, both(0.4f * 0.70710678118654752f), both(1.f));
    const float2 t = make_float2(recip_fast(u.x), recip_fast(u.y));
    float2 q = __ffma2_rn(t, both(-0.015400324f), both(0.102300011f));
    q = __ffma2_rn(q, t, both(-0.257197171f));
    q = __ffma2_rn(q, t, both(0.28417924f));
    q = __ffma2_rn(q, t, both(-0.150951371f));
    q = __ffma2_rn(q, t, both(0.140780494f));
    q = __ffma2_rn(q, t, both(0.0631824881f));
    q = __ffma2_rn(q, t, both(0.107818633f));
    q = __ffma2_rn(q, t, both(0.112432256f));
    q = __ffma2_rn(q, t, both(0.11285574f));
    const float2 a = __fmul2_rn(x, x), b = __fmul2_rn(a, both(-kHalfLog2e));
    const float2 rest = __ffma2_rn(x, x, __fmul2_rn(a, both(-1.f)));  // of a
    float2 r = __ffma2_rn(a, both(kHalfLog2e), b);
    r = __ffma2_rn(a, both(kHalfLog2eRest), r);
    r = __ffma2_rn(rest, both(kHalfLog2e), r);
    *density = exp2_rest(b, r);
    return __fmul2_rn(q, t);
}
// the same with what 16 bits need, one value
__device__ __forceinline__ float normal_tail16(float x, float* density) {
    const float t = recip_fast(fmaf(0.5f * 0.70710678118654752f, x, 1.f));
    float q = fmaf(0.0446559116f, t, -0.180322498f);
    q = fmaf(q, t, 0.197353497f);
    q = fmaf(q, t, 0.0169986133f);
    q = fmaf(q, t, 0.141485006f);
    q = fmaf(q, t, 0.138653114f);
    q = fmaf(q, t, 0.141175792f);
    *density = exp2_fast(-kHalfLog2e * x * x);
    return q * t;
}

// 1 / (1 + e^-z), 0 from z = -88 downwards. *rest: what it lacks to 1 (where it
// is not 0), which subtracting it from 1 would round off for large z.
template <bool FULL>
__device__ __forceinline__ float2 logistic(float2 z, float2* rest) {
    float2 e;
    if (FULL) {
        const float2 x = make_float2(least(most(z.x, -88.f), 88.f), least(most(z.y, -88.f), 88.f));
        const float2 b = __fmul2_rn(x, both(-kLog2e));
        e = exp2_rest(b, __ffma2_rn(x, both(kLog2eRest), __ffma2_rn(x, both(kLog2e), b)));
    } else {
        e = make_float2(least(exp2_fast(-kLog2e * z.x), 3e38f), least(exp2_fast(-kLog2e * z.y), 3e38f));
    }
    const float2 q = make_float2(recip_fast(1.f + e.x), recip_fast(1.f + e.y));
    *rest = __fmul2_rn(q, e);
    return q;
}
__device__ __forceinline__ float act_relu(float z) { return z < 0.f ? 0.f : z; }
template <bool FULL>
__device__ __forceinline__ float2 act_gelu(float2 z) {
    // z Phi(z) = max(z, 0) - |z| Phi(-|z|)
    const float2 x = make_float2(size14(z.x), size14(z.y)), top = make_float2(fmaxf(z.x, 0.f), fmaxf(z.y, 0.f));
    float2 e;
    if (FULL) return __ffma2_rn(__fmul2_rn(__fmul2_rn(normal_tail(x, &e), x), e), both(-1.f), top);
    const float qx = normal_tail16(x.x, &e.x) * e.x, qy = normal_tail16(x.y, &e.y) * e.y;
    return make_float2(fmaf(-x.x, qx, top.x), fmaf(-x.y, qy, top.y));
}
template <bool FULL>
__device__ __forceinline__ float2 act_silu(float2 z) {
    float2 rest;
    return __fmul2_rn(z, logistic<FULL>(z, &rest));
}
template <bool FULL>
__device__ __forceinline__ float2 act_sigmoid(float2 z) {
    float2 rest;
    return logistic<FULL>(z, &rest);
}
// act(z) for a result of type TO
template <typename TO>
__device__ __forceinline__ float2 activate(float2 z, int act) {
    constexpr bool FULL = sizeof(TO) == 4;
    return act == MSPLAT_ACT_RELU      ? make_float2(act_relu(z.x), act_relu(z.y))
           : act == MSPLAT_ACT_GELU    ? act_gelu<FULL>(z)
           : act == MSPLAT_ACT_SILU    ? act_silu<FULL>(z)
           : act == MSPLAT_ACT_SIGMOID ? act_sigmoid<FULL>(z)
                                       : z;
}
// act'(z) for gradients of type T
template <int ACT, typename T>
__device__ __forceinline__ float2 act_slope(float2 z) {
    constexpr bool FULL = sizeof(T) == 4;
    if (ACT == MSPLAT_ACT_RELU) return make_float2(z.x > 0.f ? 1.f : 0.f, z.y > 0.f ? 1.f : 0.f);
    if (ACT == MSPLAT_ACT_GELU) {  // Phi + z phi is s = Phi(-|z|) - |z| phi(z) below 0 and 1 - s above
        constexpr float kPhi = 0.3989422804014327f;
        const float2 x = make_float2(size14(z.x), size14(z.y));
        float2 e, s;
        if (FULL) {
            s = normal_tail(x, &e);
            s = __fmul2_rn(__ffma2_rn(x, both(-kPhi), s), e);
        } else {
            const float qx = normal_tail16(x.x, &e.x), qy = normal_tail16(x.y, &e.y);
            s = make_float2(fmaf(x.x, -kPhi, qx) * e.x, fmaf(x.y, -kPhi, qy) * e.y);
        }
        return make_float2(z.x < 0.f ? s.x : 1.f - s.x, z.y < 0.f ? s.y : 1.f - s.y);
    }
    if (ACT == MSPLAT_ACT_SILU || ACT == MSPLAT_ACT_SIGMOID) {
        float2 rest;
        const float2 q = logistic<FULL>(z, &rest);
        return __fmul2_rn(q, ACT == MSPLAT_ACT_SILU ? __ffma2_rn(z, rest, both(1.f)) : rest);
    }
    return both(1.f);
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
    const float2* norm;       // [M]: largest logit in units of log2, 1 / sum of the exponentials relative to it
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
unsigned gave_up_tc16(cudaStream_t s);
void give_up_tc16(cudaStream_t s);
void launch_product_tcv(const Product& p, cudaStream_t s);
// layers of a few rows (ops_gemv.cu)
bool can_product_gemv(const Product& p);
void launch_product_gemv(const Product& p, cudaStream_t s);
// layers with few outputs and many rows (ops_few.cu)
bool can_product_few(const Product& p);
void launch_product_few(const Product& p, cudaStream_t s);
int64_t stats_blocks_tcv(const Product& p);
unsigned gave_up_tcv(cudaStream_t s);
void give_up_tcv(cudaStream_t s);

// Many rows against a small matrix in one pass (ops_rows.cu): v x d w, at most
// 128 x 64. slab: [rows_blocks(m)][v][slab_ld(d)] partial sums of dw, sums:
// [rows_blocks(m)][v] of g; each may be null, and dx.
bool fits_rows(int64_t m, int64_t v, int64_t d);
int rows_blocks(int64_t m);
unsigned gave_up_rows(cudaStream_t s);
void give_up_rows(cudaStream_t s);
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
// Joins the column blocks' statistics of m rows into norm (as in Product; not one
// logarithm of the sum, whose rounding would be a common factor of a row's
// probabilities: 4e-5 at logits of 1000) and row_loss; partial[block] = (sum of the
// labelled rows' losses, their number).
struct JoinArgs {
    int64_t m, blocks;
    const float2* stats;
    int64_t stats_ld;
    const float* label_logit;
    const int32_t* targets;
    int64_t labels;
    float2* norm;
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
