// ops_gemv.cu — layers of up to eight rows: a warp per output.
//
// A row or a few of x leave the weights as what has to be read, once; what counts
// below a few megabytes of them is the latency of one call. Each warp walks one
// row of w in 16-byte pieces (element by element when w or x is unaligned), with
// the rows of x beside it out of the L1 cache, and joins its 32 lanes' sums at
// the end. No descriptors, no barriers. On the GPU, us here / in tiles of the
// tensor cores: 1 x 512 -> 512 bf16 1.8 / 6.0, 8 rows 2.9 / 6.2, 8 x 1024 -> 4096 7.2
// / 8.4, 8 x 4096 -> 1024 f32 13 / 81. With twice the rows (a build for 16) bf16
// 9 x 512 -> 512 5.1 / 8.4 but 9 x 1024 -> 4096 14.3 / 10.4, f32 16.6 / 27.
#include "ops.cuh"

namespace msplat {
namespace ops {
namespace {

constexpr int kWarps = 4;
constexpr int kSpan = 512;  // steps of a warp that one sum takes (LONG)

template <typename T>
__device__ __forceinline__ void unpack8(const T* g, float (&v)[16 / sizeof(T)]) {
    const uint4 p = __ldg(reinterpret_cast<const uint4*>(g));
    const uint32_t w[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        if constexpr (sizeof(T) == 4) {
            v[q] = __uint_as_float(w[q]);
        } else {
            union { uint32_t u; T t[2]; } c;
            c.u = w[q];
            v[2 * q] = to_f32(c.t[0]);
            v[2 * q + 1] = to_f32(c.t[1]);
        }
    }
}

// LONG: the sums start afresh after kSpan steps of the warp, and the rounded-off bits
// of 32-bit sums of millions of products stay small. (A kernel of its own: the outer
// loop takes 8 x 4096 -> 1024 f32 from 13 to 17 us.)
template <typename T, typename TO, int MT, bool VEC, bool LONG>
__global__ void __launch_bounds__(kWarps * 32) k_gemv(const __grid_constant__ Product p) {
    constexpr int E = VEC ? 16 / sizeof(T) : 1;
    const int lane = threadIdx.x % 32;
    const int64_t n = blockIdx.x * (int64_t)kWarps + threadIdx.x / 32;
    if (n >= p.N) return;
    const int M = (int)p.M;
    const T* x = static_cast<const T*>(p.A);
    const T* w = static_cast<const T*>(p.B) + n * p.ldb;
    float acc[MT], total[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[m] = total[m] = 0.f;
    const int64_t whole = VEC ? p.R / E * E : p.R;
    int step = 0;
#pragma unroll 2
    for (int64_t k = lane * E; k < whole; k += 32 * E) {
        if (LONG && ++step == kSpan) {
            step = 0;
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                total[m] += acc[m];
                acc[m] = 0.f;
            }
        }
        float b[E];
        if constexpr (VEC)
            unpack8<T>(w + k, b);
        else
            b[0] = to_f32(w[k]);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            const T* row = x + min(m, M - 1) * p.lda + k;
            float a[E];
            if constexpr (VEC)
                unpack8<T>(row, a);
            else
                a[0] = to_f32(*row);
#pragma unroll
            for (int e = 0; e < E; ++e) acc[m] = fmaf(a[e], b[e], acc[m]);
        }
    }
    if (VEC && whole + lane < p.R) {
        const float b = to_f32(w[whole + lane]);
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[m] = fmaf(to_f32(x[min(m, M - 1) * p.lda + whole + lane]), b, acc[m]);
    }
    float mine = 0.f;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        float s = LONG ? total[m] + acc[m] : acc[m];
#pragma unroll
        for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
        mine = lane == m ? s : mine;
    }
    if (lane >= M) return;
    const float z = mine + (p.bias ? to_f32(static_cast<const T*>(p.bias)[n]) : 0.f);
    if (p.preact) static_cast<TO*>(p.preact)[lane * p.ldz + n] = from_f32<TO>(z);
    float y = activate<TO>(both(z), p.act).x;
    if (p.residual) y += to_f32(static_cast<const TO*>(p.residual)[lane * p.ldr + n]);
    static_cast<TO*>(p.out)[lane * p.ldo + n] = from_f32<TO>(y);
}

template <typename T, typename TO, int MT>
void run(const Product& p, cudaStream_t s) {
    constexpr int E = 16 / sizeof(T);
    const bool vec = (reinterpret_cast<uintptr_t>(p.A) | reinterpret_cast<uintptr_t>(p.B)) % 16 == 0 &&
                     (p.M <= 1 || p.lda % E == 0) && (p.N <= 1 || p.ldb % E == 0);
    const unsigned grid = (unsigned)ceil_div(p.N, kWarps);
    note_launches(1);
    auto go = [&](auto kernel) { kernel<<<grid, kWarps * 32, 0, s>>>(p); };
    if (p.R > kSpan * 32 * (vec ? E : 1))
        vec ? go(k_gemv<T, TO, MT, true, true>) : go(k_gemv<T, TO, MT, false, true>);
    else
        vec ? go(k_gemv<T, TO, MT, true, false>) : go(k_gemv<T, TO, MT, false, false>);
    OPS_CK(cudaGetLastError());
}

template <typename T, typename TO>
void sized(const Product& p, cudaStream_t s) {
    if (p.M == 1) return run<T, TO, 1>(p, s);
    if (p.M == 2) return run<T, TO, 2>(p, s);
    if (p.M <= 4) return run<T, TO, 4>(p, s);
    run<T, TO, 8>(p, s);
}

template <typename T>
void typed(const Product& p, cudaStream_t s) {
    if (p.out_dtype == MSPLAT_DTYPE_F32)
        sized<T, float>(p, s);
    else
        sized<T, T>(p, s);
}

}  // namespace

bool can_product_gemv(const Product& p) {
    return p.epi == kEpiLinear && !p.a_mn && !p.b_mn && !p.targets && !p.alpha_dev && p.alpha == 1.f && p.M <= 8;
}

void launch_product_gemv(const Product& p, cudaStream_t s) {
    if (p.dtype == MSPLAT_DTYPE_F32)
        typed<float>(p, s);
    else if (p.dtype == MSPLAT_DTYPE_F16)
        typed<__half>(p, s);
    else
        typed<__nv_bfloat16>(p, s);
}

}  // namespace ops
}  // namespace msplat
