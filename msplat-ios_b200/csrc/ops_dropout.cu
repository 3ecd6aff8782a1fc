// ops_dropout.cu — dropout whose mask is a function of (seed, offset, element).
//
// Philox4x32-10 (Salmon, Moraes, Dror, Shaw: Parallel random numbers: as easy
// as 1, 2, 3, SC 2011): ten rounds of two 32 x 32 -> 64 bit products and
// exclusive ors give 128 bits from a counter and a key. One block of 128 bits
// serves eight elements with 16 bits each, which halves the integer work per
// element against 32-bit draws and makes p act in steps of 2^-16.
//
// Bound: reading x (and the residual) and writing y. Nothing else is stored;
// the backward pass draws the same bits again. 1M x 64 bf16 with a residual takes
// 65 us, 5.9 TB/s.
#include "ops.cuh"

namespace msplat {
namespace ops {
namespace {

__device__ __forceinline__ uint4 philox4x32_10(uint4 c, uint2 k) {
#pragma unroll
    for (int i = 0; i < 10; ++i) {
        const uint64_t a = (uint64_t)c.x * 0xD2511F53u, b = (uint64_t)c.z * 0xCD9E8D57u;
        c = make_uint4((uint32_t)(b >> 32) ^ c.y ^ k.x, (uint32_t)b, (uint32_t)(a >> 32) ^ c.w ^ k.y, (uint32_t)a);
        k.x += 0x9E3779B9u;
        k.y += 0xBB67AE85u;
    }
    return c;
}

template <typename T>
struct DropArgs {
    int64_t rows, cols, ldx, ldr, ldy;
    const T* x;
    const T* residual;
    T* y;
    uint32_t below;
    float scale;
    uint64_t seed, offset;
    const uint64_t* offset_dev;
};

// One thread per block of eight elements of the row-major order. FLAT: the
// matrices are contiguous and 16-byte aligned, so a block is one or two
// 16-byte accesses; otherwise each element finds its row and column (with a
// 32-bit division per block where the elements are fewer than 2^32).
template <typename T, bool FLAT>
__global__ void __launch_bounds__(256) k_dropout(DropArgs<T> a) {
    const int64_t n = a.rows * a.cols, blocks = (n + 7) / 8;
    const uint64_t c = a.offset + (a.offset_dev ? *a.offset_dev : 0);
    const uint2 key = make_uint2((uint32_t)a.seed, (uint32_t)(a.seed >> 32));
    for (int64_t b = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; b < blocks; b += (int64_t)gridDim.x * blockDim.x) {
        const uint4 r = philox4x32_10(make_uint4((uint32_t)b, (uint32_t)((uint64_t)b >> 32), (uint32_t)c,
                                                 (uint32_t)(c >> 32)), key);
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
        const int64_t e0 = 8 * b;
        if (FLAT && e0 + 8 <= n) {
            union V { uint4 q[sizeof(T) / 2]; T t[8]; } vx, vr;
#pragma unroll
            for (int q = 0; q < (int)sizeof(T) / 2; ++q)
                vx.q[q] = reinterpret_cast<const uint4*>(a.x + e0)[q];
            if (a.residual) {
#pragma unroll
                for (int q = 0; q < (int)sizeof(T) / 2; ++q)
                    vr.q[q] = reinterpret_cast<const uint4*>(a.residual + e0)[q];
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t draw = (i & 1) ? w[i / 2] >> 16 : w[i / 2] & 0xFFFFu;
                float v = draw >= a.below ? to_f32(vx.t[i]) * a.scale : 0.f;
                if (a.residual) v += to_f32(vr.t[i]);
                vx.t[i] = from_f32<T>(v);
            }
#pragma unroll
            for (int q = 0; q < (int)sizeof(T) / 2; ++q) reinterpret_cast<uint4*>(a.y + e0)[q] = vx.q[q];
        } else if (FLAT) {
            for (int i = 0; i < 8 && e0 + i < n; ++i) {  // the last block
                const uint32_t word = i < 2 ? r.x : i < 4 ? r.y : i < 6 ? r.z : r.w;
                const uint32_t draw = (i & 1) ? word >> 16 : word & 0xFFFFu;
                float v = draw >= a.below ? to_f32(a.x[e0 + i]) * a.scale : 0.f;
                if (a.residual) v += to_f32(a.residual[e0 + i]);
                a.y[e0 + i] = from_f32<T>(v);
            }
        } else {
            int64_t row = n >> 32 ? e0 / a.cols : (int64_t)((uint32_t)e0 / (uint32_t)a.cols), col = e0 - row * a.cols;
            const T* x = a.x + row * a.ldx + col;
            const T* res = a.residual + (a.residual ? row * a.ldr + col : 0);
            T* y = a.y + row * a.ldy + col;
            T vx[8], vr[8], *to[8];
            // every load before the first store, so that they overlap
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                to[i] = y;
                if (e0 + i < n) {
                    vx[i] = *x;
                    if (a.residual) vr[i] = *res;
                }
                ++x;
                ++y;
                ++res;
                if (++col == a.cols) {
                    col = 0;
                    x += a.ldx - a.cols;
                    y += a.ldy - a.cols;
                    res += a.ldr - a.cols;
                }
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (e0 + i >= n) break;
                const uint32_t draw = (i & 1) ? w[i / 2] >> 16 : w[i / 2] & 0xFFFFu;
                float v = draw >= a.below ? to_f32(vx[i]) * a.scale : 0.f;
                if (a.residual) v += to_f32(vr[i]);
                *to[i] = from_f32<T>(v);
            }
        }
    }
}

template <typename T>
void run(DropArgs<T> a, cudaStream_t s) {
    const int64_t n = a.rows * a.cols;
    const uintptr_t at = reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.y) |
                         reinterpret_cast<uintptr_t>(a.residual);
    const bool one_row = a.rows == 1;
    const bool flat = (at & 15) == 0 && (one_row || (a.ldx == a.cols && a.ldy == a.cols &&
                                                     (!a.residual || a.ldr == a.cols)));
    const int64_t ctas = ceil_div(ceil_div(n, 8), 256);
    const unsigned grid = (unsigned)(ctas < kSMs * 16 ? ctas : kSMs * 16);
    note_launches(1);
    if (flat)
        k_dropout<T, true><<<grid, 256, 0, s>>>(a);
    else
        k_dropout<T, false><<<grid, 256, 0, s>>>(a);
    OPS_CK(cudaGetLastError());
}

template <typename T>
void typed(int64_t rows, int64_t cols, const void* x, int64_t ldx, const void* residual, int64_t ldr, void* y,
           int64_t ldy, uint32_t below, float scale, uint64_t seed, uint64_t offset, const uint64_t* offset_dev,
           cudaStream_t s) {
    DropArgs<T> a{rows, cols, ldx, ldr, ldy, static_cast<const T*>(x), static_cast<const T*>(residual),
                  static_cast<T*>(y), below, scale, seed, offset, offset_dev};
    run(a, s);
}

}  // namespace

void launch_dropout(int64_t rows, int64_t cols, const void* x, int64_t ldx, const void* residual, int64_t ldr, void* y,
                    int64_t ldy, uint32_t below, float scale, uint64_t seed, uint64_t offset,
                    const uint64_t* offset_dev, int dtype, cudaStream_t s) {
    if (dtype == MSPLAT_DTYPE_F32)
        typed<float>(rows, cols, x, ldx, residual, ldr, y, ldy, below, scale, seed, offset, offset_dev, s);
    else if (dtype == MSPLAT_DTYPE_F16)
        typed<__half>(rows, cols, x, ldx, residual, ldr, y, ldy, below, scale, seed, offset, offset_dev, s);
    else
        typed<__nv_bfloat16>(rows, cols, x, ldx, residual, ldr, y, ldy, below, scale, seed, offset, offset_dev, s);
}

}  // namespace ops
}  // namespace msplat
