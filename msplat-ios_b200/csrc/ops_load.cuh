// ops_load.cuh — operands of the tensor cores that pass through registers: loads
// of any alignment, the split of 32-bit factors, the swizzled stores.
#pragma once
#include "ops_tc.cuh"

namespace msplat {
namespace ops {

// Parts of a factor: h + m + l of 32-bit ones. h and m of factors above 3.39e38
// are the largest bf16 number in place of an infinity, so that finite factors stay
// exact up to their type's largest and an infinite one is (largest, largest,
// infinity): of the six products the infinite ones, l h' and h l', have the
// product's sign, and the others stay finite beside them as long as m' is below 1,
// which it is for a second factor below 256. (Any second factor would take a branch
// per stage: 8% of the 1M-row layer of 32 inputs, 16% of 8192 x 512 -> 512.)
template <typename T>
constexpr int planes() { return sizeof(T) == 4 ? 3 : 1; }
// Two values rounded to bf16 in one word, no infinity for finite ones or infinities.
__device__ __forceinline__ uint32_t pack2_finite(float a, float b) {
    uint32_t w;
    asm("cvt.rn.satfinite.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(b), "f"(a));
    return w;
}

// Eight consecutive elements on their way to shared memory, as 32-bit words.
template <typename T>
struct Chunk {
    static constexpr int kWords = 8 * sizeof(T) / 4, kPieces = kWords / 4;
    uint32_t w[kWords];

    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int q = 0; q < kWords; ++q) w[q] = 0;
    }
    // Element by element: the first n.
    __device__ __forceinline__ void load_each(const T* g, int n) {
        zero();
#pragma unroll
        for (int q = 0; q < 8; ++q)
            if (q < n) {
                if constexpr (sizeof(T) == 4)
                    w[q] = __ldg(reinterpret_cast<const uint32_t*>(g) + q);
                else
                    w[q / 2] |= (uint32_t)__ldg(reinterpret_cast<const uint16_t*>(g) + q) << 16 * (q & 1);
            }
    }
    // From a 16-byte boundary.
    __device__ __forceinline__ void load_aligned(const T* g) {
#pragma unroll
        for (int q = 0; q < kWords / 4; ++q) {
            const uint4 v = __ldg(reinterpret_cast<const uint4*>(g) + q);
            w[4 * q] = v.x; w[4 * q + 1] = v.y; w[4 * q + 2] = v.z; w[4 * q + 3] = v.w;
        }
    }
    // From any element: the 16-byte pieces around it, shifted into place.
    __device__ __forceinline__ void load_around(const T* g) {
        const uintptr_t a = reinterpret_cast<uintptr_t>(g);
        const uint32_t off = (uint32_t)(a & 15);
        const uint4* at = reinterpret_cast<const uint4*>(a & ~(uintptr_t)15);
        uint32_t r[kWords + 4];
#pragma unroll
        for (int q = 0; q < kWords / 4 + 1; ++q) {
            const uint4 v = q < kWords / 4 || off ? __ldg(at + q) : make_uint4(0, 0, 0, 0);
            r[4 * q] = v.x; r[4 * q + 1] = v.y; r[4 * q + 2] = v.z; r[4 * q + 3] = v.w;
        }
#pragma unroll
        for (int q = 0; q < kWords + 2; ++q) r[q] = off & 8 ? r[q + 2] : r[q];
#pragma unroll
        for (int q = 0; q < kWords + 1; ++q) r[q] = off & 4 ? r[q + 1] : r[q];
#pragma unroll
        for (int q = 0; q < kWords; ++q) w[q] = sizeof(T) == 4 ? r[q] : __funnelshift_r(r[q], r[q + 1], (off & 2) * 8);
    }
    // Zeros behind the first n elements.
    __device__ __forceinline__ void keep(int n) {
#pragma unroll
        for (int q = 0; q < kWords; ++q) {
            if constexpr (sizeof(T) == 4)
                w[q] = q < n ? w[q] : 0;
            else
                w[q] = 2 * q + 1 < n ? w[q] : 2 * q < n ? w[q] & 0xFFFF : 0;
        }
    }
    // The parts, `plane` bytes apart.
    __device__ __forceinline__ void store(uint8_t* s, uint32_t plane) const {
        store_to([&](int k) { return s + k * plane; });
    }
    // Part k to place(k).
    template <typename F>
    __device__ __forceinline__ void store_to(F place) const {
        if constexpr (sizeof(T) == 4) {
            uint32_t o[3][4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                float a = __uint_as_float(w[2 * q]), b = __uint_as_float(w[2 * q + 1]);
#pragma unroll
                for (int k = 0; k < 3; ++k) {
                    o[k][q] = k < 2 ? pack2_finite(a, b) : pack2<__nv_bfloat16>(a, b);
                    a -= __uint_as_float(o[k][q] << 16);
                    b -= __uint_as_float(o[k][q] & 0xFFFF0000u);
                }
            }
#pragma unroll
            for (int k = 0; k < 3; ++k)
                *reinterpret_cast<uint4*>(place(k)) = make_uint4(o[k][0], o[k][1], o[k][2], o[k][3]);
        } else {
            *reinterpret_cast<uint4*>(place(0)) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
};

// One operand as rows of consecutive elements: [i][r], or [r][i] when mn.
template <typename T>
struct Operand {
    const T* p;
    int64_t ld, rows, cols;
    bool mn, vec;
    const T* end;  // behind the last element
};
template <typename T>
__device__ __forceinline__ Operand<T> operand(const void* p, int64_t ld, int64_t I, int64_t R, bool mn, bool vec) {
    Operand<T> o{static_cast<const T*>(p), ld, mn ? R : I, mn ? I : R, mn, vec, nullptr};
    o.end = o.p + (o.rows - 1) * ld + o.cols;
    return o;
}

// A tile of an operand, WIDE x 64 elements: thread t of THREADS takes chunk t % 8
// of rows t / 8, t / 8 + THREADS / 8, .. (eight lanes read one row's 64
// elements and fill one 128-byte row of shared memory).
template <typename T, int WIDE, int THREADS>
__device__ __forceinline__ void load_tile(const Operand<T>& o, int64_t i0, int64_t r0, int t,
                                          Chunk<T> (&c)[WIDE * 8 / THREADS]) {
#pragma unroll
    for (int q = 0; q < WIDE * 8 / THREADS; ++q) {
        const int line = t / 8 + THREADS / 8 * q;
        // mn: 64 rows of r per group of 64 i
        const int64_t row = o.mn ? r0 + line % 64 : i0 + line;
        const int64_t col = (o.mn ? i0 + line / 64 * 64 : r0) + t % 8 * 8;
        if (row >= o.rows || col >= o.cols) {
            c[q].zero();
            continue;
        }
        const T* g = o.p + row * o.ld + col;
        const int n = (int)min((int64_t)8, o.cols - col);
        // whole 16-byte pieces are read where the matrix has all of them
        const uintptr_t from = reinterpret_cast<uintptr_t>(g) & ~(uintptr_t)15;
        if (o.vec && n == 8) {
            c[q].load_aligned(g);
        } else if (from >= reinterpret_cast<uintptr_t>(o.p) &&
                   from + 8 * sizeof(T) + 16 <= reinterpret_cast<uintptr_t>(o.end)) {
            c[q].load_around(g);
            if (n < 8) c[q].keep(n);
        } else {
            c[q].load_each(g, n);
        }
    }
}
template <typename T, int WIDE, int THREADS>
__device__ __forceinline__ void store_tile(uint8_t* s, int t, const Chunk<T> (&c)[WIDE * 8 / THREADS]) {
#pragma unroll
    for (int q = 0; q < WIDE * 8 / THREADS; ++q) {
        const int line = t / 8 + THREADS / 8 * q;
        c[q].store(s + line * 128 + ((t % 8) ^ (line & 7)) * 16, WIDE * 128);
    }
}

template <typename T>
bool vectors(const void* q, int64_t ld, int64_t rows) {
    return reinterpret_cast<uintptr_t>(q) % 16 == 0 && (rows <= 1 || ld % (16 / (int64_t)sizeof(T)) == 0);
}

}  // namespace ops
}  // namespace msplat
