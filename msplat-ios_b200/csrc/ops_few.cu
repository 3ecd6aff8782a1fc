// ops_few.cu — layers with few outputs (a colour, a handful of attributes) on
// the FP32 pipes: one thread per row.
//
// With n outputs a row of k inputs brings only 2 n operations per input, far
// below what the tensor cores need to be worth a tile, so the bytes of x are
// the bound. A warp brings 128 bytes of each of its 32 rows at a time into
// shared memory with cp.async, in the 16-byte pieces around them whatever the
// rows' alignment, one group ahead of the one it works on; neighbouring lanes
// take neighbouring pieces. (Each thread reading its own row touches 32 lines
// per instruction.) 1M x 61 -> 3 f16 of an unaligned record takes 54-57 us, 2.4 TB/s;
// what bounds it is issuing the conversions and the masks of a row's two ends.
// The weights are in shared memory as float, read as broadcasts.
#include "ops.cuh"

namespace msplat {
namespace ops {
namespace {

constexpr int kThreads = 128, kWarps = kThreads / 32;
constexpr int kPieces = 9;            // a group: 128 bytes of a row at any alignment
constexpr int kPitch = kPieces * 16;  // a row's group in shared memory: conflict-free in quarters of a warp
constexpr int kBuffer = 32 * kPitch;

__device__ __forceinline__ void copy16(uint32_t to, const void* from, bool ok) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(ok ? 16 : 0) : "memory");
}

template <typename T>
__device__ __forceinline__ void unpack(const uint4& p, float (&v)[16 / sizeof(T)]) {
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

template <typename T, typename TO, int NT, int PIECES>
__global__ void __launch_bounds__(kThreads, 6) k_few(const __grid_constant__ Product p) {
    constexpr int E = 16 / sizeof(T), kGroup = (kPieces - 1) * E;
    extern __shared__ __align__(16) uint8_t dyn[];
    const int N = (int)p.N, K = (int)p.R;
    // weights by input, with a piece's length of zeros on both sides
    float(*ws)[NT] = reinterpret_cast<float(*)[NT]>(dyn) + E;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    uint8_t* buffers = dyn + (size_t)(K + 2 * E) * NT * 4 + warp * 2 * kBuffer;
    const T* x = static_cast<const T*>(p.A);
    const T* w = static_cast<const T*>(p.B);
    const uintptr_t lo = reinterpret_cast<uintptr_t>(x);
    const uintptr_t hi = reinterpret_cast<uintptr_t>(x + (p.M - 1) * p.lda + p.R);
    for (int e = threadIdx.x; e < (K + 2 * E) * NT; e += kThreads) {
        const int k = e / NT - E, n = e % NT;
        ws[k][n] = n < N && k >= 0 && k < K ? to_f32(w[n * p.ldb + k]) : 0.f;
    }
    __syncthreads();
    float bias[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) bias[n] = p.bias && n < N ? to_f32(static_cast<const T*>(p.bias)[n]) : 0.f;

    const int groups = (K + kGroup - 1) / kGroup;
    const int64_t step = (int64_t)gridDim.x * kWarps * 32, row_bytes = p.lda * (int64_t)sizeof(T);
    // this group of the rows from i0 on into a buffer
    auto fetch = [&](int64_t i0, int g, int buffer) {
        const uint32_t to = (uint32_t)__cvta_generic_to_shared(buffers + buffer * kBuffer);
        const uintptr_t base = lo + i0 * row_bytes + (uintptr_t)g * kGroup * sizeof(T);
        const int rows = (int)min((int64_t)32, p.M - i0);
        #pragma unroll
        for (int c = 0; c < PIECES; ++c) {
            const int e = c * 32 + lane, r = e / PIECES, q = e - r * PIECES;
            const uintptr_t from = ((base + r * row_bytes) & ~(uintptr_t)15) + 16 * q;
            const bool ok = r < rows && from >= lo && from + 16 <= hi;
            // (what is not copied still names an aligned address, which the instruction asks for)
            copy16(to + r * kPitch + q * 16, reinterpret_cast<const void*>(ok ? from : lo & ~(uintptr_t)15), ok);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    int64_t i0 = ((int64_t)blockIdx.x * kWarps + warp) * 32;
    int buffer = 0;
    if (i0 < p.M) fetch(i0, 0, 0);
    for (; i0 < p.M; i0 += step) {
        const int64_t i = i0 + lane;
        const T* row = x + min(i, p.M - 1) * p.lda;
        float acc[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[n] = 0.f;
        for (int g = 0; g < groups; ++g) {
            if (g + 1 < groups)
                fetch(i0, g + 1, buffer ^ 1);
            else if (i0 + step < p.M)
                fetch(i0 + step, 0, buffer ^ 1);
            else
                asm volatile("cp.async.commit_group;" ::: "memory");
            asm volatile("cp.async.wait_group 1;" ::: "memory");
            __syncwarp();
            const uintptr_t at = reinterpret_cast<uintptr_t>(row + g * kGroup);
            const int off = (int)(at & 15) / (int)sizeof(T);  // elements before the row's first in its piece
            const uintptr_t from = at & ~(uintptr_t)15;
            const uint8_t* mine = buffers + buffer * kBuffer + lane * kPitch;
            const int begin = g * kGroup, end = min(K, begin + kGroup);
#pragma unroll
            for (int q = 0; q < PIECES; ++q) {
                const int k = begin + q * E - off;  // of the piece's first element
                if (k >= end) continue;
                float f[E];
                unpack<T>(*reinterpret_cast<const uint4*>(mine + q * 16), f);
                const bool each = from + 16 * q < lo || from + 16 * q + 16 > hi;
                if (k < begin || k + E > end || each) {
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        const bool is = k + e >= begin && k + e < end;
                        f[e] = !is ? 0.f : each ? to_f32(row[k + e]) : f[e];
                    }
                }
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const float* we = ws[k] + e * NT;
#pragma unroll
                    for (int n = 0; n < NT; n += 4) {
                        const float4 b = *reinterpret_cast<const float4*>(we + n);
                        acc[n] = fmaf(f[e], b.x, acc[n]);
                        acc[n + 1] = fmaf(f[e], b.y, acc[n + 1]);
                        acc[n + 2] = fmaf(f[e], b.z, acc[n + 2]);
                        acc[n + 3] = fmaf(f[e], b.w, acc[n + 3]);
                    }
                }
            }
            __syncwarp();
            buffer ^= 1;
        }
        if (i >= p.M) continue;
#pragma unroll
        for (int n = 0; n < NT; n += 2) {
            if (n >= N) break;
            const float2 z = make_float2(acc[n] + bias[n], acc[n + 1] + bias[n + 1]), y = activate<TO>(z, p.act);
            auto put = [&](int q, float zq, float yq) {
                if (p.preact) static_cast<TO*>(p.preact)[i * p.ldz + q] = from_f32<TO>(zq);
                if (p.residual) yq += to_f32(static_cast<const TO*>(p.residual)[i * p.ldr + q]);
                static_cast<TO*>(p.out)[i * p.ldo + q] = from_f32<TO>(yq);
            };
            put(n, z.x, y.x);
            if (n + 1 < N) put(n + 1, z.y, y.y);
        }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
}

constexpr int kMostWeights = 32 * 1024;  // bytes of the weights in shared memory

int outputs(int64_t n) { return n <= 4 ? 4 : 8; }

template <typename T, typename TO, int NT>
void run(const Product& p, cudaStream_t s) {
    const bool whole = reinterpret_cast<uintptr_t>(p.A) % 16 == 0 && p.lda * sizeof(T) % 16 == 0;
    const int bytes = (int)(p.R + 32 / sizeof(T)) * NT * 4 + kWarps * 2 * kBuffer;
    constexpr int most = kMostWeights + 16 * NT * 4 + kWarps * 2 * kBuffer;
    // as many blocks as are resident
    const int64_t per = std::min<int64_t>(16, 227 * 1024 / (bytes + 1024));
    const unsigned grid = (unsigned)std::min<int64_t>(ceil_div(p.M, kThreads), kSMs * per);
    note_launches(1);
    if (whole) {
        allow_shared<k_few<T, TO, NT, kPieces - 1>>(most);
        k_few<T, TO, NT, kPieces - 1><<<grid, kThreads, bytes, s>>>(p);
    } else {
        allow_shared<k_few<T, TO, NT, kPieces>>(most);
        k_few<T, TO, NT, kPieces><<<grid, kThreads, bytes, s>>>(p);
    }
    OPS_CK(cudaGetLastError());
}

template <typename T, typename TO>
void sized(const Product& p, cudaStream_t s) {
    if (outputs(p.N) == 4)
        run<T, TO, 4>(p, s);
    else
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

// Measured against the tensor-core kernels (1M rows; 524288 of 256), us here /
// there: f32 16 -> 3 32 / 100, 64 -> 3 61 / 106, 256 -> 3 111 / 168, 64 -> 8
// 75 / 102, 64 -> 16 141 / 106; f16 61 -> 3 unaligned 54 / 165; aligned bf16 16
// -> 3 32 / 71, 16 -> 8 42 / 66, 64 -> 3 44 / 52, 64 -> 8 58 / 46, 256 -> 3 75
// / 63. Few rows leave too few warps for long ones: f32 256 -> 3 takes 16 / 14 with
// 1024 to 8192 rows and 23 / 29 with 65536, 64 -> 3 8 / 10 to 9 / 11, 16 -> 3 6 / 10.
bool can_product_few(const Product& p) {
    if (p.epi != kEpiLinear || p.a_mn || p.b_mn || p.targets || p.alpha_dev || p.alpha != 1.f) return false;
    if (p.N > 8 || p.M < 4096 || p.R * outputs(p.N) * 4 > kMostWeights) return false;
    return !can_product_tc16(p) || p.R <= 32 || (p.N <= 4 && p.R <= 64);
}

void launch_product_few(const Product& p, cudaStream_t s) {
    if (p.dtype == MSPLAT_DTYPE_F32)
        typed<float>(p, s);
    else if (p.dtype == MSPLAT_DTYPE_F16)
        typed<__half>(p, s);
    else
        typed<__nv_bfloat16>(p, s);
}

}  // namespace ops
}  // namespace msplat
