// ops_rows.cu — everything that many rows need against a small matrix, in one
// pass over the rows: the gradients of a narrow layer, and the label loss with
// its gradients against a small table.
//
// With at most 128 columns of w (labels, or a layer's outputs) and 64 of x, all
// that belongs to 128 rows fits into one SM, so x is read once and dx written
// once, and nothing of size rows x columns leaves the chip:
//   labels: s = x w^T; row statistics; g = softmax - one-hot; dx = g w; dw += g^T x
//   layer:  g = dy act'(z);                                dx = g w; dw += g^T x
// x, g and w lie in shared memory once each, in the 128-byte swizzle; the tensor
// cores read the same bytes as rows or transposed (x as A of s and B of dw, g as A
// of dx and of dw, w as B of s and of dx). 32-bit factors are split into three
// bf16 parts as in ops_tcv.cu. dw stays in TMEM for four tiles (512 elements of
// its reduction, because the tensor cores truncate) and is then added to the
// block's own partial sums; the blocks' are summed by launch_slab_sum.
//
// PACK (32-bit x of at most 32 columns): the parts of x and of w lie side by side,
// [h m] in one block of 128-byte rows and [l] in the next, so that one
// instruction multiplies a part of g with all three (or two) of them: three
// reads of g per 16 elements in place of six, which is what the products spend
// their time on (128 x 16 of g are 4 KB of shared memory, as many of x 1 KB).
//
// Warp 0 issues the products, warps 8-15 make g (two warps per 32 rows share a
// row's columns), warps 4-7 load and split x for the next tile and then write dx
// of this one; dw has two accumulators so that one can be drained meanwhile.
// What bounds the kernel is the chain of a tile's steps: x into place, s, g, dw and
// dx, of which those that shared memory has two buffers for overlap. 1M rows x 101
// labels x 32 f32 take 306 us (products, statistics and gradients as passes of
// their own: 1147), the gradients of 1M x 32 -> 64 f32 240 (459); in bf16 199 and 136.
#include <cstddef>

#include "ops_load.cuh"

namespace msplat {
namespace ops {

struct RowsArgs {
    int64_t m;
    int v, d;             // columns of g (rows of w), columns of x and w
    const void* x;
    int64_t ldx;
    const void* w;
    int64_t ldw;
    // labels
    const int32_t* targets;
    float to2, g_scale;   // logits in log2 units; factor of g in 16 bits
    const float* alpha;   // factor of dx
    float* row_loss;
    double* partial;      // [blocks][2]
    // layer
    const void* z;
    int64_t ldz;
    int act;
    const void* dy;
    int64_t lddy;
    float* sums;          // [blocks][v] column sums of g, or null
    // outputs
    void* dx;
    int64_t lddx;
    float* slab;          // [blocks][v][slab_ld(d)], or null
    int dx_tma;
    int vec_x, vec_w, vec_z, vec_dy;
};

namespace {

constexpr int kThreads = 512;
constexpr int kDrain = 4;  // tiles that dw stays in TMEM
constexpr int kSmall = 64 * 128;  // bytes of 64 lines

struct Smem {
    uint64_t x_full[2], x_free[2], s_full, g_full[2], g_free[2], done, out_empty, drain, pair[4];
    alignas(16) float2 half[2][2][kBM];  // by tile parity and half: a row's largest logit and sum
    float sums[8][128];
    double loss[8][2];
    uint32_t tmem;
    int gave_up;
};

__device__ __forceinline__ uint32_t float_bits(float v) { return __float_as_uint(v); }

// Eight values into the parts' swizzled places.
template <typename T>
__device__ __forceinline__ void put8(uint8_t* at, uint32_t plane, const float* v) {
    Chunk<T> c;
#pragma unroll
    for (int q = 0; q < Chunk<T>::kWords; ++q) {
        if constexpr (sizeof(T) == 4)
            c.w[q] = float_bits(v[q]);
        else
            c.w[q] = pack2<T>(v[2 * q], v[2 * q + 1]);
    }
    c.store(at, plane);
}
template <typename T>
__device__ __forceinline__ float chunk_at(const Chunk<T>& c, int q) {
    if constexpr (sizeof(T) == 4) {
        return __uint_as_float(c.w[q]);
    } else {
        const float2 f = unpack2<T>(c.w[q / 2]);
        return q & 1 ? f.y : f.x;
    }
}

__device__ __forceinline__ uint4 load16(const uint4* g, bool ok) {
    // volatile: not moved down to its use, behind the wait that it overlaps
    uint4 v;
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %5, 0;\n\t"
        "mov.b32 %0, 0;\n\tmov.b32 %1, 0;\n\tmov.b32 %2, 0;\n\tmov.b32 %3, 0;\n\t"
        "@p ld.global.nc.v4.b32 {%0, %1, %2, %3}, [%4];\n\t}"
        : "=&r"(v.x), "=&r"(v.y), "=&r"(v.z), "=&r"(v.w)
        : "l"(g), "r"((uint32_t)ok));
    return v;
}

// 128 rows from i0, columns c0 .. c0 + 63, by THREADS threads as load_tile; all
// loads of an aligned matrix are issued before any is used. With targets, rows
// without a label are zeros.
template <typename T, int THREADS>
__device__ __forceinline__ void load_rows(const Operand<T>& o, int64_t i0, int c0, int t, Chunk<T> (&c)[kBM * 8 / THREADS],
                                          const int32_t* targets = nullptr, int labels = 0) {
    constexpr int kN = kBM * 8 / THREADS;
    bool has[kN];
#pragma unroll
    for (int q = 0; q < kN; ++q) {
        const int64_t row = i0 + t / 8 + THREADS / 8 * q;
        has[q] = row < o.rows;
        if (targets && has[q]) {
            const int32_t l = __ldg(targets + row);
            has[q] = l >= 0 && l < labels;
        }
    }
    if (!o.vec) {
        load_tile<T, kBM, THREADS>(o, i0, c0, t, c);
#pragma unroll
        for (int q = 0; q < kN; ++q)
            if (!has[q]) c[q].zero();
        return;
    }
    const int col = c0 + t % 8 * 8, n = (int)min((int64_t)8, o.cols - col);
    const T* g = o.p + (i0 + t / 8) * o.ld + col;
#pragma unroll
    for (int q = 0; q < kN; ++q)
#pragma unroll
        for (int k = 0; k < Chunk<T>::kPieces; ++k) {
            const uint4 v = load16(reinterpret_cast<const uint4*>(g + (int64_t)(THREADS / 8 * q) * o.ld) + k, n == 8 && has[q]);
            c[q].w[4 * k] = v.x; c[q].w[4 * k + 1] = v.y; c[q].w[4 * k + 2] = v.z; c[q].w[4 * k + 3] = v.w;
        }
    if (n > 0 && n < 8) {
#pragma unroll
        for (int q = 0; q < kN; ++q)
            if (has[q]) c[q].load_each(g + (int64_t)(THREADS / 8 * q) * o.ld, n);
    }
}

// The corrections of the parts' products (in front of them, or apart).
template <int P>
__device__ __forceinline__ void corrections(uint32_t d, const uint64_t (&a)[P], const uint64_t (&b)[P], uint32_t idesc,
                                            bool fresh) {
    if constexpr (P > 1) {
        const int pa[5] = {0, 2, 1, 0, 1}, pb[5] = {2, 0, 1, 1, 0};
#pragma unroll
        for (int q = 0; q < 5; ++q) tc_mma(d, a[pa[q]], b[pb[q]], idesc, !fresh || q > 0);
    }
}

template <int P>  // P > 1: with the corrections; 4: with two blocks of them
__device__ __forceinline__ void accumulators(uint32_t d, uint32_t corr, float (&v)[32]) {
    uint32_t raw[32];
    tmem_load32(d, raw);
    tmem_wait();
#pragma unroll
    for (int q = 0; q < 32; ++q) v[q] = __uint_as_float(raw[q]);
    if constexpr (P > 1) {
        tmem_load32(corr, raw);
        tmem_wait();
#pragma unroll
        for (int q = 0; q < 32; ++q) v[q] += __uint_as_float(raw[q]);
    }
    if constexpr (P == 4) {
        tmem_load32(corr + 32, raw);
        tmem_wait();
#pragma unroll
        for (int q = 0; q < 32; ++q) v[q] += __uint_as_float(raw[q]);
    }
}

// Shared memory: the parts of x, w and g, x and then g twice where that fits, and
// dx's boxes.
template <typename T, int VG, bool PACK>
struct Layout {
    static constexpr int P = planes<T>(), kXBlock = kBM * 128, kWBlock = VG * kSmall, kGPlane = VG * kBM * 128;
    static constexpr int blocks = PACK ? 2 : P;  // of x and of w
    static constexpr int most = 227 * 1024 - sizeof(Smem) - 1024, w = blocks * kWBlock, rest = 4 * kBoxBytes + 1024,
                         x = blocks * kXBlock, g = P * kGPlane;
    static constexpr int x_buffers = 2 * x + w + g + rest <= most ? 2 : 1;
    static constexpr int g_buffers = x_buffers * x + w + 2 * g + rest <= most ? 2 : 1;
    static constexpr int bytes = x_buffers * x + w + g_buffers * g + rest;
    static_assert(bytes <= most, "shared memory of a block");
    // where part q begins in blocks of `block` bytes
    __device__ static constexpr int part(int q, int block) { return PACK ? (q >> 1) * block + (q & 1) * 64 : q * block; }
};
// The parts of eight elements of a line, `piece` the first of them / 8.
template <typename T, bool PACK>
__device__ __forceinline__ void store_parts(const Chunk<T>& c, uint8_t* s, int line, int piece, int block) {
    if (PACK && piece >= 4) return;
    c.store_to([&](int k) {
        const int at = PACK ? piece + 4 * (k & 1) : piece;
        return s + (PACK ? k >> 1 : k) * block + line * 128 + ((at ^ (line & 7)) << 4);
    });
}

// v[at] for at in 0 .. 31, by halving
__device__ __forceinline__ float pick32(const float (&v)[32], int at) {
    float a[16];
#pragma unroll
    for (int q = 0; q < 16; ++q) a[q] = at & 1 ? v[2 * q + 1] : v[2 * q];
#pragma unroll
    for (int q = 0; q < 8; ++q) a[q] = at & 2 ? a[2 * q + 1] : a[2 * q];
#pragma unroll
    for (int q = 0; q < 4; ++q) a[q] = at & 4 ? a[2 * q + 1] : a[2 * q];
#pragma unroll
    for (int q = 0; q < 2; ++q) a[q] = at & 8 ? a[2 * q + 1] : a[2 * q];
    return at & 16 ? a[1] : a[0];
}

template <typename T, bool LABELS, int VG, int ACT, bool PACK>
__global__ void __launch_bounds__(kThreads, 1)
    k_rows(const __grid_constant__ RowsArgs p, const __grid_constant__ CUtensorMap map_dx, const uint32_t idesc_s,
           const uint32_t idesc_x, const uint32_t idesc_w) {
    static_assert(!PACK || sizeof(T) == 4, "parts");
    constexpr int P = planes<T>();
    using L = Layout<T, VG, PACK>;
    constexpr int kXBlock = L::kXBlock, kWBlock = L::kWBlock, kGPlane = L::kGPlane, kGGroup = kBM * 128;
    constexpr int kXBuffers = L::x_buffers, kBuffers = L::g_buffers;
    // with two buffers of x a tile's s comes before the last tile's dw and dx, so
    // that its g is made while they run
    constexpr bool kAhead = LABELS && kXBuffers == 2;
    // TMEM: s (its corrections are added first, while the sums are small), dx and
    // two times dw with their corrections apart (PACK: in the 64 columns after
    // the 32 of the sum)
    constexpr uint32_t kS = 0, kX = 128, kW = 256, kCorr = PACK ? 32 : 64, kWNext = 128;
    const uint32_t narrower = 4u << 17;  // 32 columns less in an instruction descriptor
    extern __shared__ __align__(1024) uint8_t dyn[];
    __shared__ Smem sm;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    uint8_t* xs = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(dyn) + 1023) & ~(uintptr_t)1023);
    uint8_t* ws = xs + kXBuffers * L::x;
    uint8_t* g0 = ws + L::blocks * kWBlock;
    uint8_t* boxes = g0 + kBuffers * P * kGPlane;
    const int64_t tiles = (p.m + kBM - 1) / kBM;

    if (threadIdx.x == 0) {
        mbar_init(smem_u32(&sm.s_full), 1);
        for (int q = 0; q < 2; ++q) {
            mbar_init(smem_u32(&sm.x_full[q]), 4);
            mbar_init(smem_u32(&sm.x_free[q]), 1);
            mbar_init(smem_u32(&sm.g_full[q]), 8);
            mbar_init(smem_u32(&sm.g_free[q]), 1);
        }
        mbar_init(smem_u32(&sm.done), 1);
        mbar_init(smem_u32(&sm.out_empty), 4);
        mbar_init(smem_u32(&sm.drain), 1);
        for (int q = 0; q < 4; ++q) mbar_init(smem_u32(&sm.pair[q]), 2);
        sm.gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) tmem_alloc(smem_u32(&sm.tmem), 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sm.tmem;
    volatile int* gave_up = &sm.gave_up;
    uint32_t phase = 0;  // of this block's current tile, for the barriers with one buffer
    const int count_all = (int)((tiles - blockIdx.x + gridDim.x - 1) / gridDim.x);

    // dx of tile count - 1 out of TMEM, whose products are done, and dw after
    // every kDrain tiles: by the loaders between two tiles, or for a layer, whose
    // g takes less time, by the first four of the warps that make it.
    const int quarter = warp % 4;
    const uint32_t d = tmem + ((uint32_t)quarter << 21);
    uint8_t* box = boxes + quarter * kBoxBytes;
    const float alpha = LABELS ? __ldg(p.alpha) : 1.f;
    float* mine = p.slab ? p.slab + ((int64_t)blockIdx.x * p.v + quarter * 32 + lane) * slab_ld(p.d) : nullptr;
    const bool keeps = p.slab && quarter * 32 + lane < p.v;
    auto write_out = [&](int count) {
        const int64_t i0 = (blockIdx.x + (int64_t)(count - 1) * gridDim.x) * kBM + quarter * 32;
        tc_fence_after();
        if (p.dx && i0 < p.m) {
            bool zero = false;
            if (LABELS && i0 + lane < p.m) {
                const int32_t l = __ldg(p.targets + i0 + lane);
                zero = l < 0 || l >= p.v;
            }
            for (int c = 0; c < p.d; c += 32) {
                float v[32];
                accumulators<PACK ? 4 : P>(d + kX + c, d + kX + kCorr + c, v);
                if (LABELS) {
#pragma unroll
                    for (int q = 0; q < 32; ++q) v[q] = zero ? 0.f : v[q] * alpha;
                }
                const int first = sizeof(T) == 2 && c ? 4 : 0;
                const bool send = sizeof(T) == 4 || c + 32 >= p.d;
                if (p.dx_tma && first == 0) {
                    if (lane == 0) bulk_wait_read(0);
                    __syncwarp();
                }
                box_write<T>(box, lane, first, v);
                if (p.dx_tma) {
                    if (!send) continue;
                    fence_async();
                    __syncwarp();
                    if (lane == 0) {
                        tma_store(&map_dx, smem_u32(box), first ? 0 : c, (int)i0, 0, false);
                        bulk_commit();
                    }
                } else {
                    __syncwarp();
                    box_copy<T, false>(box, first, static_cast<T*>(p.dx), p.lddx, i0, c, p.m, p.d, lane);
                    __syncwarp();
                }
            }
        }
        // dx's accumulators are free; dw's other ones too: they were drained
        // before this step, in program order
        const bool drains = p.slab && (count % kDrain == 0 || count == count_all);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sm.out_empty));
        if (drains) {
            const uint32_t dw = d + kW + ((count - 1) / kDrain & 1) * kWNext;
            for (int c = 0; c < p.d; c += 32) {
                float v[32];
                accumulators<PACK ? 4 : P>(dw + c, dw + kCorr + c, v);
                if (!keeps) continue;
                // only this thread adds to its row, in this order
                float* o = mine + c;
                const int n = ((int)slab_ld(p.d) - c) / 4;
#pragma unroll
                for (int q = 0; q < 8; ++q) {
                    if (q >= n) break;
                    if (count <= kDrain)
                        *reinterpret_cast<float4*>(o + 4 * q) =
                            make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
                    else
                        asm volatile("red.relaxed.gpu.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(o + 4 * q),
                                     "f"(v[4 * q]), "f"(v[4 * q + 1]), "f"(v[4 * q + 2]), "f"(v[4 * q + 3])
                                     : "memory");
                }
            }
            tc_fence_before();
        }
    };

    if (warp < 4) {
        const uint32_t w = smem_u32(ws);
        auto issue_s = [&](int count) {
            const uint32_t x = smem_u32(xs + count % kXBuffers * L::x);
            if (elect_one()) {
                const int steps = (p.d + 15) / 16;
                const uint64_t da = smem_desc(x, 16), db = smem_desc(w, 16);
                uint64_t a[P], b[P];
                for (int turn = P > 1 ? 0 : 1; turn < 2; ++turn) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        if (k >= steps) break;
#pragma unroll
                        for (int q = 0; q < P; ++q) {
                            a[q] = da + ((L::part(q, kXBlock) + k * 32) >> 4);
                            b[q] = db + ((L::part(q, kWBlock) + k * 32) >> 4);
                        }
                        if (turn == 0)
                            corrections<P>(tmem + kS, a, b, idesc_s, k == 0);
                        else
                            tc_mma(tmem + kS, a[0], b[0], idesc_s, P > 1 || k > 0);
                    }
                }
                tc_commit(smem_u32(&sm.s_full));
            }
            __syncwarp();
        };
        auto issue_gradients = [&](int count) {
            const int buffer = count % kBuffers;
            const uint32_t x = smem_u32(xs + count % kXBuffers * L::x), g = smem_u32(g0 + buffer * L::g);
            if (elect_one()) {
                // dw first: x is free for the next tile while dx runs
                // (descriptors advance by constants: this one thread's instructions
                // are what the products wait for when the other warps are busy)
                uint64_t a[P], b[P];
                if (p.slab) {
                    // of a single group the second 64 rows of the result are not read
                    const uint64_t da = smem_desc(g, kGGroup), db = smem_desc(x, PACK ? kXBlock : 16);
                    const uint32_t dw = tmem + kW + (count / kDrain & 1) * kWNext;
                    const bool add = count % kDrain != 0;
#pragma unroll
                    for (int k = 0; k < kBM / 16; ++k) {
#pragma unroll
                        for (int q = 0; q < P; ++q) {
                            a[q] = da + ((q * kGPlane + k * 2048) >> 4);
                            b[q] = db + (((PACK ? 0 : q * kXBlock) + k * 2048) >> 4);
                        }
                        if constexpr (PACK) {
                            tc_mma(dw, a[0], b[0], idesc_w, add || k > 0);
                            tc_mma(dw + 32, a[1], b[0], idesc_w - narrower, true);
                            tc_mma(dw + 64, a[2], b[0], idesc_w - 2 * narrower, true);
                        } else {
                            corrections<P>(dw + kCorr, a, b, idesc_w, !add && k == 0);
                            tc_mma(dw, a[0], b[0], idesc_w, add || k > 0);
                        }
                    }
                }
                tc_commit(smem_u32(&sm.x_free[count % kXBuffers]));
                if (p.dx) {
                    const uint64_t da = smem_desc(g, 16), db = smem_desc(w, PACK ? kWBlock : 16);
#pragma unroll
                    for (int k = 0; k < 4 * VG; ++k) {
                        if (k * 16 >= p.v) break;
#pragma unroll
                        for (int q = 0; q < P; ++q) {
                            a[q] = da + ((q * kGPlane + k / 4 * kGGroup + k % 4 * 32) >> 4);
                            b[q] = db + (((PACK ? 0 : q * kWBlock) + k * 2048) >> 4);
                        }
                        if constexpr (PACK) {
                            tc_mma(tmem + kX, a[0], b[0], idesc_x, k > 0);
                            tc_mma(tmem + kX + 32, a[1], b[0], idesc_x - narrower, true);
                            tc_mma(tmem + kX + 64, a[2], b[0], idesc_x - 2 * narrower, true);
                        } else {
                            corrections<P>(tmem + kX + kCorr, a, b, idesc_x, k == 0);
                            tc_mma(tmem + kX, a[0], b[0], idesc_x, k > 0);
                        }
                    }
                }
                tc_commit(smem_u32(&sm.g_free[buffer]));
                tc_commit(smem_u32(&sm.done));
            }
            __syncwarp();
        };
        bool ok = true;
        for (int count = 0; warp == 0 && count < count_all; ++count, phase ^= 1) {
            if (!(ok = mbar_wait(smem_u32(&sm.x_full[count % kXBuffers]), count / kXBuffers & 1, gave_up))) break;
            tc_fence_after();
            if (LABELS) issue_s(count);
            if (kAhead && count > 0) {
                if (!(ok = mbar_wait(smem_u32(&sm.out_empty), phase, gave_up))) break;
                tc_fence_after();
                issue_gradients(count - 1);
            }
            if (!(ok = mbar_wait(smem_u32(&sm.g_full[count % kBuffers]), count / kBuffers & 1, gave_up))) break;
            tc_fence_after();
            if (!kAhead) {
                if (!(ok = mbar_wait(smem_u32(&sm.out_empty), phase ^ 1, gave_up))) break;
                tc_fence_after();
                issue_gradients(count);
            }
        }
        if (kAhead && ok && warp == 0) {
            if ((ok = mbar_wait(smem_u32(&sm.out_empty), phase, gave_up))) {
                tc_fence_after();
                issue_gradients(count_all - 1);
            }
        }
        if (!ok && warp == 0) {
            if (elect_one()) {
                tc_commit(smem_u32(&sm.drain));
                mbar_wait_bounded(smem_u32(&sm.drain), 0, nullptr);
            }
            __syncwarp();
        }
    } else if (warp < 8) {
        const int t = threadIdx.x - 128;
        const Operand<T> ox = operand<T>(p.x, p.ldx, p.m, p.d, false, p.vec_x);
        const Operand<T> ow = operand<T>(p.w, p.ldw, p.v, p.d, false, p.vec_w);
        // a layer's x is read for dw only, its w for dx only (either may be null)
        const bool reads_x = LABELS || p.slab, reads_w = LABELS || p.dx;
        for (int q = 0; reads_w && q < VG; ++q) {
            Chunk<T> c[4];
            load_tile<T, 64, 128>(ow, 64 * q, 0, t, c);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int line = t / 8 + 16 * e;
                store_parts<T, PACK>(c[e], ws + q * kSmall, line, t % 8, kWBlock);
            }
        }
        // x of a tile into its buffer
        auto bring = [&](int count) {
            const int64_t tile = blockIdx.x + (int64_t)count * gridDim.x;
            Chunk<T> c[8];
            if (reads_x) load_rows<T, 128>(ox, tile * kBM, 0, t, c, LABELS ? p.targets : nullptr, p.v);
            const int buffer = count % kXBuffers;
            if (!mbar_wait(smem_u32(&sm.x_free[buffer]), (count / kXBuffers & 1) ^ 1, gave_up)) return false;
            if (reads_x) {
#pragma unroll
                for (int q = 0; q < 8; ++q)
                    store_parts<T, PACK>(c[q], xs + buffer * L::x, t / 8 + 16 * q, t % 8, kXBlock);
            }
            fence_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&sm.x_full[buffer]));
            // the next tile's rows start towards L2
            const int64_t ahead = (tile + gridDim.x) * kBM + t;
            if (reads_x && ahead < p.m)
                for (int e = 0; e < p.d; e += 128 / (int)sizeof(T))
                    asm volatile("prefetch.global.L2 [%0];" ::"l"(ox.p + ahead * p.ldx + e));
            return true;
        };
        // step `count`: x goes in as far ahead as there are buffers, dx of the
        // tile before comes out
        bool ok = kXBuffers == 1 || bring(0);
        for (int count = 0; ok && count <= count_all; ++count, phase ^= 1) {
            if (count + kXBuffers - 1 < count_all && !bring(count + kXBuffers - 1)) break;
            if (!LABELS || count == 0) continue;
            if (!mbar_wait(smem_u32(&sm.done), phase ^ 1, gave_up)) break;
            write_out(count);
        }
        if (lane == 0) bulk_wait_all();
    } else {
        if constexpr (LABELS) {
            const int half = (warp - 8) / 4, line = quarter * 32 + lane;
            const uint32_t s = tmem + ((uint32_t)quarter << 21) + half * 32 * VG;
            double sum = 0, count = 0;
            int turn = 0;
            for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x, phase ^= 1, ++turn) {
                const int64_t i = tile * kBM + line;
                const int32_t target = i < p.m ? __ldg(p.targets + i) : -1;
                const bool has = target >= 0 && target < p.v;
                if (!mbar_wait(smem_u32(&sm.s_full), phase, gave_up)) break;
                tc_fence_after();
                float v[VG][32], top = -INFINITY, mine = 0.f;
                const int at = target - half * 32 * VG;
                const bool holds = has && at >= 0 && at < 32 * VG;
#pragma unroll
                for (int c = 0; c < VG; ++c) {
                    accumulators<1>(s + kS + 32 * c, 0, v[c]);
#pragma unroll
                    for (int q = 0; q < 32; ++q) v[c][q] = __fmul_rn(v[c][q], p.to2);
                    const int left = p.v - half * 32 * VG - 32 * c;
                    if (left < 32) {
#pragma unroll
                        for (int q = 0; q < 32; ++q) v[c][q] = q < left ? v[c][q] : -INFINITY;
                    }
                    float tops[4] = {top, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int q = 0; q < 32; ++q) tops[q % 4] = fmaxf(tops[q % 4], v[c][q]);
                    top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
                    const float picked = pick32(v[c], at);
                    mine = at >> 5 == c ? picked : mine;
                }
                const float ref = top == -INFINITY ? 0.f : top;
                float more[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int c = 0; c < VG; ++c)
#pragma unroll
                    for (int q = 0; q < 32; ++q) {
                        v[c][q] = exp2_fast(v[c][q] - ref);
                        more[q % 4] += v[c][q];
                    }
                const float total = (more[0] + more[1]) + (more[2] + more[3]);
                // the two halves of a row
                const int parity = phase;
                sm.half[parity][half][line] = make_float2(ref, total);
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&sm.pair[quarter]));
                if (!mbar_wait(smem_u32(&sm.pair[quarter]), phase, gave_up)) break;
                const float2 o = sm.half[parity][half ^ 1][line];
                // (a half without columns has the sum 0 and no say)
                const float all = o.y == 0.f ? ref : total == 0.f ? o.x : fmaxf(ref, o.x);
                const float up = total == 0.f ? 0.f : exp2_fast(ref - all);
                const float sums = total * up + (o.y == 0.f ? 0.f : o.y * exp2_fast(o.x - all));
                const float row = ((all - mine) + log2f(sums)) * kLn2;
                if (holds) {
                    sum += row;
                    count += 1;
                }
                if (p.row_loss && i < p.m && (holds || (!has && half == 0))) p.row_loss[i] = has ? row : 0.f;
                // rows without a label have x = 0 here and the factor 0; their values are
                // finite unless a label's w is not (0 times that is NaN, and so is the sum)
                const float factor = has ? up / sums : 0.f, scaled = sizeof(T) == 2 ? factor * p.g_scale : factor;
                if (!has && sums != sums) {
#pragma unroll
                    for (int c = 0; c < VG; ++c)
#pragma unroll
                        for (int q = 0; q < 32; ++q) v[c][q] = 0.f;
                }
                const int buffer = turn % kBuffers;
                if (!mbar_wait(smem_u32(&sm.g_free[buffer]), (turn / kBuffers & 1) ^ 1, gave_up)) break;
                uint8_t* out = g0 + buffer * P * kGPlane + line * 128;
#pragma unroll
                for (int c = 0; c < VG; ++c)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int piece = half * 4 * VG + 4 * c + e;
                        float g[8];
#pragma unroll
                        for (int q = 0; q < 8; ++q) g[q] = v[c][8 * e + q] * scaled;
                        put8<T>(out + piece / 8 * kGGroup + ((piece % 8) ^ (line & 7)) * 16, kGPlane, g);
                    }
                if (holds) {  // the one-hot, over what was just written
                    float g = exp2_fast(mine - ref) * factor - 1.f;
                    if (sizeof(T) == 2) g *= p.g_scale;
                    uint8_t* one = out + target / 64 * kGGroup + ((target / 8 % 8) ^ (line & 7)) * 16 + target % 8 * 2;
                    if constexpr (sizeof(T) == 2) {
                        *reinterpret_cast<T*>(one) = from_f32<T>(g);
                    } else {
#pragma unroll
                        for (int q = 0; q < P; ++q) {
                            const __nv_bfloat16 h = __float2bfloat16_rn(g);
                            *reinterpret_cast<__nv_bfloat16*>(one + q * kGPlane) = h;
                            g -= __bfloat162float(h);
                        }
                    }
                }
                fence_async();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&sm.g_full[buffer]));
            }
            for (int q = 16; q; q >>= 1) {
                sum += __shfl_xor_sync(~0u, sum, q);
                count += __shfl_xor_sync(~0u, count, q);
            }
            if (lane == 0) {
                sm.loss[warp - 8][0] = sum;
                sm.loss[warp - 8][1] = count;
            }
        } else {
            const int t = threadIdx.x - 256;
            const Operand<T> oy = operand<T>(p.dy, p.lddy, p.m, p.v, false, p.vec_dy);
            const Operand<T> oz = operand<T>(p.z, p.ldz, p.m, p.v, false, p.vec_z);
            float sums[VG][8];
#pragma unroll
            for (int c = 0; c < VG; ++c)
#pragma unroll
                for (int e = 0; e < 8; ++e) sums[c][e] = 0.f;
            bool ok = true;
            int turn = 0;
            for (int64_t tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x, ++turn) {
                const int buffer = turn % kBuffers;
                uint8_t* gs = g0 + buffer * P * kGPlane;
#pragma unroll
                for (int c = 0; c < VG; ++c) {
                    Chunk<T> a[4], b[4];
                    load_rows<T, 256>(oy, tile * kBM, 64 * c, t, a);
                    if (ACT != MSPLAT_ACT_NONE) load_rows<T, 256>(oz, tile * kBM, 64 * c, t, b);
                    if (c == 0 && !(ok = mbar_wait(smem_u32(&sm.g_free[buffer]), (turn / kBuffers & 1) ^ 1, gave_up))) break;
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const int line = t / 8 + 32 * q;
                        float g[8];
#pragma unroll
                        for (int e = 0; e < 8; e += 2) {
                            float2 v = make_float2(chunk_at(a[q], e), chunk_at(a[q], e + 1));
                            if (ACT != MSPLAT_ACT_NONE)
                                v = __fmul2_rn(v, act_slope<ACT, T>(make_float2(chunk_at(b[q], e), chunk_at(b[q], e + 1))));
                            g[e] = v.x;
                            g[e + 1] = v.y;
                            sums[c][e] += v.x;
                            sums[c][e + 1] += v.y;
                        }
                        put8<T>(gs + c * kGGroup + line * 128 + ((t % 8) ^ (line & 7)) * 16, kGPlane, g);
                    }
                }
                if (!ok) break;
                fence_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&sm.g_full[buffer]));
                // the next tile's rows start towards L2, two threads a row
                const int64_t ahead = (tile + gridDim.x) * kBM + t / 2;
                if (ahead < p.m)
                    for (int e = t % 2 * (128 / (int)sizeof(T)); e < p.v; e += 256 / (int)sizeof(T)) {
                        asm volatile("prefetch.global.L2 [%0];" ::"l"(oy.p + ahead * p.lddy + e));
                        if (ACT != MSPLAT_ACT_NONE)
                            asm volatile("prefetch.global.L2 [%0];" ::"l"(oz.p + ahead * p.ldz + e));
                    }
                if (warp < 12 && turn > 0) {
                    if (!(ok = mbar_wait(smem_u32(&sm.done), (turn & 1) ^ 1, gave_up))) break;
                    write_out(turn);
                }
            }
            if (warp < 12 && ok && mbar_wait(smem_u32(&sm.done), (count_all & 1) ^ 1, gave_up)) write_out(count_all);
            if (lane == 0) bulk_wait_all();
#pragma unroll
            for (int c = 0; c < VG; ++c)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    float s = sums[c][e];
                    s += __shfl_xor_sync(~0u, s, 8);
                    s += __shfl_xor_sync(~0u, s, 16);
                    if (lane < 8) sm.sums[warp - 8][64 * c + 8 * lane + e] = s;
                }
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 1) tmem_free(tmem, 512);
    if (LABELS) {
        if (threadIdx.x == 0) {
            double sum = 0, count = 0;
            for (int q = 0; q < 8; ++q) {
                sum += sm.loss[q][0];
                count += sm.loss[q][1];
            }
            p.partial[2 * blockIdx.x] = sum;
            p.partial[2 * blockIdx.x + 1] = count;
        }
    } else if (p.sums && threadIdx.x < p.v) {
        float s = 0.f;
        for (int q = 0; q < 8; ++q) s += sm.sums[q][threadIdx.x];
        p.sums[(int64_t)blockIdx.x * p.v + threadIdx.x] = s;
    }
}

template <typename T, bool LABELS, int VG, int ACT, bool PACK>
void run(const RowsArgs& a, const CUtensorMap& dx, cudaStream_t s) {
    constexpr int bytes = Layout<T, VG, PACK>::bytes;
    const bool bf16 = !std::is_same<T, __half>::value;
    const int nv = (int)round_up(a.v, 16), nd = PACK ? 96 : (int)round_up(a.d, 16);
    allow_shared<k_rows<T, LABELS, VG, ACT, PACK>>(bytes);
    note_launches(1);
    k_rows<T, LABELS, VG, ACT, PACK><<<rows_blocks(a.m), kThreads, bytes, s>>>(
        a, dx, instr_desc(bf16, false, false, nv), instr_desc(bf16, false, true, nd), instr_desc(bf16, true, true, nd));
    OPS_CK(cudaGetLastError());
}

template <typename T, bool LABELS, int ACT, bool PACK>
void wide(const RowsArgs& a, const CUtensorMap& dx, cudaStream_t s) {
    if (a.v <= 64)
        run<T, LABELS, 1, ACT, PACK>(a, dx, s);
    else
        run<T, LABELS, 2, ACT, PACK>(a, dx, s);
}
template <typename T, bool LABELS, int ACT>
void sized(const RowsArgs& a, const CUtensorMap& dx, cudaStream_t s) {
    if constexpr (sizeof(T) == 4) {
        if (a.d <= 32) return wide<T, LABELS, ACT, true>(a, dx, s);
    }
    wide<T, LABELS, ACT, false>(a, dx, s);
}

template <typename T>
void typed(RowsArgs a, int dtype, cudaStream_t s) {
    a.vec_x = vectors<T>(a.x, a.ldx, a.m);
    a.vec_w = vectors<T>(a.w, a.ldw, a.v);
    a.vec_z = a.z && vectors<T>(a.z, a.ldz, a.m);
    a.vec_dy = a.dy && vectors<T>(a.dy, a.lddy, a.m);
    CUtensorMap dx{};
    a.dx_tma = a.dx && tma_ready(a.dx, a.lddx, a.m, sizeof(T));
    if (a.dx_tma) dx = map_output(a.dx, a.m, a.d, a.lddx, 1, dtype);
    if (a.targets) return sized<T, true, MSPLAT_ACT_NONE>(a, dx, s);
    switch (a.act) {
        case MSPLAT_ACT_RELU: return sized<T, false, MSPLAT_ACT_RELU>(a, dx, s);
        case MSPLAT_ACT_GELU: return sized<T, false, MSPLAT_ACT_GELU>(a, dx, s);
        case MSPLAT_ACT_SILU: return sized<T, false, MSPLAT_ACT_SILU>(a, dx, s);
        case MSPLAT_ACT_SIGMOID: return sized<T, false, MSPLAT_ACT_SIGMOID>(a, dx, s);
        default: return sized<T, false, MSPLAT_ACT_NONE>(a, dx, s);
    }
}

void launch(const RowsArgs& a, int dtype, cudaStream_t s) {
    if (dtype == MSPLAT_DTYPE_F32)
        typed<float>(a, dtype, s);
    else if (dtype == MSPLAT_DTYPE_F16)
        typed<__half>(a, dtype, s);
    else
        typed<__nv_bfloat16>(a, dtype, s);
}

}  // namespace

unsigned gave_up_rows(cudaStream_t s) { return count_gave_up(s); }
void give_up_rows(cudaStream_t s) { launch_give_up(s); }

// Measured against the passes of ops_tcv.cu and ops_tc16.cu, us here / there with
// m rows, gradients of a layer with GELU and label loss with gradients:
//   f32   128 x 64: m 4096 26 / 45, 35 / 69; 8192 27 / 45, 37 / 71; 1M 470 / 688, 379 / 1057
//   f32   16 x 16:  m 8192 20 / 39, 27 / 64; 1M 213 / 338, 250 / 533
//   bf16  128 x 64: m 4096 21 / 31, 29 / 51; 8192 21 / 31, 29 / 51; 1M 260 / 313, 230 / 559
//   bf16  16 x 16:  m 8192 18 / 29, 26 / 49; 1M 129 / 162, 152 / 309
// A loss without gradients is slower here (f32 128 x 64: 8192 27 / 22, 1M 283 / 216),
// but is the same number as with them. 128 x 64 is what shared memory and TMEM
// hold; fewer rows leave SMs without a tile.
bool fits_rows(int64_t m, int64_t v, int64_t d) { return v <= 128 && d <= 64 && m >= 8192; }
int rows_blocks(int64_t m) { return (int)std::min<int64_t>(ceil_div(m, kBM), kSMs); }

void launch_rows_labels(int64_t m, int64_t v, int64_t d, const void* x, int64_t ldx, const void* w, int64_t ldw,
                        const int32_t* targets, float logit_scale, float g_scale, const float* alpha, float* row_loss,
                        double* partial, void* dx, int64_t lddx, float* slab, int dtype, cudaStream_t s) {
    RowsArgs a{};
    a.m = m; a.v = (int)v; a.d = (int)d;
    a.x = x; a.ldx = ldx; a.w = w; a.ldw = ldw;
    a.targets = targets; a.to2 = logit_scale * kLog2e; a.g_scale = g_scale; a.alpha = alpha;
    a.row_loss = row_loss; a.partial = partial;
    a.dx = dx; a.lddx = lddx; a.slab = slab;
    launch(a, dtype, s);
}

void launch_rows_layer(int64_t m, int64_t n, int64_t k, const void* x, int64_t ldx, const void* w, int64_t ldw,
                       const void* z, int64_t ldz, int act, const void* dy, int64_t lddy, void* dx, int64_t lddx,
                       float* slab, float* sums, int dtype, cudaStream_t s) {
    RowsArgs a{};
    a.m = m; a.v = (int)n; a.d = (int)k;
    a.x = x; a.ldx = ldx; a.w = w; a.ldw = ldw;
    a.z = z; a.ldz = ldz; a.act = act; a.dy = dy; a.lddy = lddy;
    a.dx = dx; a.lddx = lddx; a.slab = slab; a.sums = sums;
    launch(a, dtype, s);
}

}  // namespace ops
}  // namespace msplat
