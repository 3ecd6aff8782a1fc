// ops_tc.cuh — the pieces of the tensor-core kernels: barriers, TMA, tcgen05,
// and the ends of a product (ops.cuh) for accumulators that live in TMEM.
#pragma once
#include <cuda.h>

#include "ops_epilogue.cuh"

namespace msplat {
namespace ops {

constexpr int kBM = 128;       // rows of a tile: the lanes of TMEM
constexpr int kBR = 64;        // reduction length of one stage: 128 bytes of a 16-bit type, one swizzle span
constexpr int kEpiWarps = 8;
constexpr int kStagePitch = 20;  // floats per row of the staging buffers (16 columns + 4: conflict-free)
constexpr int kStagingBytes = kEpiWarps * 32 * kStagePitch * 4;

// Set when a wait in a kernel ran out (read and cleared by take_gave_up).
static __device__ unsigned g_ops_gave_up;

// A wait gives up after this many nanoseconds; a block waits only for its own
// copies and products, which take microseconds.
constexpr uint64_t kWaitNs = 2000000000;
__device__ __forceinline__ uint64_t now_ns() {
    uint64_t t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
    return t;
}

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok;
}
// Waits for the phase, at most kWaitNs.
__device__ __forceinline__ bool mbar_wait_bounded(uint32_t bar, uint32_t parity, volatile int* gave_up) {
    const uint64_t end = now_ns() + kWaitNs;
    do {
        if (mbar_try(bar, parity)) return true;
        if (gave_up && *gave_up) return false;
    } while (now_ns() < end);
    return mbar_try(bar, parity);
}
// Waits for the phase; false when this wait, or any other wait of the block,
// gave up.
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile int* gave_up) {
    if (mbar_try(bar, parity)) return true;
    if (mbar_wait_bounded(bar, parity, gave_up)) return true;
    *gave_up = 1;
    atomicOr(&g_ops_gave_up, 1u);
    return false;
}

__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
        ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar)
        : "memory");
}

__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p;
}

__device__ __forceinline__ void tmem_alloc(uint32_t dst, uint32_t cols) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
__device__ __forceinline__ void tmem_free(uint32_t addr, uint32_t cols) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols));
}
__device__ __forceinline__ void tc_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
        : "memory");
}
__device__ __forceinline__ void tmem_load32(uint32_t addr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
}
__device__ __forceinline__ void tmem_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// Shared-memory operand descriptor, 128-byte swizzle. Rows of 128 bytes in
// groups of eight (1024 bytes). Reduction contiguous: a row is one i, the
// groups follow each other along i. Reduction across rows: a row is 64
// consecutive i of one r, the groups follow each other along r, and the next 64
// i start `lead` bytes further on.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lead) {
    return (uint64_t)((addr >> 4) & 0x3FFF) | (uint64_t)((lead >> 4) & 0x3FFF) << 16 | (uint64_t)(1024 >> 4) << 32 |
           1ull << 46 | 2ull << 61;
}
// kind::f16 instruction descriptor: float accumulators, both operands fp16 or
// both bf16, M = 128, N = bn.
inline uint32_t instr_desc(bool bf16, bool a_mn, bool b_mn, int bn) {
    return 1u << 4 | (uint32_t)bf16 << 7 | (uint32_t)bf16 << 10 | (uint32_t)a_mn << 15 | (uint32_t)b_mn << 16 |
           (uint32_t)(bn >> 3) << 17 | (uint32_t)(kBM >> 4) << 24;
}

// Whether a wait gave up in this translation unit's kernels since the last call.
inline bool take_gave_up(cudaStream_t s) {
    unsigned v = 0;
    const unsigned zero = 0;
    OPS_CK(cudaMemcpyFromSymbolAsync(&v, g_ops_gave_up, sizeof(v), 0, cudaMemcpyDeviceToHost, s));
    OPS_CK(cudaStreamSynchronize(s));
    if (v) {
        OPS_CK(cudaMemcpyToSymbolAsync(g_ops_gave_up, &zero, sizeof(v), 0, cudaMemcpyHostToDevice, s));
        OPS_CK(cudaStreamSynchronize(s));
    }
    return v != 0;
}

// How a product is cut into tiles.
struct Tiles {
    int bn;              // columns of a tile: 64, 128 or 256
    int tiles_m, tiles_n;
    int total;           // with the splits of the reduction
    int stages, stage_bytes;
    uint32_t idesc;
    int vec;             // outputs, residual and bias can be accessed four elements at a time
};

// Tile w of a product: its place, its piece of the reduction.
__device__ __forceinline__ void tile_of(const Product& p, const Tiles& tl, int w, int& tm, int& tn, int& split,
                                        int64_t& r0, int64_t& r1) {
    const int per = tl.tiles_m * tl.tiles_n;
    split = w / per;
    w -= split * per;
    tm = w / tl.tiles_n;
    tn = w - tm * tl.tiles_n;
    r0 = 0;
    r1 = p.R;
    if (p.epi == kEpiSlab) {
        r0 = split * p.split_len;
        r1 = min(p.R, r0 + p.split_len);
    }
}

// The end of a product for the 16 columns from j0 of the warp's 32 rows from
// i0, out of the staging buffer: VEC = 4 gives a lane four columns of a row
// (full sectors, one 8 or 16 byte access), VEC = 1 a single one.
template <typename T, typename TO, int EPI, int VEC>
__device__ __forceinline__ void flush16(const Product& p, const float* st, int64_t i0, int64_t j0, int split,
                                        float alpha, uint32_t zero_rows, int lane) {
    constexpr int kLanes = 16 / VEC, kRows = 32 / kLanes;
    const int c = (lane % kLanes) * VEC;
    const int64_t j = j0 + c;
    if (j >= p.N) return;
    float bias[VEC];
#pragma unroll
    for (int q = 0; q < VEC; ++q)
        bias[q] = EPI == kEpiLinear && p.bias && j + q < p.N ? to_f32(static_cast<const T*>(p.bias)[j + q]) : 0.f;
    const bool whole = j + VEC <= p.N;
    union Vec { TO t[VEC]; uint4 q4; uint2 q2; };
#pragma unroll
    for (int k = 0; k < 32 / kRows; ++k) {
        const int row = k * kRows + lane / kLanes;
        const int64_t i = i0 + row;
        if (i >= p.M) continue;
        float v[VEC];
#pragma unroll
        for (int q = 0; q < VEC; ++q) v[q] = st[row * kStagePitch + c + q];
        auto put = [&](TO* to) {
            if (VEC > 1 && whole) {
                Vec o;
#pragma unroll
                for (int q = 0; q < VEC; ++q) o.t[q] = from_f32<TO>(v[q]);
                if (sizeof(TO) == 4)
                    *reinterpret_cast<uint4*>(to) = o.q4;
                else
                    *reinterpret_cast<uint2*>(to) = o.q2;
            } else {
#pragma unroll
                for (int q = 0; q < VEC; ++q)
                    if (j + q < p.N) to[q] = from_f32<TO>(v[q]);
            }
        };
        auto add = [&](const TO* from) {
            if (VEC > 1 && whole) {
                Vec o;
                if (sizeof(TO) == 4)
                    o.q4 = *reinterpret_cast<const uint4*>(from);
                else
                    o.q2 = *reinterpret_cast<const uint2*>(from);
#pragma unroll
                for (int q = 0; q < VEC; ++q) v[q] += to_f32(o.t[q]);
            } else {
#pragma unroll
                for (int q = 0; q < VEC; ++q)
                    if (j + q < p.N) v[q] += to_f32(from[q]);
            }
        };
        if (EPI == kEpiLinear) {
            const bool zero = zero_rows >> row & 1;
#pragma unroll
            for (int q = 0; q < VEC; ++q) v[q] = zero ? 0.f : fmaf(v[q], alpha, bias[q]);
            if (p.preact) put(static_cast<TO*>(p.preact) + i * p.ldz + j);
            if (p.act != MSPLAT_ACT_NONE) {
#pragma unroll
                for (int q = 0; q < VEC; ++q) v[q] = activate(v[q], p.act);
            }
            if (p.residual) add(static_cast<const TO*>(p.residual) + i * p.ldr + j);
            put(static_cast<TO*>(p.out) + i * p.ldo + j);
        } else if (EPI == kEpiSlab) {
            TO* to = reinterpret_cast<TO*>(p.slab) + ((int64_t)split * p.M + i) * p.N + j;
            if (p.accumulate) add(to);
            put(to);
        } else {
            put(static_cast<TO*>(p.out) + i * p.ldo + j);
        }
    }
}

// What a warp needs of its rows over the columns of a tile: thread = row.
struct RowState {
    int64_t i;
    bool in;
    int32_t target;
    float lse, top, sum;
    uint32_t zero_rows;  // kEpiLinear: rows of the warp without a label
    float alpha;
};

template <int EPI>
__device__ __forceinline__ RowState row_begin(const Product& p, int64_t i0, int lane) {
    RowState r;
    r.i = i0 + lane;
    r.in = r.i < p.M;
    r.target = -1;
    r.lse = 0.f;
    r.top = -INFINITY;
    r.sum = 0.f;
    r.zero_rows = 0;
    r.alpha = p.alpha;
    if (EPI == kEpiStats || EPI == kEpiGrad) {
        if (r.in) r.target = __ldg(p.targets + r.i);
        if (EPI == kEpiGrad && r.in) r.lse = __ldg(p.lse + r.i);
    }
    if (EPI == kEpiLinear) {
        if (p.alpha_dev) r.alpha *= __ldg(p.alpha_dev);
        if (p.targets && !p.label_reduces) r.zero_rows = __ballot_sync(~0u, r.in && !labelled(p, r.i));
    }
    return r;
}

// 32 columns from j0 of the accumulators, one row per thread.
template <typename T, int EPI>
__device__ __forceinline__ void columns32(const Product& p, const Tiles& tl, RowState& r, float (&v)[32], int64_t i0,
                                          int64_t j0, int split, float* st, int lane) {
    if (j0 >= p.N) return;
    const int n = (int)min((int64_t)32, p.N - j0);
    if (EPI == kEpiStats) {
        const float to2 = p.logit_scale * kLog2e;
        float top = r.top;
#pragma unroll
        for (int q = 0; q < 32; ++q) {
            v[q] = __fmul_rn(v[q], to2);
            if (q < n) top = fmaxf(top, v[q]);
        }
        const float ref = top == -INFINITY ? 0.f : top;
        float sum = r.sum * (r.top == -INFINITY ? 0.f : exp2f(r.top - ref));
        if (r.top == -INFINITY && r.sum != 0.f) sum = r.sum;  // NaN stays
        const int64_t at = r.target - p.col0 - j0;
#pragma unroll
        for (int q = 0; q < 32; ++q) {
            if (q < n) sum += exp2f(v[q] - ref);
            if (q == at && r.in) p.label_logit[r.i] = v[q];
        }
        r.top = top;
        r.sum = sum;
        return;
    }
    if (EPI == kEpiGrad) {
        const float to2 = p.logit_scale * kLog2e;
        const int64_t at = r.target - p.col0 - j0;
        const bool has = r.in && r.target >= 0 && r.target < p.labels;
#pragma unroll
        for (int q = 0; q < 32; ++q)
            v[q] = has ? epi_grad(__fmul_rn(v[q], to2), r.lse, q == at, p.g_scale) : 0.f;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        if (16 * h >= n) break;
        float4* row = reinterpret_cast<float4*>(st + lane * kStagePitch);
#pragma unroll
        for (int q = 0; q < 4; ++q)
            row[q] = make_float4(v[16 * h + 4 * q], v[16 * h + 4 * q + 1], v[16 * h + 4 * q + 2], v[16 * h + 4 * q + 3]);
        __syncwarp();
        if (EPI == kEpiSlab) {
            if (tl.vec == 4)
                flush16<T, float, EPI, 4>(p, st, i0, j0 + 16 * h, split, 0.f, 0, lane);
            else
                flush16<T, float, EPI, 1>(p, st, i0, j0 + 16 * h, split, 0.f, 0, lane);
        } else if (EPI == kEpiLinear && p.out_dtype == MSPLAT_DTYPE_F32) {
            if (tl.vec == 4)
                flush16<T, float, EPI, 4>(p, st, i0, j0 + 16 * h, split, r.alpha, r.zero_rows, lane);
            else
                flush16<T, float, EPI, 1>(p, st, i0, j0 + 16 * h, split, r.alpha, r.zero_rows, lane);
        } else {
            if (tl.vec == 4)
                flush16<T, T, EPI, 4>(p, st, i0, j0 + 16 * h, split, r.alpha, r.zero_rows, lane);
            else
                flush16<T, T, EPI, 1>(p, st, i0, j0 + 16 * h, split, r.alpha, r.zero_rows, lane);
        }
        __syncwarp();
    }
}

template <int EPI>
__device__ __forceinline__ void row_end(const Product& p, const RowState& r, int64_t block) {
    if (EPI == kEpiStats && r.in) p.stats[(p.stats_block0 + block) * p.stats_ld + r.i] = make_float2(r.top, r.sum);
}

// Columns of a tile: the widest that still gives every SM one, and for the
// label statistics a function of the columns alone (stats_block).
inline int tile_columns(const Product& p, int widest) {
    const int need = p.N > 128 ? 256 : p.N > 64 ? 128 : 64;
    int bn = need < widest ? need : widest;
    if (p.epi == kEpiStats) return bn;
    const int64_t tm = ceil_div(p.M, kBM) * (p.epi == kEpiSlab ? p.splits : 1);
    while (bn > 64 && tm * ceil_div(p.N, bn) < kSMs) bn /= 2;
    return bn;
}

inline bool aligned4(const void* q, int64_t ld, int64_t rows, int es) {
    return !q || (reinterpret_cast<uintptr_t>(q) % (4 * es) == 0 && (rows <= 1 || ld % 4 == 0));
}
inline int pick_vec(const Product& p) {
    if (p.epi == kEpiSlab) return p.N % 4 == 0 ? 4 : 1;
    const int eo = dtype_size(p.out_dtype);
    return aligned4(p.out, p.ldo, p.M, eo) && aligned4(p.residual, p.ldr, p.M, eo) &&
                   aligned4(p.preact, p.ldz, p.M, eo)
               ? 4
               : 1;
}

inline void set_tiles(const Product& p, Tiles& tl) {
    const int64_t tm = ceil_div(p.M, kBM), tn = ceil_div(p.N, tl.bn);
    const int64_t total = tm * tn * (p.epi == kEpiSlab ? p.splits : 1);
    if (total > 0x3fffffff) throw Error(MSPLAT_ERR_CAPACITY, "too many tiles");
    tl.tiles_m = (int)tm;
    tl.tiles_n = (int)tn;
    tl.total = (int)total;
    tl.vec = pick_vec(p);
}

}  // namespace ops
}  // namespace msplat
