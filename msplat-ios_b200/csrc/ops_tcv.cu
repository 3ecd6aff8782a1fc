// ops_tcv.cu — products on the tensor cores whose operands pass through
// registers on their way to shared memory: 32-bit matrices, and 16-bit ones
// that TMA cannot address (odd row strides or starting columns).
//
// A 32-bit factor is the sum of three bf16 numbers, x = h + m + l, each the
// rounded rest of the one before: together they keep its 24 bits. The product
// of two factors is then h h' (accumulated on its own) and h m' + m h' + m m' +
// h l' + l h' (accumulated together, 2^-8 smaller), six tcgen05.mma in place of
// one; what is left out is below 2^-24 of the product. The tensor cores
// truncate when they add (measured: 2e-9 of a sum of one sign per element of the
// reduction, 7e-7 after 512), so a 32-bit reduction changes to a fresh accumulator
// after every 512 elements, and the accumulators are added with rounding by the
// ends, after three of them already where the reduction is longer (LONG: 16384
// elements of one sign are off by 1e-6 of their sum, with the last accumulator
// taking all the rest they were off by 7e-5; 8192 x 2048 -> 1024 takes 350 us, 348
// without). 16-bit reductions take passes where pass_length16 says so, and stay in the
// last accumulator before.
//
// A block owns 128 x bn tiles (bn 64 or 128) and walks its share of them. Warps
// 12-19 load, split and store the stages (the layout is TMA's 128-byte swizzle,
// 64 elements of the reduction per stage), warp 0 issues the products, warps
// 4-11 do the ends of the finished tile from TMEM meanwhile. When the parts of B
// for a tile's columns fit beside the stages (a layer's weights for many rows), a
// block keeps to one column of tiles and loads them once (resident).
//
// 1M x 32 -> 64 f32 takes 117 us without and 179 with GELU and preact kept
// (3.6 TB/s): issuing the split and the ends takes half of the slots, and two
// stages are all that three parts leave room for; one where preact is kept, n is
// above 64 and k in 65 .. 512 (96 KB a stage beside the outputs' boxes).
#include <cstddef>

#include "ops_load.cuh"

namespace msplat {
namespace ops {
namespace {

constexpr int kThreads = 640;
constexpr int kLoaders = 256;
constexpr int kEpiWarps = 8;
constexpr int kLoadWarp = 12;  // the first of the loaders
// Registers per thread of the three kinds of warps, out of the launch's 96 x
// 640: 128 x 40 + 256 x 128 + 256 x 88 = 60416 of 61440.
constexpr int kIssueRegs = 40, kEpiRegs = 128, kLoadRegs = 88;
static_assert(128 * kIssueRegs + 256 * kEpiRegs + 256 * kLoadRegs <= kThreads * 96, "setmaxnreg would wait forever");
constexpr int kMaxStages = 8;
constexpr int kGroup = 8;  // stages (of 64) that one accumulator takes

struct Smem {
    uint64_t full[kMaxStages], empty[kMaxStages];
    uint64_t acc_full[2], acc_empty[2], drain, residual[kEpiWarps][2];
    alignas(16) float bias[kEpiWarps][32];
    uint32_t tmem;
    int gave_up;
};
static_assert(offsetof(Smem, bias) % 16 == 0 && sizeof(Smem) <= 2048, "read as float4; share_memory counts 2048");

// LONG: a reduction longer than a tile's accumulators take (16 bits: than
// pass_length16) goes through them in passes. 32 bits (64 columns): the two groups
// of warps take half of a tile's columns each and hold the passes' sums in
// registers; 16 bits (128 columns): in the columns of TMEM that one accumulator per
// tile leaves.
template <typename T, int EPI, int BN, bool LONG>
__global__ void __launch_bounds__(kThreads, 1)
    k_product_tcv(const __grid_constant__ Product p, const __grid_constant__ Tiles tl,
                  const __grid_constant__ OutMaps maps, const bool vec_a, const bool vec_b) {
    constexpr int P = planes<T>();
    constexpr int kA = P * kBM * 128, kB = P * BN * 128;
    // accumulators of one tile: the groups' and, for split factors, the corrections'
    constexpr bool kInTmem = LONG && P == 1;
    constexpr int kGroups = kInTmem ? 1 : 512 / 2 / BN - (P > 1 ? 1 : 0);
    constexpr int kTileCols = 256;
    constexpr int kPass = kInTmem ? 4096 / kBR : kGroups * kGroup;  // stages of a pass
    static_assert(!LONG || BN == (P > 1 ? 64 : 128), "32 columns per thread are held, boxes of 16 bits have 64");
    // tiles of 64 columns: the two groups of warps take every other tile; wider
    // ones and passes: each takes half of the columns
    constexpr bool kByTile = BN == 64 && !LONG;
    const int stage_bytes = tl.stage_bytes;  // A, and B unless it is resident
    extern __shared__ __align__(1024) uint8_t dyn[];
    __shared__ Smem sm;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    uint8_t* tiles = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(dyn) + 1023) & ~(uintptr_t)1023);
    uint8_t* resident = tiles + (size_t)tl.stages * stage_bytes;
    uint8_t* boxes = resident + (size_t)tl.resident * kB;

    if (threadIdx.x == 0) {
        for (int q = 0; q < tl.stages; ++q) {
            mbar_init(smem_u32(&sm.full[q]), kLoaders / 32);
            mbar_init(smem_u32(&sm.empty[q]), 1);
        }
        for (int q = 0; q < 2; ++q) {
            mbar_init(smem_u32(&sm.acc_full[q]), 1);
            mbar_init(smem_u32(&sm.acc_empty[q]), kByTile ? kEpiWarps / 2 : kEpiWarps);
        }
        mbar_init(smem_u32(&sm.drain), 1);
        for (int q = 0; q < 2 * kEpiWarps; ++q) mbar_init(smem_u32(&sm.residual[q / 2][q % 2]), 1);
        sm.gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) tmem_alloc(smem_u32(&sm.tmem), 2 * kTileCols);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sm.tmem;
    volatile int* gave_up = &sm.gave_up;

    if (warp >= kLoadWarp) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kLoadRegs));
        const int t = threadIdx.x - kLoadWarp * 32;
        const Operand<T> oa = operand<T>(p.A, p.lda, p.M, p.R, p.a_mn, vec_a);
        const Operand<T> ob = operand<T>(p.B, p.ldb, p.N, p.R, p.b_mn, vec_b);
        for (int q = 0; q < tl.resident; ++q) {
            Chunk<T> b[BN / 32];
            load_tile<T, BN, kLoaders>(ob, (int64_t)(blockIdx.x % tl.tiles_n) * BN, (int64_t)q * kBR, t, b);
            store_tile<T, BN, kLoaders>(resident + (size_t)q * kB, t, b);
        }
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int w = blockIdx.x; w < tl.total && ok; w += gridDim.x) {
            int tm, tn, split;
            int64_t r0, r1;
            tile_of(p, tl, w, tm, tn, split, r0, r1);
            for (int64_t r = r0; r < r1; r += kBR) {
                Chunk<T> a[kBM / 32], b[BN / 32];
                load_tile<T, kBM, kLoaders>(oa, (int64_t)tm * kBM, r, t, a);
                if (!tl.resident) load_tile<T, BN, kLoaders>(ob, (int64_t)tn * BN, r, t, b);
                if (!(ok = mbar_wait(smem_u32(&sm.empty[stage]), phase ^ 1, gave_up))) break;
                uint8_t* s = tiles + (size_t)stage * stage_bytes;
                store_tile<T, kBM, kLoaders>(s, t, a);
                if (!tl.resident) store_tile<T, BN, kLoaders>(s + kA, t, b);
                fence_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&sm.full[stage]));
                if (++stage == tl.stages) {
                    stage = 0;
                    phase ^= 1;
                }
            }
        }
    } else if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kIssueRegs));
        int stage = 0, acc = 0;
        uint32_t phase = 0, acc_phase = 0;
        bool ok = true;
        for (int w = blockIdx.x; w < tl.total && ok && warp == 0; w += gridDim.x) {
            int tm, tn, split;
            int64_t r0, r1;
            tile_of(p, tl, w, tm, tn, split, r0, r1);
            if (!(ok = mbar_wait(smem_u32(&sm.acc_empty[acc]), acc_phase ^ 1, gave_up))) break;
            tc_fence_after();
            uint32_t d = tmem + acc * kTileCols, dc = d + kGroups * BN;
            int block = 0;
            for (int64_t r = r0; r < r1; r += kBR, ++block) {
                if (LONG && block == kPass) {
                    if (elect_one()) tc_commit(smem_u32(&sm.acc_full[acc]));
                    __syncwarp();
                    acc ^= 1;
                    if (acc == 0) acc_phase ^= 1;
                    if (!(ok = mbar_wait(smem_u32(&sm.acc_empty[acc]), acc_phase ^ 1, gave_up))) break;
                    tc_fence_after();
                    d = tmem + acc * kTileCols;
                    dc = d + kGroups * BN;
                    block = 0;
                }
                if (!(ok = mbar_wait(smem_u32(&sm.full[stage]), phase, gave_up))) break;
                tc_fence_after();
                if (elect_one()) {
                    const uint32_t a = smem_u32(tiles + (size_t)stage * stage_bytes);
                    const uint32_t b = tl.resident ? smem_u32(resident) + block * kB : a + kA;
                    const uint32_t step_a = p.a_mn ? 2048 >> 4 : 32 >> 4, step_b = p.b_mn ? 2048 >> 4 : 32 >> 4;
                    uint64_t da[P], db[P];
#pragma unroll
                    for (int q = 0; q < P; ++q) {
                        da[q] = smem_desc(a + q * kBM * 128, p.a_mn ? 8192 : 16);
                        db[q] = smem_desc(b + q * BN * 128, p.b_mn ? 8192 : 16);
                    }
                    const int group = min(block / kGroup, kGroups - 1);
                    const bool fresh = block % kGroup == 0 && block / kGroup < kGroups;
                    const int steps = (int)min((int64_t)(kBR / 16), (r1 - r + 15) / 16);
                    for (int k = 0; k < steps; ++k) {
                        if (P > 1) {
                            const int pa[5] = {0, 2, 1, 0, 1}, pb[5] = {2, 0, 1, 1, 0};
#pragma unroll
                            for (int q = 0; q < 5; ++q)
                                tc_mma(dc, da[pa[q]] + k * step_a, db[pb[q]] + k * step_b, tl.idesc,
                                       block > 0 || k > 0 || q > 0);
                        }
                        tc_mma(d + group * BN, da[0] + k * step_a, db[0] + k * step_b, tl.idesc, !fresh || k > 0);
                    }
                    tc_commit(smem_u32(&sm.empty[stage]));
                }
                __syncwarp();
                if (++stage == tl.stages) {
                    stage = 0;
                    phase ^= 1;
                }
            }
            if (!ok) break;
            if (elect_one()) tc_commit(smem_u32(&sm.acc_full[acc]));
            __syncwarp();
            acc ^= 1;
            if (acc == 0) acc_phase ^= 1;
        }
        if (!ok) {
            // products in flight must end before the block frees TMEM
            if (elect_one()) {
                tc_commit(smem_u32(&sm.drain));
                mbar_wait_bounded(smem_u32(&sm.drain), 0, nullptr);
            }
            __syncwarp();
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kEpiRegs));
        constexpr int kHalf = kByTile ? BN : BN / 2;
        const int quarter = warp % 4, group = (warp - 4) / 4, half = kByTile ? 0 : group;
        WarpOut o;
        o.y = boxes + (warp - 4) * tl.warp_bytes;
        o.z = o.y + tl.ring * kBoxBytes;
        o.bias = sm.bias[warp - 4];
        o.bar = smem_u32(sm.residual[warp - 4]);
        o.phase = 0;
        o.k = 0;
        int acc = 0;
        uint32_t acc_phase = 0;
        bool ok = true;
        for (int w = blockIdx.x; w < tl.total && ok; w += gridDim.x) {
            if (kByTile && acc != group) {
                acc ^= 1;
                if (acc == 0) acc_phase ^= 1;
                continue;
            }
            int tm, tn, split;
            int64_t r0, r1;
            tile_of(p, tl, w, tm, tn, split, r0, r1);
            const int64_t i0 = (int64_t)tm * kBM + quarter * 32, j0 = (int64_t)tn * BN + half * kHalf;
            const int64_t j_end = min(p.N, j0 + kHalf);
            RowState row = row_begin<EPI>(p, i0, lane);
            if (EPI == kEpiLinear && j0 < j_end) fetch_residual(p, tl, maps, o, i0, j0, lane);
            float total[LONG && !kInTmem ? 32 : 1];
            const uint32_t sums = tmem + ((uint32_t)quarter << 21) + BN + half * kHalf;  // (kInTmem)
            bool summed = false;
            if (LONG) {  // all passes but the last
#pragma unroll
                for (int q = 0; q < (LONG && !kInTmem ? 32 : 0); ++q) total[q] = 0.f;
                for (; r1 - r0 > kPass * kBR; r0 += kPass * kBR, summed = true) {
                    if (!(ok = mbar_wait(smem_u32(&sm.acc_full[acc]), acc_phase, gave_up))) break;
                    tc_fence_after();
                    const uint32_t d = tmem + ((uint32_t)quarter << 21) + acc * kTileCols + half * kHalf;
                    if constexpr (kInTmem) {
                        for (int c = 0; c < kHalf; c += 32) tmem_sum32(d + c, sums + c, summed);
                    } else {
                        for (int g = kGroups; g >= 0; --g) {  // (the corrections first)
                            uint32_t raw[32];
                            tmem_load32(d + g * BN, raw);
                            tmem_wait();
#pragma unroll
                            for (int q = 0; q < (LONG && !kInTmem ? 32 : 0); ++q) total[q] += __uint_as_float(raw[q]);
                        }
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&sm.acc_empty[acc]));
                    acc ^= 1;
                    if (acc == 0) acc_phase ^= 1;
                }
                if (!ok) break;
            }
            const int parts = (int)min((int64_t)kGroups, (r1 - r0 + kGroup * kBR - 1) / (kGroup * kBR));
            if (!(ok = mbar_wait(smem_u32(&sm.acc_full[acc]), acc_phase, gave_up))) break;
            tc_fence_after();
            if (i0 < p.M) {
                const uint32_t d = tmem + ((uint32_t)quarter << 21) + acc * kTileCols + half * kHalf;
                for (int64_t j = j0; j < j_end && ok; j += 32) {
                    const uint32_t c = (uint32_t)(j - j0);
                    uint32_t raw[32];
                    float v[32];
                    if (P > 1) {
                        tmem_load32(d + kGroups * BN + c, raw);
                        tmem_wait();
#pragma unroll
                        for (int q = 0; q < 32; ++q) v[q] = __uint_as_float(raw[q]);
                    } else {
#pragma unroll
                        for (int q = 0; q < 32; ++q) v[q] = 0.f;
                    }
                    for (int g = 0; g < parts; ++g) {
                        tmem_load32(d + g * BN + c, raw);
                        tmem_wait();
#pragma unroll
                        for (int q = 0; q < 32; ++q) v[q] += __uint_as_float(raw[q]);
                    }
#pragma unroll
                    for (int q = 0; q < (LONG && !kInTmem ? 32 : 0); ++q) v[q] += total[q];
                    if (kInTmem && summed) {
                        tmem_load32(sums + c, raw);
                        tmem_wait();
#pragma unroll
                        for (int q = 0; q < 32; ++q) v[q] += __uint_as_float(raw[q]);
                    }
                    ok = columns32<T, EPI>(p, tl, maps, o, row, v, i0, j0, j, j + 32 < j_end ? j + 32 : p.N, split, lane,
                                           gave_up);
                }
                row_end<EPI>(p, row, kByTile ? tn : 2 * tn + half);
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&sm.acc_empty[acc]));
            acc ^= 1;
            if (acc == 0) acc_phase ^= 1;
        }
        if (EPI != kEpiStats && lane == 0) {
            bulk_wait_all();
            if (!ok && p.residual && tl.tma_out)  // a residual's box may be on its way
                mbar_wait_bounded(o.bar + 8 * (o.k % tl.ring), o.phase >> (o.k % tl.ring) & 1, nullptr);
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 1) tmem_free(tmem, 2 * kTileCols);
}

template <typename T, int EPI, int BN, bool LONG = false>
void run(const Product& p, Tiles tl, cudaStream_t s) {
    OutMaps maps{};
    set_outputs(p, tl, maps);
    constexpr int a_bytes = planes<T>() * kBM * 128, b_bytes = planes<T>() * BN * 128;
    // B's parts stay when a block has several tiles and they leave two stages of A
    const int64_t blocks = ceil_div(p.R, kBR);
    tl.resident = 0;
    int grid = std::min(tl.total, kSMs), bytes = 0;
    if (EPI != kEpiSlab && tl.total > kSMs && tl.tiles_n <= kSMs && blocks * b_bytes <= kBlockBytes) {
        tl.stage_bytes = a_bytes;
        bytes = share_memory(p, tl, kEpiWarps, (int)blocks * b_bytes, 2, kMaxStages);
        if (tl.stages >= 2) {
            tl.resident = (int)blocks;
            grid = kSMs / tl.tiles_n * tl.tiles_n;
        }
    }
    if (!tl.resident) {
        tl.stage_bytes = a_bytes + b_bytes;
        bytes = share_memory(p, tl, kEpiWarps, 0, 2, kMaxStages);
    }
    allow_shared<k_product_tcv<T, EPI, BN, LONG>>(kBlockBytes + 1024);
    note_launches(1);
    k_product_tcv<T, EPI, BN, LONG><<<grid, kThreads, bytes, s>>>(
        p, tl, maps, vectors<T>(p.A, p.lda, p.a_mn ? p.R : p.M), vectors<T>(p.B, p.ldb, p.b_mn ? p.R : p.N));
    OPS_CK(cudaGetLastError());
}

// 32-bit reductions longer than the accumulators of a tile of 64 columns take,
// and 16-bit ones longer than a pass may be.
bool in_passes(const Product& p) {
    return reduction(p) > (p.dtype == MSPLAT_DTYPE_F32 ? 3 * kGroup * kBR : pass_length16(p));
}

template <typename T, int EPI>
void sized(const Product& p, const Tiles& tl, cudaStream_t s) {
    if (in_passes(p)) return run<T, EPI, sizeof(T) == 4 ? 64 : 128, true>(p, tl, s);
    if (tl.bn == 64)
        run<T, EPI, 64>(p, tl, s);
    else
        run<T, EPI, 128>(p, tl, s);
}

template <typename T>
void typed(const Product& p, const Tiles& tl, cudaStream_t s) {
    switch (p.epi) {
        case kEpiLinear: return sized<T, kEpiLinear>(p, tl, s);
        case kEpiSlab: return sized<T, kEpiSlab>(p, tl, s);
        case kEpiStats: return sized<T, kEpiStats>(p, tl, s);
        default: return sized<T, kEpiGrad>(p, tl, s);
    }
}

// 64 columns leave room for more accumulators, which a reduction longer than
// one accumulator's share needs (for 32-bit results).
int columns_tcv(const Product& p) {
    const bool exact = p.dtype == MSPLAT_DTYPE_F32;
    if (in_passes(p)) return exact ? 64 : 128;
    return tile_columns(p, exact && reduction(p) > kGroup * kBR ? 64 : 128);
}

}  // namespace

unsigned gave_up_tcv(cudaStream_t s) { return count_gave_up(s); }
void give_up_tcv(cudaStream_t s) { launch_give_up(s); }

int64_t stats_blocks_tcv(const Product& p) { return in_passes(p) ? 2 * ceil_div(p.N, columns_tcv(p)) : stats_blocks_of(p, columns_tcv(p)); }

void launch_product_tcv(const Product& p, cudaStream_t s) {
    Tiles tl{};
    tl.bn = columns_tcv(p);
    set_tiles(p, tl);
    // the parts of 32-bit factors are bf16
    tl.idesc = instr_desc(p.dtype != MSPLAT_DTYPE_F16, p.a_mn, p.b_mn, tl.bn);
    if (p.dtype == MSPLAT_DTYPE_F32)
        typed<float>(p, tl, s);
    else if (p.dtype == MSPLAT_DTYPE_F16)
        typed<__half>(p, tl, s);
    else
        typed<__nv_bfloat16>(p, tl, s);
}

}  // namespace ops
}  // namespace msplat
