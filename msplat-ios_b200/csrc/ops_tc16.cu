// ops_tc16.cu — products of 16-bit matrices on the 5th-generation tensor cores.
//
// A block owns a 128 x bn tile of the result at a time (bn 64, 128 or 256) and
// walks the tiles of its SM. Warp 0 brings 64 columns of the reduction per stage
// with TMA (128-byte swizzle, out-of-range elements read as zeros, so no size is
// special); warp 1 issues tcgen05.mma from shared memory into one of two
// accumulators in TMEM; warps 4-11 read the other accumulator, 32 lanes x 32
// columns at a time, and do the end of the product while the next tile runs.
// Either operand may have the reduction across its rows (dx, dw): TMA then
// brings boxes of 64 x 64 and the instruction reads them transposed, so no
// operand is ever copied into another layout.
//
// 65536 x 1024 x 1024 bf16 takes 113 us without an activation (1216 TFLOP/s; the
// library's product 102), 144 with GELU and a residual (176 at a sustained run's
// clocks), whose ends then take as long as the products; 8192 x 32768 x 512 softmax
// statistics 183 (1500 TFLOP/s, tensor pipe 84%). With a reduction of 64 the ends bound it: 65536 x 1024 in 54.
#include <cstddef>

#include "ops_tc.cuh"

namespace msplat {
namespace ops {

namespace {

constexpr int kThreads = 384;
constexpr int kEpiWarps = 8;
constexpr int kMaxStages = 8;

struct Smem {
    uint64_t full[kMaxStages], empty[kMaxStages];
    uint64_t acc_full[2], acc_empty[2], drain, residual[kEpiWarps][2];
    alignas(16) float bias[kEpiWarps][32];
    uint32_t tmem;
    int gave_up;
};
static_assert(offsetof(Smem, bias) % 16 == 0 && sizeof(Smem) <= 2048, "read as float4; share_memory counts 2048");

// LONG: a reduction longer than pass_length16 goes through the accumulators in
// passes, whose sums the ends keep in the TMEM behind them: tiles of 128 columns with
// two accumulators, or of 256 with one (8192 x 8192 -> 4096 bf16 into f32 takes
// 423 us so, 546 in tiles of 128, and 410 in one pass with three times the error). A
// kernel of its own: tests for passes took 11% of 1M x 64 -> 64 and 4% of the wide
// layer.
template <typename T, int EPI, bool LONG>
__global__ void __launch_bounds__(kThreads, 1)
    k_product_tc16(const __grid_constant__ Product p, const __grid_constant__ Tiles tl,
                   const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                   const __grid_constant__ OutMaps maps) {
    extern __shared__ __align__(1024) uint8_t dyn[];
    __shared__ Smem sm;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    uint8_t* tiles = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(dyn) + 1023) & ~(uintptr_t)1023);
    uint8_t* boxes = tiles + (size_t)tl.stages * tl.stage_bytes;
    const uint32_t tmem_cols = LONG ? 512 : 2 * tl.bn;

    if (threadIdx.x == 0) {
        for (int q = 0; q < tl.stages; ++q) {
            mbar_init(smem_u32(&sm.full[q]), 1);
            mbar_init(smem_u32(&sm.empty[q]), 1);
        }
        for (int q = 0; q < 2; ++q) {
            mbar_init(smem_u32(&sm.acc_full[q]), 1);
            mbar_init(smem_u32(&sm.acc_empty[q]), tl.bn == 64 ? kEpiWarps / 2 : kEpiWarps);
        }
        mbar_init(smem_u32(&sm.drain), 1);
        for (int q = 0; q < 2 * kEpiWarps; ++q) mbar_init(smem_u32(&sm.residual[q / 2][q % 2]), 1);
        sm.gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 2) tmem_alloc(smem_u32(&sm.tmem), tmem_cols);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sm.tmem;
    volatile int* gave_up = &sm.gave_up;
    // to the next accumulator
    auto next = [&](int& acc, uint32_t& acc_phase) {
        const bool one = LONG && tl.bn == 256;
        if (!one) acc ^= 1;
        if (acc == 0) acc_phase ^= 1;
    };

    if (warp == 0) {
        if (elect_one()) {
            int stage = 0;
            uint32_t phase = 0;
            int64_t fills = 0;
            bool ok = true;
            for (int w = blockIdx.x; w < tl.total && ok; w += gridDim.x) {
                int tm, tn, split;
                int64_t r0, r1;
                tile_of(p, tl, w, tm, tn, split, r0, r1);
                for (int64_t r = r0; r < r1; r += kBR) {
                    if (!(ok = mbar_wait(smem_u32(&sm.empty[stage]), phase ^ 1, gave_up))) break;
                    const uint32_t bar = smem_u32(&sm.full[stage]);
                    const uint32_t a = smem_u32(tiles + (size_t)stage * tl.stage_bytes), b = a + kBM * 128;
                    mbar_expect(bar, tl.stage_bytes);
                    if (p.a_mn) {
                        for (int q = 0; q < kBM / 64; ++q)
                            tma_load(a + q * 8192, &map_a, tm * kBM + q * 64, (int)r, bar);
                    } else {
                        tma_load(a, &map_a, (int)r, tm * kBM, bar);
                    }
                    if (p.b_mn) {
                        for (int q = 0; q < tl.bn / 64; ++q)
                            tma_load(b + q * 8192, &map_b, tn * tl.bn + q * 64, (int)r, bar);
                    } else {
                        tma_load(b, &map_b, (int)r, tn * tl.bn, bar);
                    }
                    ++fills;
                    if (++stage == tl.stages) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
            }
            if (!ok) {
                // the copies in flight must land before the block may end
                const int out = (int)min(fills, (int64_t)tl.stages);
                for (int q = 0; q < out; ++q) {
                    if (--stage < 0) {
                        stage = tl.stages - 1;
                        phase ^= 1;
                    }
                    mbar_wait_bounded(smem_u32(&sm.full[stage]), phase, nullptr);
                }
            }
        }
    } else if (warp == 1) {
        int stage = 0, acc = 0;
        uint32_t phase = 0, acc_phase = 0;
        bool ok = true;
        for (int w = blockIdx.x; w < tl.total && ok; w += gridDim.x) {
            int tm, tn, split;
            int64_t r0, r1;
            tile_of(p, tl, w, tm, tn, split, r0, r1);
            if (!(ok = mbar_wait(smem_u32(&sm.acc_empty[acc]), acc_phase ^ 1, gave_up))) break;
            tc_fence_after();
            uint32_t d = tmem + acc * tl.bn;
            int block = 0;
            for (int64_t r = r0; r < r1; r += kBR, ++block) {
                if (LONG && block == tl.pass) {
                    if (elect_one()) tc_commit(smem_u32(&sm.acc_full[acc]));
                    __syncwarp();
                    next(acc, acc_phase);
                    if (!(ok = mbar_wait(smem_u32(&sm.acc_empty[acc]), acc_phase ^ 1, gave_up))) break;
                    tc_fence_after();
                    d = tmem + acc * tl.bn;
                    block = 0;
                }
                if (!(ok = mbar_wait(smem_u32(&sm.full[stage]), phase, gave_up))) break;
                tc_fence_after();
                if (elect_one()) {
                    const uint32_t a = smem_u32(tiles + (size_t)stage * tl.stage_bytes), b = a + kBM * 128;
                    const uint64_t da = smem_desc(a, p.a_mn ? 8192 : 16), db = smem_desc(b, p.b_mn ? 8192 : 16);
                    const uint32_t step_a = p.a_mn ? 2048 >> 4 : 32 >> 4, step_b = p.b_mn ? 2048 >> 4 : 32 >> 4;
#pragma unroll
                    for (int k = 0; k < kBR / 16; ++k)
                        tc_mma(d, da + k * step_a, db + k * step_b, tl.idesc, (LONG ? block > 0 : r > r0) || k > 0);
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
            next(acc, acc_phase);
        }
        if (!ok) {
            // products in flight must end before the block frees TMEM
            if (elect_one()) {
                tc_commit(smem_u32(&sm.drain));
                mbar_wait_bounded(smem_u32(&sm.drain), 0, nullptr);
            }
            __syncwarp();
        }
    } else if (warp >= 4) {
        // tiles of 64 columns: the two groups of warps take every other tile;
        // wider ones: each takes half of the columns
        const int quarter = warp % 4, group = (warp - 4) / 4;
        const bool by_tile = tl.bn == 64;
        const int half = by_tile ? 0 : group, columns = by_tile ? 64 : tl.bn / 2;
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
            if (by_tile && acc != group) {
                next(acc, acc_phase);
                continue;
            }
            int tm, tn, split;
            int64_t r0, r1;
            tile_of(p, tl, w, tm, tn, split, r0, r1);
            const int64_t i0 = (int64_t)tm * kBM + quarter * 32, j0 = (int64_t)tn * tl.bn + half * columns;
            const int64_t j_end = min(p.N, j0 + columns);
            RowState row = row_begin<EPI>(p, i0, lane);
            if (EPI == kEpiLinear && j0 < j_end) fetch_residual(p, tl, maps, o, i0, j0, lane);
            // the sums of all passes but the last
            const uint32_t sums = tmem + ((uint32_t)quarter << 21) + 256 + half * columns;
            bool summed = false;
            for (; LONG && r1 - r0 > tl.pass * kBR; r0 += tl.pass * kBR, summed = true) {
                if (!(ok = mbar_wait(smem_u32(&sm.acc_full[acc]), acc_phase, gave_up))) break;
                tc_fence_after();
                const uint32_t d = tmem + ((uint32_t)quarter << 21) + acc * tl.bn + half * columns;
                for (int c = 0; c < columns; c += 32) tmem_sum32(d + c, sums + c, summed);
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&sm.acc_empty[acc]));
                next(acc, acc_phase);
            }
            if (LONG && !ok) break;
            if (!(ok = mbar_wait(smem_u32(&sm.acc_full[acc]), acc_phase, gave_up))) break;
            tc_fence_after();
            if (i0 < p.M) {
                const uint32_t d = tmem + ((uint32_t)quarter << 21) + acc * tl.bn + half * columns;
                for (int64_t j = j0; j < j_end && ok; j += 32) {
                    uint32_t raw[32];
                    tmem_load32(d + (uint32_t)(j - j0), raw);
                    tmem_wait();
                    float v[32];
#pragma unroll
                    for (int q = 0; q < 32; ++q) v[q] = __uint_as_float(raw[q]);
                    if (LONG && summed) {
                        tmem_load32(sums + (uint32_t)(j - j0), raw);
                        tmem_wait();
#pragma unroll
                        for (int q = 0; q < 32; ++q) v[q] += __uint_as_float(raw[q]);
                    }
                    ok = columns32<T, EPI>(p, tl, maps, o, row, v, i0, j0, j, j + 32 < j_end ? j + 32 : p.N, split, lane,
                                           gave_up);
                }
                row_end<EPI>(p, row, by_tile ? tn : 2 * tn + half);
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&sm.acc_empty[acc]));
            next(acc, acc_phase);
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
    if (warp == 2) tmem_free(tmem, tmem_cols);
}

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn encoder() {
    static EncodeFn fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult found;
        OPS_CK(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &found));
        if (found != cudaDriverEntryPointSuccess || !p) throw Error(MSPLAT_ERR_CUDA, "no cuTensorMapEncodeTiled");
        return reinterpret_cast<EncodeFn>(p);
    }();
    return fn;
}

struct Maps {
    CUtensorMap a, b;
    OutMaps out;
};

template <typename T, int EPI, bool LONG>
void run_as(const Product& p, const Tiles& tl, const Maps& m, int bytes, cudaStream_t s) {
    allow_shared<k_product_tc16<T, EPI, LONG>>(kBlockBytes + 1024);
    note_launches(1);
    k_product_tc16<T, EPI, LONG><<<std::min(tl.total, kSMs), kThreads, bytes, s>>>(p, tl, m.a, m.b, m.out);
    OPS_CK(cudaGetLastError());
}
template <typename T, int EPI>
void run(const Product& p, const Tiles& tl, const Maps& m, int bytes, cudaStream_t s) {
    tl.pass ? run_as<T, EPI, true>(p, tl, m, bytes, s) : run_as<T, EPI, false>(p, tl, m, bytes, s);
}

template <typename T>
void typed(const Product& p, const Tiles& tl, const Maps& m, int bytes, cudaStream_t s) {
    switch (p.epi) {
        case kEpiLinear: return run<T, kEpiLinear>(p, tl, m, bytes, s);
        case kEpiSlab: return run<T, kEpiSlab>(p, tl, m, bytes, s);
        case kEpiStats: return run<T, kEpiStats>(p, tl, m, bytes, s);
        default: return run<T, kEpiGrad>(p, tl, m, bytes, s);
    }
}

}  // namespace

CUtensorMap map_operand(const void* base, int64_t rows, int64_t cols, int64_t ld, int box_rows, int dtype) {
    CUtensorMap m;
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)(rows > 1 ? ld * 2 : round_up(cols * 2, 16))};
    const cuuint32_t box[2] = {64, (cuuint32_t)box_rows}, step[2] = {1, 1};
    const CUresult r = encoder()(
        &m, dtype == MSPLAT_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2,
        const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) throw Error(MSPLAT_ERR_CUDA, "cuTensorMapEncodeTiled failed");
    return m;
}

CUtensorMap map_output(const void* base, int64_t rows, int64_t cols, int64_t ld, int64_t layers, int dtype) {
    CUtensorMap m;
    const int es = dtype_size(dtype);
    const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)layers};
    const cuuint64_t row = (cuuint64_t)(rows > 1 || layers > 1 ? ld * es : round_up(cols * es, 16));
    const cuuint64_t strides[2] = {row, row * (cuuint64_t)rows};
    const cuuint32_t box[3] = {(cuuint32_t)(128 / es), 32, 1}, step[3] = {1, 1, 1};
    const CUresult r = encoder()(
        &m, dtype == MSPLAT_DTYPE_F32    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
            : dtype == MSPLAT_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                         : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
        3, const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) throw Error(MSPLAT_ERR_CUDA, "cuTensorMapEncodeTiled failed");
    return m;
}

// Strides of a descriptor stay below 2^40 bytes.
bool tma_ready(const void* p, int64_t ld, int64_t rows, int elem) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 &&
           (rows <= 1 || (ld * elem % 16 == 0 && ld * elem < (1ll << 40) / rows));
}

unsigned gave_up_tc16(cudaStream_t s) { return count_gave_up(s); }
void give_up_tc16(cudaStream_t s) { launch_give_up(s); }

bool can_product_tc16(const Product& p) {
    return p.dtype != MSPLAT_DTYPE_F32 && tma_ready(p.A, p.lda, p.a_mn ? p.R : p.M, 2) &&
           tma_ready(p.B, p.ldb, p.b_mn ? p.R : p.N, 2);
}

static bool in_passes(const Product& p) { return reduction(p) > pass_length16(p); }
static int columns_tc16(const Product& p) { return std::max(in_passes(p) ? 128 : 64, tile_columns(p, 256)); }
int64_t stats_blocks_tc16(const Product& p) { return stats_blocks_of(p, columns_tc16(p)); }

void launch_product_tc16(const Product& p, cudaStream_t s) {
    Tiles tl{};
    tl.bn = columns_tc16(p);
    tl.pass = in_passes(p) ? (int)(pass_length16(p) / kBR) : 0;
    set_tiles(p, tl);
    tl.stage_bytes = (kBM + tl.bn) * 128;
    tl.idesc = instr_desc(p.dtype == MSPLAT_DTYPE_BF16, p.a_mn, p.b_mn, tl.bn);
    Maps m{};
    m.a = p.a_mn ? map_operand(p.A, p.R, p.M, p.lda, kBR, p.dtype) : map_operand(p.A, p.M, p.R, p.lda, kBM, p.dtype);
    m.b = p.b_mn ? map_operand(p.B, p.R, p.N, p.ldb, kBR, p.dtype)
                 : map_operand(p.B, p.N, p.R, p.ldb, tl.bn, p.dtype);
    set_outputs(p, tl, m.out);
    const int bytes = share_memory(p, tl, kEpiWarps, 0, tl.bn == 256 ? 4 : 5, kMaxStages);
    if (p.dtype == MSPLAT_DTYPE_F16)
        typed<__half>(p, tl, m, bytes, s);
    else
        typed<__nv_bfloat16>(p, tl, m, bytes, s);
}

}  // namespace ops
}  // namespace msplat
