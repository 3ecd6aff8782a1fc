// ops_tc.cuh — the pieces of the tensor-core kernels: barriers, TMA, tcgen05,
// and the ends of a product (ops.cuh) for accumulators that live in TMEM.
#pragma once
#include <atomic>
#include <cuda.h>

#include "ops.cuh"

namespace msplat {
namespace ops {

constexpr int kBM = 128;       // rows of a tile: the lanes of TMEM
constexpr int kBR = 64;        // reduction length of one stage: 128 bytes of a 16-bit type, one swizzle span

// How many waits of this file's kernels ran out (each .cu file has its own).
static __device__ unsigned g_ops_gave_up;

// A wait gives up after this many nanoseconds; a block waits only for its own
// copies and products, which take microseconds.
constexpr uint64_t kWaitNs = 2000000000;
__device__ __forceinline__ uint64_t now_ns() {
    uint64_t t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
    return t;
}

__device__ __forceinline__ bool labelled(const Product& p, int64_t row) {
    const int32_t t = __ldg(p.targets + row);
    return t >= 0 && t < p.labels;
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
// Waits for the phase, at most `ns`.
__device__ __forceinline__ bool mbar_wait_bounded(uint32_t bar, uint32_t parity, volatile int* gave_up,
                                                  uint64_t ns = kWaitNs) {
    const uint64_t end = now_ns() + ns;
    do {
        if (mbar_try(bar, parity)) return true;
        if (gave_up && *gave_up) return false;
    } while (now_ns() < end);
    return mbar_try(bar, parity);
}
// Waits for the phase; false when this wait, or any other wait of the block,
// gave up.
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile int* gave_up, uint64_t ns = kWaitNs) {
    if (mbar_try(bar, parity)) return true;
    if (mbar_wait_bounded(bar, parity, gave_up, ns)) return true;
    *gave_up = 1;
    atomicAdd(&g_ops_gave_up, 1u);
    return false;
}

__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
        ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar)
        : "memory");
}

__device__ __forceinline__ void tma_store(const CUtensorMap* map, uint32_t src, int x, int y, int z, bool add) {
    if (add)
        asm volatile("cp.reduce.async.bulk.tensor.3d.global.shared::cta.add.tile.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(
                         map),
                     "r"(src), "r"(x), "r"(y), "r"(z)
                     : "memory");
    else
        asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(map),
                     "r"(src), "r"(x), "r"(y), "r"(z)
                     : "memory");
}
__device__ __forceinline__ void tma_load3(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
        ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(0), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
// all but the last `pending` (0 or 1) groups of stores have read their buffers
__device__ __forceinline__ void bulk_wait_read(int pending) {
    if (pending)
        asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
    else
        asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
}
__device__ __forceinline__ void bulk_wait_all() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

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
__device__ __forceinline__ void tmem_store32(uint32_t addr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};"
        ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
        "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
        "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(addr)
        : "memory");
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// Adds 32 columns of an accumulator, with rounding, to (or first puts them in) sums
// that the warp keeps in TMEM.
__device__ __forceinline__ void tmem_sum32(uint32_t acc, uint32_t sums, bool add) {
    uint32_t v[32], w[32];
    tmem_load32(acc, v);
    if (add) tmem_load32(sums, w);
    tmem_wait();
    if (add) {
#pragma unroll
        for (int q = 0; q < 32; ++q) v[q] = __float_as_uint(__uint_as_float(v[q]) + __uint_as_float(w[q]));
    }
    tmem_store32(sums, v);
}

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

// How many waits gave up in this file's kernels, once the stream (of the current
// device) has finished. Static, as the counter is: one definition for all files
// would read one file's.
static unsigned count_gave_up(cudaStream_t s) {
    unsigned v = 0;
    OPS_CK(cudaMemcpyFromSymbolAsync(&v, g_ops_gave_up, sizeof(v), 0, cudaMemcpyDeviceToHost, s));
    OPS_CK(cudaStreamSynchronize(s));
    return v;
}
// A wait of a millisecond for a barrier at which nobody arrives.
static __global__ void k_give_up() {
    __shared__ uint64_t bar;
    __shared__ int gave_up;
    gave_up = 0;
    mbar_init(smem_u32(&bar), 1);
    mbar_wait(smem_u32(&bar), 0, &gave_up, 1000000);
}
static void launch_give_up(cudaStream_t s) {
    note_launches(1);
    k_give_up<<<1, 1, 0, s>>>();
    OPS_CK(cudaGetLastError());
}

// How a product is cut into tiles.
struct Tiles {
    int bn;              // columns of a tile: 64, 128 or 256
    int tiles_m, tiles_n;
    int total;           // with the splits of the reduction
    int stages, stage_bytes;
    uint32_t idesc;
    int resident;        // stages of B that stay in shared memory (ops_tcv.cu)
    int pass;            // stages of a pass through the accumulators, 0: all in one (ops_tc16.cu)
    // the outputs' boxes in shared memory
    int tma_out;         // they move by TMA (16-byte aligned outputs), else element by element
    int ring;            // boxes per output and warp, 1 or 2
    int warp_bytes;      // what a warp needs: boxes of y and preact
};

struct OutMaps {
    CUtensorMap y, z, r;
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

// Dynamic shared memory for stages and boxes: without the static part (2048)
// and, in kBlockBytes + 1024, with room to align the stages.
constexpr int kBlockBytes = 227 * 1024 - 2048 - 1024;

// A warp's boxes. A box holds 32 rows of 128 bytes (32 or 64 columns) in TMA's
// 128-byte swizzle: a thread writes its row's 16-byte pieces without bank
// conflicts and one instruction stores the box, clipped at the matrix' edges.
// (Rows of 64 bytes halve what the TMA unit stores per clock: 65536 x 1024 bf16
// from a reduction of 64 took 53 us with them.)
constexpr int kBoxBytes = 32 * 128;
struct WarpOut {
    uint8_t* y;       // ring boxes
    uint8_t* z;       // ring boxes, with preact
    float* bias;      // 32 floats
    uint32_t bar;     // 2 barriers for the residual's boxes
    uint32_t phase;   // their phases
    int k;            // boxes done
};

__device__ __forceinline__ uint32_t box_piece(int row, int piece) { return row * 128 + ((piece ^ (row & 7)) << 4); }
// Two values rounded into one 32-bit word of a 16-bit type, and back.
template <typename TO>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename TO>
__device__ __forceinline__ float2 unpack2(uint32_t w);
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t w) {
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
// 32 columns of a row from piece `first` on
template <typename TO>
__device__ __forceinline__ void box_write(uint8_t* box, int row, int first, const float (&v)[32]) {
    if constexpr (sizeof(TO) == 4) {
#pragma unroll
        for (int q = 0; q < 8; ++q)
            *reinterpret_cast<float4*>(box + box_piece(row, first + q)) =
                make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
    } else {
#pragma unroll
        for (int q = 0; q < 4; ++q)
            *reinterpret_cast<uint4*>(box + box_piece(row, first + q)) =
                make_uint4(pack2<TO>(v[8 * q], v[8 * q + 1]), pack2<TO>(v[8 * q + 2], v[8 * q + 3]),
                           pack2<TO>(v[8 * q + 4], v[8 * q + 5]), pack2<TO>(v[8 * q + 6], v[8 * q + 7]));
    }
}
template <typename TO>
__device__ __forceinline__ void box_add(const uint8_t* box, int row, int first, float (&v)[32]) {
    if constexpr (sizeof(TO) == 4) {
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            const float4 f = *reinterpret_cast<const float4*>(box + box_piece(row, first + q));
            v[4 * q] += f.x;
            v[4 * q + 1] += f.y;
            v[4 * q + 2] += f.z;
            v[4 * q + 3] += f.w;
        }
    } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const uint4 w = *reinterpret_cast<const uint4*>(box + box_piece(row, first + q));
            const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float2 f = unpack2<TO>(u[e]);
                v[8 * q + 2 * e] += f.x;
                v[8 * q + 2 * e + 1] += f.y;
            }
        }
    }
}
// Element by element between 32 columns of a box and rows i0 .., columns j0 ..
// of a matrix: consecutive lanes take consecutive elements.
template <typename TO, bool IN>
__device__ __forceinline__ void box_copy(uint8_t* box, int first, TO* g, int64_t ld, int64_t i0, int64_t j0, int64_t M,
                                         int64_t N, int lane) {
    constexpr int per = 16 / sizeof(TO);
    const int n = (int)min((int64_t)32, N - j0), rows = (int)min((int64_t)32, M - i0);
    if (rows == 32) {
        // a row per step, sixteen of them in flight (lanes behind the last column
        // read it once more)
        TO* m = g + i0 * ld + j0 + min(lane, n - 1);
        const int piece = first + lane / per, within = lane % per;
        const bool mine = lane < n;
#pragma unroll
        for (int r0 = 0; r0 < 32; r0 += 16) {
            TO v[16];
#pragma unroll
            for (int r = 0; r < 16; ++r)
                v[r] = IN ? m[(r0 + r) * ld] : reinterpret_cast<TO*>(box + box_piece(r0 + r, piece))[within];
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                if (IN)
                    reinterpret_cast<TO*>(box + box_piece(r0 + r, piece))[within] = v[r];
                else if (mine)
                    m[(r0 + r) * ld] = v[r];
            }
        }
        return;
    }
    for (int e = lane; e < rows * n; e += 32) {
        const int r = e / n, c = e - r * n;
        TO* b = reinterpret_cast<TO*>(box + box_piece(r, first + c / per)) + c % per;
        TO* m = g + (i0 + r) * ld + j0 + c;
        if (IN)
            *b = *m;
        else
            *m = *b;
    }
}

template <typename TO>
__device__ __forceinline__ void activate32(float (&v)[32], int act) {
    constexpr bool FULL = sizeof(TO) == 4;
    auto pairs = [&](auto f) {
#pragma unroll
        for (int q = 0; q < 32; q += 2) {
            const float2 y = f(make_float2(v[q], v[q + 1]));
            v[q] = y.x;
            v[q + 1] = y.y;
        }
    };
    switch (act) {
        case MSPLAT_ACT_RELU: pairs([](float2 z) { return make_float2(act_relu(z.x), act_relu(z.y)); }); break;
        case MSPLAT_ACT_GELU: pairs([](float2 z) { return act_gelu<FULL>(z); }); break;
        case MSPLAT_ACT_SILU: pairs([](float2 z) { return act_silu<FULL>(z); }); break;
        case MSPLAT_ACT_SIGMOID: pairs([](float2 z) { return act_sigmoid<FULL>(z); }); break;
        default: break;
    }
}

// What a warp needs of its rows over the columns of a tile: thread = row.
struct RowState {
    int64_t i;
    bool in, zero;
    int32_t target;
    float top, sum, alpha;  // (kEpiGrad: sum is the factor of the exponentials)
};

template <int EPI>
__device__ __forceinline__ RowState row_begin(const Product& p, int64_t i0, int lane) {
    RowState r;
    r.i = i0 + lane;
    r.in = r.i < p.M;
    r.target = -1;
    r.top = -INFINITY;
    r.sum = 0.f;
    r.zero = false;
    r.alpha = p.alpha;
    if (EPI == kEpiStats || EPI == kEpiGrad) {
        if (r.in) r.target = __ldg(p.targets + r.i);
        if (EPI == kEpiGrad && r.in) {
            const float2 norm = __ldg(p.norm + r.i);
            r.top = norm.x;
            r.sum = norm.y * p.g_scale;
        }
    }
    if (EPI == kEpiLinear) {
        if (p.alpha_dev) r.alpha *= __ldg(p.alpha_dev);
        if (p.targets) r.zero = r.in && !labelled(p, r.i);
    }
    return r;
}

// Starts the residual's box at (i0, j0) towards the warp's next box. Its store
// of `ring` boxes ago has been read (bulk_wait_read).
__device__ __forceinline__ void fetch_residual(const Product& p, const Tiles& tl, const OutMaps& maps, const WarpOut& o,
                                               int64_t i0, int64_t j0, int lane) {
    if (!p.residual || !tl.tma_out || j0 >= p.N || i0 >= p.M || lane != 0) return;
    const int b = o.k % tl.ring;
    mbar_expect(o.bar + 8 * b, kBoxBytes);
    tma_load3(smem_u32(o.y + b * kBoxBytes), &maps.r, (int)j0, (int)i0, o.bar + 8 * b);
}

__device__ __forceinline__ void boxes_free(const Tiles& tl, int lane) {
    if (lane == 0) bulk_wait_read(tl.ring - 1);
    __syncwarp();
}

// The end of a product for 32 x 32 results, one row per thread, through the
// warp's boxes. j_begin: the warp's first columns of the tile; j_next: the tile's next columns (N or above: none).
template <typename T, typename TO, int EPI>
__device__ __forceinline__ bool write32(const Product& p, const Tiles& tl, const OutMaps& maps, WarpOut& o,
                                        const RowState& r, float (&v)[32], int64_t i0, int64_t j_begin, int64_t j0,
                                          int64_t j_next,
                                        int split, int lane, volatile int* gave_up) {
    // 16-bit boxes take two calls: the second fills and sends the box
    constexpr bool kTwo = sizeof(TO) == 2;
    const bool second = kTwo && ((j0 - j_begin) & 32);
    const bool send = !kTwo || second || j_next >= p.N;
    const int first = second ? 4 : 0;
    const int b = o.k % tl.ring;
    uint8_t* y = o.y + b * kBoxBytes;
    uint8_t* z = o.z + b * kBoxBytes;
    // the boxes are free once the store of `ring` boxes ago has read them; with a
    // residual that wait came before its fetch
    const bool free_now = EPI == kEpiLinear && p.residual;
    if (EPI == kEpiLinear) {
        if (p.bias) {
            o.bias[lane] = j0 + lane < p.N ? to_f32(static_cast<const T*>(p.bias)[j0 + lane]) : 0.f;
            __syncwarp();
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                const float4 f = reinterpret_cast<const float4*>(o.bias)[q];
                v[4 * q] = fmaf(v[4 * q], r.alpha, f.x);
                v[4 * q + 1] = fmaf(v[4 * q + 1], r.alpha, f.y);
                v[4 * q + 2] = fmaf(v[4 * q + 2], r.alpha, f.z);
                v[4 * q + 3] = fmaf(v[4 * q + 3], r.alpha, f.w);
            }
        } else if (r.alpha != 1.f) {
#pragma unroll
            for (int q = 0; q < 32; ++q) v[q] *= r.alpha;
        }
        if (p.targets && __any_sync(~0u, r.zero)) {
#pragma unroll
            for (int q = 0; q < 32; ++q) v[q] = r.zero ? 0.f : v[q];
        }
        if (p.preact) {
            if (tl.tma_out && !free_now && !second) boxes_free(tl, lane);
            box_write<TO>(z, lane, first, v);
        }
        activate32<TO>(v, p.act);
        if (p.residual) {
            if (tl.tma_out) {
                if (!second) {
                    if (!mbar_wait(o.bar + 8 * b, o.phase >> b & 1, gave_up)) return false;
                    o.phase ^= 1u << b;
                }
            } else {
                box_copy<TO, true>(y, first, const_cast<TO*>(static_cast<const TO*>(p.residual)), p.ldr, i0, j0, p.M, p.N, lane);
                __syncwarp();
            }
            box_add<TO>(y, lane, first, v);
        }
    }
    if (tl.tma_out && !free_now && !second && !(EPI == kEpiLinear && p.preact)) boxes_free(tl, lane);
    box_write<TO>(y, lane, first, v);
    if (tl.tma_out) {
        if (!send) return true;
        fence_async();
        __syncwarp();
        if (lane == 0) {
            if (EPI == kEpiLinear && p.preact) tma_store(&maps.z, smem_u32(z), (int)(second ? j0 - 32 : j0), (int)i0, 0, false);
            tma_store(&maps.y, smem_u32(y), (int)(second ? j0 - 32 : j0), (int)i0, split, EPI == kEpiSlab && p.accumulate);
            bulk_commit();
            if (free_now) bulk_wait_read(tl.ring - 1);
        }
    } else {
        __syncwarp();
        if (p.preact) box_copy<TO, false>(z, first, static_cast<TO*>(p.preact), p.ldz, i0, j0, p.M, p.N, lane);
        box_copy<TO, false>(y, first, static_cast<TO*>(p.out), p.ldo, i0, j0, p.M, p.N, lane);
    }
    ++o.k;
    fetch_residual(p, tl, maps, o, i0, j_next, lane);
    __syncwarp();
    return true;
}

// 32 columns from j0 of the accumulators, one row per thread; false when a wait
// gave up.
template <typename T, int EPI>
__device__ __forceinline__ bool columns32(const Product& p, const Tiles& tl, const OutMaps& maps, WarpOut& o,
                                          RowState& r, float (&v)[32], int64_t i0, int64_t j_begin, int64_t j0,
                                          int64_t j_next,
                                          int split, int lane, volatile int* gave_up) {
    if (EPI == kEpiStats) {
        const float to2 = p.logit_scale * kLog2e;
        float top = r.top;
        // rounded products here and in the gradient, never part of a fused
        // multiply-add: at large logits one bit of them is a large difference
#pragma unroll
        for (int q = 0; q < 32; ++q) v[q] = __fmul_rn(v[q], to2);
        if (j0 + 32 > p.N) {
            const int n = (int)(p.N - j0);
#pragma unroll
            for (int q = 0; q < 32; ++q) v[q] = q < n ? v[q] : -INFINITY;
        }
        float tops[4] = {top, v[1], v[2], v[3]};
#pragma unroll
        for (int q = 0; q < 32; ++q) tops[q % 4] = fmaxf(tops[q % 4], v[q]);
        top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
        const int64_t at = r.target - p.col0 - j0;
        if (__any_sync(~0u, r.in && at >= 0 && at < 32)) {
#pragma unroll
            for (int q = 0; q < 32; ++q)
                if (q == at && r.in) p.label_logit[r.i] = v[q];
        }
        const float ref = top == -INFINITY ? 0.f : top;
        float sum = r.top == -INFINITY ? r.sum : r.sum * exp2_fast(r.top - ref);  // a NaN stays
        float more[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int q = 0; q < 32; ++q) more[q % 4] += exp2_fast(v[q] - ref);
        r.top = top;
        r.sum = sum + ((more[0] + more[1]) + (more[2] + more[3]));
        return true;
    }
    if (EPI == kEpiGrad) {
        const float to2 = p.logit_scale * kLog2e;
#pragma unroll
        for (int q = 0; q < 32; ++q) {
            v[q] = exp2_fast(__fmul_rn(v[q], to2) - r.top) * r.sum;
        }
        const int64_t at = r.target - p.col0 - j0;
        if (__any_sync(~0u, at >= 0 && at < 32)) {
#pragma unroll
            for (int q = 0; q < 32; ++q)
                if (q == at) v[q] -= p.g_scale;
        }
        const bool has = r.in && r.target >= 0 && r.target < p.labels;
        if (__any_sync(~0u, !has)) {
#pragma unroll
            for (int q = 0; q < 32; ++q) v[q] = has ? v[q] : 0.f;
        }
    }
    if (EPI == kEpiSlab || (EPI == kEpiLinear && sizeof(T) == 2 && p.out_dtype == MSPLAT_DTYPE_F32))
        return write32<T, float, EPI>(p, tl, maps, o, r, v, i0, j_begin, j0, j_next, split, lane, gave_up);
    return write32<T, T, EPI>(p, tl, maps, o, r, v, i0, j_begin, j0, j_next, split, lane, gave_up);
}

template <int EPI>
__device__ __forceinline__ void row_end(const Product& p, const RowState& r, int64_t block) {
    if (EPI == kEpiStats && r.in) p.stats[block * p.stats_ld + r.i] = make_float2(r.top, r.sum);
}

// The length of the reduction that one tile makes.
inline int64_t reduction(const Product& p) { return p.epi == kEpiSlab ? std::min(p.R, p.split_len) : p.R; }
// How much of a reduction of 16-bit factors goes through the accumulators before
// their sum is added with rounding. They truncate: of sums of one sign they take
// (bf16 / f16) 1.1e-5 / 2.5e-5 after 4096 elements, 1.6e-4 / 2e-4 after 32768, 3e-3
// after 524288. A 16-bit result's half step is 3.9e-3 / 4.9e-4; 32-bit results
// and logits get the shorter pass.
inline int64_t pass_length16(const Product& p) {
    return p.epi == kEpiSlab || (p.epi == kEpiLinear && p.out_dtype == p.dtype) ? 32768 : 4096;
}

// Columns of a tile: the widest that still gives three SMs of four one, and for the
// label statistics a function of the columns alone (stats_block).
inline int tile_columns(const Product& p, int widest) {
    const int need = p.N > 128 ? 256 : p.N > 64 ? 128 : 64;
    int bn = need < widest ? need : widest;
    if (p.epi == kEpiStats) return bn;
    const int64_t tm = ceil_div(p.M, kBM) * (p.epi == kEpiSlab ? p.splits : 1);
    while (bn > 64 && tm * ceil_div(p.N, bn) < kSMs * 3 / 4) bn /= 2;
    return bn;
}

// TMA descriptors (ops_tc16.cu): a [rows, cols] matrix in boxes of 64 columns
// of 16 bits x box_rows; an output in boxes of 32 x 32, with `layers` matrices
// of rows * ld elements behind one another.
CUtensorMap map_operand(const void* base, int64_t rows, int64_t cols, int64_t ld, int box_rows, int dtype);
CUtensorMap map_output(const void* base, int64_t rows, int64_t cols, int64_t ld, int64_t layers, int dtype);
bool tma_ready(const void* p, int64_t ld, int64_t rows, int elem);

// Boxes of the outputs and, when TMA can move them, their descriptors.
inline void set_outputs(const Product& p, Tiles& tl, OutMaps& maps) {
    if (p.epi == kEpiStats) return;
    const int dtype = p.epi == kEpiSlab ? MSPLAT_DTYPE_F32 : p.out_dtype, es = dtype_size(dtype);
    tl.tma_out = 1;
    if (p.epi == kEpiSlab) {
        maps.y = map_output(p.slab, p.M, p.N, slab_ld(p.N), p.splits, dtype);
        return;
    }
    tl.tma_out = tma_ready(p.out, p.ldo, p.M, es) && (!p.preact || tma_ready(p.preact, p.ldz, p.M, es)) &&
                 (!p.residual || tma_ready(p.residual, p.ldr, p.M, es));
    if (!tl.tma_out) return;
    maps.y = map_output(p.out, p.M, p.N, p.ldo, 1, dtype);
    if (p.preact) maps.z = map_output(p.preact, p.M, p.N, p.ldz, 1, dtype);
    if (p.residual) maps.r = map_output(p.residual, p.M, p.N, p.ldr, 1, dtype);
}

// Shares the block's memory between the stages and `warps` warps' boxes: two
// boxes per output where that leaves least_stages. Returns the dynamic bytes.
inline int share_memory(const Product& p, Tiles& tl, int warps, int fixed, int least_stages, int most_stages) {
    const int outputs = p.epi == kEpiStats ? 0 : 1 + (p.epi == kEpiLinear && p.preact);
    for (tl.ring = 2;; --tl.ring) {
        tl.warp_bytes = tl.ring * outputs * kBoxBytes;
        const int rest = kBlockBytes - fixed - warps * tl.warp_bytes;
        tl.stages = rest > 0 ? std::min(most_stages, rest / tl.stage_bytes) : 0;
        if ((rest > 0 && tl.stages >= least_stages) || tl.ring == 1) break;
    }
    return 1024 + fixed + tl.stages * tl.stage_bytes + warps * tl.warp_bytes;
}

// Column blocks of the label statistics: tiles of 64 columns, halves of wider ones.
inline int64_t stats_blocks_of(const Product& p, int bn) { return ceil_div(p.N, bn) * (bn == 64 ? 1 : 2); }

inline void set_tiles(const Product& p, Tiles& tl) {
    const int64_t tm = ceil_div(p.M, kBM), tn = ceil_div(p.N, tl.bn);
    const int64_t total = tm * tn * (p.epi == kEpiSlab ? p.splits : 1);
    if (total > 0x3fffffff) throw Error(MSPLAT_ERR_CAPACITY, "too many tiles");
    tl.tiles_m = (int)tm;
    tl.tiles_n = (int)tn;
    tl.total = (int)total;
}

}  // namespace ops
}  // namespace msplat
