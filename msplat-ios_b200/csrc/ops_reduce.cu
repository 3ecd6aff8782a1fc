// ops_reduce.cu — the elementwise and reducing passes around the products:
// dz with its column sums, sums of partial products, and the join of the
// softmax statistics. All are bound by the bytes they read and write (dz of
// 65536 x 1024 bf16 with GELU: 402 MB in 88 us, 4.6 TB/s); every sum has a fixed
// order.
#include "ops.cuh"

namespace msplat {
namespace ops {
namespace {

// dz of 16-bit types is rounded to the type, since it is a factor of two products
// on the tensor cores: in two parts they would be twice as long (110 and 98 us for
// the wide case below). Its rounding, independent from element to element, adds to
// the output's: 0.0024 of the norm of dx and dw in bf16 where rounding the output
// alone is 0.0017. The column sums add dz before it is rounded.
//
// A block takes a piece of the rows and up to 32 vectors of V columns (16 bytes
// when the matrices are aligned, else one element); `lanes` threads (a power of
// two) share a row. Bound by reading z and dy and writing dz: each thread has
// two rows of both in flight.
template <typename T, int ACT, int V>
__global__ void __launch_bounds__(256) k_dz(int64_t m, int64_t n, const T* z, int64_t ldz, const T* dy,
                                            int64_t lddy, T* dz, int64_t lddz, float* partial, int64_t piece_rows,
                                            int lanes) {
    __shared__ float sums[256 * V];
    const int cx = threadIdx.x % lanes, ry = threadIdx.x / lanes, rows = 256 / lanes;
    const int64_t j = ((int64_t)blockIdx.x * lanes + cx) * V;
    const int64_t i0 = blockIdx.y * piece_rows, i1 = min(m, i0 + piece_rows);
    union Vec {
        T t[V];
        uint4 w;
        __device__ Vec() {}
    };
    float sum[V];
#pragma unroll
    for (int q = 0; q < V; ++q) sum[q] = 0.f;
    // the last vector of an aligned row may end behind the row's last column
    const int count = V == 1 ? 1 : (int)min((int64_t)V, n - j);
    auto get = [&](Vec& v, const T* g) {
        if (V > 1 && count == V) {
            v.w = __ldg(reinterpret_cast<const uint4*>(g));
        } else {
#pragma unroll
            for (int q = 0; q < V; ++q) v.t[q] = q < count ? g[q] : from_f32<T>(0.f);
        }
    };
    auto one = [&](const Vec& a, const Vec& b, int64_t i) {
        Vec o;
#pragma unroll
        for (int q = 0; q < V; q += 2) {
            constexpr int kNext = V > 1 ? 1 : 0;  // (one element is taken twice)
            float2 v = make_float2(to_f32(a.t[q]), to_f32(a.t[q + kNext]));
            if (ACT != MSPLAT_ACT_NONE)
                v = __fmul2_rn(v, act_slope<ACT, T>(make_float2(to_f32(b.t[q]), to_f32(b.t[q + kNext]))));
            o.t[q] = from_f32<T>(v.x);
            sum[q] += v.x;
            if (V > 1) {
                o.t[q + kNext] = from_f32<T>(v.y);
                sum[q + kNext] += v.y;
            }
        }
        if (!dz) return;
        T* g = dz + i * lddz + j;
        if (V > 1 && count == V) {
            *reinterpret_cast<uint4*>(g) = o.w;
        } else {
#pragma unroll
            for (int q = 0; q < V; ++q)
                if (q < count) g[q] = o.t[q];
        }
    };
    if (j < n) {
        int64_t i = i0 + ry;
        for (; i + rows < i1; i += 2 * rows) {
            Vec a0, a1, b0, b1;
            get(a0, dy + i * lddy + j);
            get(a1, dy + (i + rows) * lddy + j);
            if (ACT != MSPLAT_ACT_NONE) {
                get(b0, z + i * ldz + j);
                get(b1, z + (i + rows) * ldz + j);
            }
            one(a0, b0, i);
            one(a1, b1, i + rows);
        }
        if (i < i1) {
            Vec a0, b0;
            get(a0, dy + i * lddy + j);
            if (ACT != MSPLAT_ACT_NONE) get(b0, z + i * ldz + j);
            one(a0, b0, i);
        }
    }
    if (!partial) return;
#pragma unroll
    for (int q = 0; q < V; ++q) sums[(ry * lanes + cx) * V + q] = sum[q];
    __syncthreads();
    for (int c = threadIdx.x; c < lanes * V; c += 256) {
        const int64_t col = (int64_t)blockIdx.x * lanes * V + c;
        if (col >= n) break;
        float t = 0.f;
        for (int q = 0; q < rows; ++q) t += sums[q * lanes * V + c];
        partial[(int64_t)blockIdx.y * n + col] = t;
    }
}

// Threads of a block: `across` consecutive elements (a power of two) x 256 /
// across shares of the pieces, whose sums are joined through shared memory. Few
// elements with many pieces (the column sums, a small dw) thus have as many
// reads in flight as many elements with few.
template <typename T>
__global__ void __launch_bounds__(256) k_slab_sum(int64_t rows, int64_t cols, const float* slab, int64_t ld, int pieces,
                                                  T* out, int64_t ldo, float alpha, const float* alpha_dev,
                                                  const int32_t* targets, int64_t labels, int across) {
    __shared__ float sums[256];
    const int64_t n = rows * cols, layer = rows * ld;
    const float a = alpha * (alpha_dev ? *alpha_dev : 1.f);
    const int ex = threadIdx.x % across, share = threadIdx.x / across, shares = 256 / across;
    for (int64_t e0 = (int64_t)blockIdx.x * across; e0 < n; e0 += (int64_t)gridDim.x * across) {
        const int64_t e = e0 + ex, i = e < n ? e / cols : 0, j = e < n ? e - i * cols : 0;
        const float* at = slab + i * ld + j;
        float t = 0.f;
        if (e < n) {
            int q = share;
            for (; q + 3 * shares < pieces; q += 4 * shares) {
                const float v0 = __ldcs(at + q * layer), v1 = __ldcs(at + (q + shares) * layer),
                            v2 = __ldcs(at + (q + 2 * shares) * layer), v3 = __ldcs(at + (q + 3 * shares) * layer);
                t += (v0 + v1) + (v2 + v3);
            }
            for (; q < pieces; q += shares) t += __ldcs(at + q * layer);
        }
        if (shares > 1) {
            sums[threadIdx.x] = t;
            __syncthreads();
            if (share == 0)
                for (int q = 1; q < shares; ++q) t += sums[q * across + ex];
            __syncthreads();
        }
        if (share == 0 && e < n) {
            t *= a;
            if (targets && !(targets[i] >= 0 && targets[i] < labels)) t = 0.f;
            out[i * ldo + j] = from_f32<T>(t);
        }
    }
}

// Each warp takes 32 rows (its lanes) and one share of the column blocks;
// `shares` warps (a power of two) join theirs through shared memory.
__global__ void __launch_bounds__(1024) k_join(JoinArgs a, int shares) {
    __shared__ float tops[32][33], sums[32][33];
    const int lane = threadIdx.x, warp = threadIdx.y, share = warp % shares;
    const int64_t rows = 32 * (32 / shares);
    double sum = 0, count = 0;
    for (int64_t g0 = blockIdx.x * rows; g0 < a.m; g0 += gridDim.x * rows) {
        const int64_t i0 = g0 + warp / shares * 32, i = i0 + lane;
        // a block whose sum is 0 (columns beyond the last, or logits of -inf
        // only) has no reference; a sum of NaN counts
        float top = -INFINITY, total = 0.f;
        if (i < a.m)
            for (int64_t b = share; b < a.blocks; b += 8 * shares) {
                float2 v[8];  // eight reads in flight
#pragma unroll
                for (int q = 0; q < 8; ++q)
                    v[q] = b + q * shares < a.blocks ? __ldcs(a.stats + (b + q * shares) * a.stats_ld + i)
                                                     : make_float2(0.f, 0.f);
                float t = top;
#pragma unroll
                for (int q = 0; q < 8; ++q)
                    if (v[q].y != 0.f) t = fmaxf(t, v[q].x);
                total = total == 0.f ? 0.f : total * exp2f(top - t);
#pragma unroll
                for (int q = 0; q < 8; ++q)
                    if (v[q].y != 0.f) total += v[q].y * exp2f(v[q].x - t);
                top = t;
            }
        tops[warp][lane] = top;
        sums[warp][lane] = total;
        if (shares > 1) __syncthreads();
        if (share == 0) {
            for (int q = warp + 1; q < warp + shares; ++q) {
                const float t = fmaxf(top, tops[q][lane]);
                if (sums[q][lane] == 0.f) continue;
                total = (total == 0.f ? 0.f : total * exp2f(top - t)) + sums[q][lane] * exp2f(tops[q][lane] - t);
                top = t;
            }
            const int32_t t = i < a.m ? a.targets[i] : -1;
            const bool has = t >= 0 && t < a.labels;
            if (i < a.m) {
                const float row = has ? ((top - a.label_logit[i]) + log2f(total)) * kLn2 : 0.f;
                a.norm[i] = make_float2(top, 1.f / total);
                if (a.row_loss) a.row_loss[i] = row;
                if (has) {
                    sum += row;
                    count += 1;
                }
            }
        }
        if (shares > 1) __syncthreads();
    }
    __shared__ double ssum[32], scount[32];
    for (int o = 16; o; o >>= 1) {
        sum += __shfl_xor_sync(~0u, sum, o);
        count += __shfl_xor_sync(~0u, count, o);
    }
    if (lane == 0) {
        ssum[warp] = sum;
        scount[warp] = count;
    }
    __syncthreads();
    if (warp == 0 && lane == 0) {
        for (int q = 1; q < 32; ++q) {
            sum += ssum[q];
            count += scount[q];
        }
        a.partial[2 * blockIdx.x] = sum;
        a.partial[2 * blockIdx.x + 1] = count;
    }
}

__global__ void __launch_bounds__(256) k_count_labels(int64_t m, const int32_t* targets, int64_t labels,
                                                      double* partial) {
    int n = 0;
    for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < m; i += gridDim.x * 256ll) {
        const int32_t t = targets[i];
        n += t >= 0 && t < labels;
    }
    __shared__ int warps[8];
    n = __reduce_add_sync(~0u, n);
    if (threadIdx.x % 32 == 0) warps[threadIdx.x / 32] = n;
    __syncthreads();
    if (threadIdx.x == 0) {
        double t = 0;
        for (int q = 0; q < 8; ++q) t += warps[q];
        partial[2 * blockIdx.x] = 0;
        partial[2 * blockIdx.x + 1] = t;
    }
}

__global__ void __launch_bounds__(256) k_loss_total(const double* partial, int blocks, float weight, float factor,
                                                    float* loss, float* alpha) {
    __shared__ double ssum[256], scount[256];
    double sum = 0, count = 0;
    for (int b = threadIdx.x; b < blocks; b += 256) {
        sum += partial[2 * b];
        count += partial[2 * b + 1];
    }
    ssum[threadIdx.x] = sum;
    scount[threadIdx.x] = count;
    for (int o = 128; o; o >>= 1) {
        __syncthreads();
        if (threadIdx.x < o) {
            ssum[threadIdx.x] += ssum[threadIdx.x + o];
            scount[threadIdx.x] += scount[threadIdx.x + o];
        }
    }
    if (threadIdx.x == 0) {
        const bool any = scount[0] > 0;
        if (loss) *loss = any ? (float)(weight * ssum[0] / scount[0]) : 0.f;
        if (alpha) *alpha = any ? (float)(factor / scount[0]) : 0.f;
    }
}

// `lanes` threads (a power of two) share a row, in vectors of V elements.
template <typename T, int V>
__global__ void __launch_bounds__(256) k_labelled_rows(int64_t m, int64_t d, const T* x, int64_t ldx,
                                                       const int32_t* targets, int64_t labels, T* out, int64_t ldo,
                                                       int lanes) {
    const int rows = 256 / lanes;
    for (int64_t i = blockIdx.x * (int64_t)rows + threadIdx.x / lanes; i < m; i += gridDim.x * (int64_t)rows) {
        bool has = true;
        if (targets) {
            const int32_t t = __ldg(targets + i);
            has = t >= 0 && t < labels;
        }
        const T* from = x + i * ldx;
        T* to = out + i * ldo;
#pragma unroll 4
        for (int64_t j = threadIdx.x % lanes * V; j < d; j += lanes * V) {
            if (V > 1)
                *reinterpret_cast<uint4*>(to + j) =
                    has ? __ldg(reinterpret_cast<const uint4*>(from + j)) : make_uint4(0, 0, 0, 0);
            else
                to[j] = has ? from[j] : from_f32<T>(0.f);
        }
    }
}

template <typename T>
void labelled_typed(int64_t m, int64_t d, const void* x, int64_t ldx, const int32_t* targets, int64_t labels, void* out,
                    int64_t ldo, cudaStream_t s) {
    constexpr int V = 16 / sizeof(T);
    const bool vec = reinterpret_cast<uintptr_t>(x) % 16 == 0 && (m <= 1 || ldx % V == 0) && d % V == 0;
    int lanes = 1;
    while (lanes < 32 && lanes * (vec ? V : 1) < d) lanes *= 2;
    const unsigned grid = (unsigned)std::min<int64_t>(ceil_div(m * lanes, 256), kSMs * 16);
    note_launches(1);
    if (vec)
        k_labelled_rows<T, V><<<grid, 256, 0, s>>>(m, d, static_cast<const T*>(x), ldx, targets, labels,
                                                   static_cast<T*>(out), ldo, lanes);
    else
        k_labelled_rows<T, 1><<<grid, 256, 0, s>>>(m, d, static_cast<const T*>(x), ldx, targets, labels,
                                                   static_cast<T*>(out), ldo, lanes);
    OPS_CK(cudaGetLastError());
}

template <typename T, int V>
void dz_typed(int64_t m, int64_t n, const void* z, int64_t ldz, int act, const void* dy, int64_t lddy, void* dz,
              int64_t lddz, float* partial, cudaStream_t s) {
    const int pieces = dz_pieces(m, n);
    int lanes = 1;
    while (lanes < 32 && lanes * V < n) lanes *= 2;
    const dim3 grid((unsigned)ceil_div(n, (int64_t)lanes * V), pieces);
    note_launches(1);
    auto go = [&](auto kernel) {
        kernel<<<grid, 256, 0, s>>>(m, n, static_cast<const T*>(z), ldz, static_cast<const T*>(dy), lddy,
                                    static_cast<T*>(dz), lddz, partial, ceil_div(m, pieces), lanes);
    };
    switch (act) {
        case MSPLAT_ACT_RELU: go(k_dz<T, MSPLAT_ACT_RELU, V>); break;
        case MSPLAT_ACT_GELU: go(k_dz<T, MSPLAT_ACT_GELU, V>); break;
        case MSPLAT_ACT_SILU: go(k_dz<T, MSPLAT_ACT_SILU, V>); break;
        case MSPLAT_ACT_SIGMOID: go(k_dz<T, MSPLAT_ACT_SIGMOID, V>); break;
        default: go(k_dz<T, MSPLAT_ACT_NONE, V>); break;
    }
    OPS_CK(cudaGetLastError());
}

template <typename T>
void dz_any(int64_t m, int64_t n, const void* z, int64_t ldz, int act, const void* dy, int64_t lddy, void* dz,
            int64_t lddz, float* partial, cudaStream_t s) {
    constexpr int V = 16 / sizeof(T);
    auto ready = [&](const void* p, int64_t ld) {
        return !p || (reinterpret_cast<uintptr_t>(p) % 16 == 0 && (m <= 1 || ld % V == 0));
    };
    if (n >= V && ready(dy, lddy) && ready(dz, lddz) && (act == MSPLAT_ACT_NONE || ready(z, ldz)))
        dz_typed<T, V>(m, n, z, ldz, act, dy, lddy, dz, lddz, partial, s);
    else
        dz_typed<T, 1>(m, n, z, ldz, act, dy, lddy, dz, lddz, partial, s);
}

}  // namespace

int dz_pieces(int64_t m, int64_t n) {
    // about eight blocks per SM (of 128 to 256 columns), at least 64 rows each
    const int64_t want = ceil_div(kSMs * 8, ceil_div(n, 256));
    const int64_t most = ceil_div(m, 64);
    return (int)(want < most ? want : most);
}

void launch_dz(int64_t m, int64_t n, const void* z, int64_t ldz, int act, const void* dy, int64_t lddy, void* dz,
               int64_t lddz, float* partial, int dtype, cudaStream_t s) {
    if (dtype == MSPLAT_DTYPE_F32)
        dz_any<float>(m, n, z, ldz, act, dy, lddy, dz, lddz, partial, s);
    else if (dtype == MSPLAT_DTYPE_F16)
        dz_any<__half>(m, n, z, ldz, act, dy, lddy, dz, lddz, partial, s);
    else
        dz_any<__nv_bfloat16>(m, n, z, ldz, act, dy, lddy, dz, lddz, partial, s);
}

void launch_slab_sum(int64_t rows, int64_t cols, const float* slab, int64_t ld, int pieces, void* out, int64_t ldo, float alpha,
                     const float* alpha_dev, const int32_t* targets, int64_t labels, int dtype, cudaStream_t s) {
    // shares of at least four pieces, as long as the blocks do not fill the SMs
    int across = 256;
    while (across > 8 && ceil_div(rows * cols, across) < kSMs * 8 && 256 / across * 4 < pieces) across /= 2;
    const int64_t ctas = ceil_div(rows * cols, across);
    const unsigned grid = (unsigned)(ctas < kSMs * 8 ? ctas : kSMs * 8);
    note_launches(1);
    auto go = [&](auto* o) {
        k_slab_sum<<<grid, 256, 0, s>>>(rows, cols, slab, ld, pieces, o, ldo, alpha, alpha_dev, targets, labels, across);
    };
    if (dtype == MSPLAT_DTYPE_F32)
        go(static_cast<float*>(out));
    else if (dtype == MSPLAT_DTYPE_F16)
        go(static_cast<__half*>(out));
    else
        go(static_cast<__nv_bfloat16*>(out));
    OPS_CK(cudaGetLastError());
}

void launch_labelled_rows(int64_t m, int64_t d, const void* x, int64_t ldx, const int32_t* targets, int64_t labels,
                          void* out, int64_t ldo, int dtype, cudaStream_t s) {
    if (dtype == MSPLAT_DTYPE_F32)
        labelled_typed<float>(m, d, x, ldx, targets, labels, out, ldo, s);
    else if (dtype == MSPLAT_DTYPE_F16)
        labelled_typed<__half>(m, d, x, ldx, targets, labels, out, ldo, s);
    else
        labelled_typed<__nv_bfloat16>(m, d, x, ldx, targets, labels, out, ldo, s);
}

int join_blocks(int64_t m) {
    const int64_t b = ceil_div(m, 32);
    return (int)(b < kSMs * 2 ? b : kSMs * 2);
}

void launch_join(const JoinArgs& a, cudaStream_t s) {
    note_launches(1);
    int shares = 1;
    while (shares < 32 && shares < a.blocks) shares *= 2;
    k_join<<<join_blocks(a.m), dim3(32, 32), 0, s>>>(a, shares);
    OPS_CK(cudaGetLastError());
}

void launch_count_labels(int64_t m, const int32_t* targets, int64_t labels, double* partial, int blocks,
                         cudaStream_t s) {
    note_launches(1);
    k_count_labels<<<blocks, 256, 0, s>>>(m, targets, labels, partial);
    OPS_CK(cudaGetLastError());
}

void launch_loss_total(const double* partial, int blocks, float weight, float factor, float* loss, float* alpha,
                       cudaStream_t s) {
    note_launches(1);
    k_loss_total<<<1, 256, 0, s>>>(partial, blocks, weight, factor, loss, alpha);
    OPS_CK(cudaGetLastError());
}

}  // namespace ops
}  // namespace msplat
