// ops_reduce.cu — the elementwise and reducing passes around the products:
// dz with its column sums, sums of partial products, and the join of the
// softmax statistics. All are bound by the bytes they read and write; every
// sum has a fixed order.
#include "ops.cuh"

namespace msplat {
namespace ops {
namespace {

// A block takes a piece of the rows and 32 columns; eight warps walk the rows.
template <typename T, int ACT>
__global__ void __launch_bounds__(256) k_dz(int64_t m, int64_t n, const T* z, int64_t ldz, const T* dy,
                                            int64_t lddy, T* dz, int64_t lddz, float* partial, int64_t piece_rows) {
    __shared__ float sums[8][33];
    const int64_t j = blockIdx.x * 32 + threadIdx.x;
    const int64_t i0 = blockIdx.y * piece_rows, i1 = min(m, i0 + piece_rows);
    float sum = 0.f;
    if (j < n)
        for (int64_t i = i0 + threadIdx.y; i < i1; i += 8) {
            float v = to_f32(dy[i * lddy + j]);
            if (ACT != MSPLAT_ACT_NONE) v *= act_slope<ACT>(to_f32(z[i * ldz + j]));
            if (dz) dz[i * lddz + j] = from_f32<T>(v);
            sum += v;
        }
    sums[threadIdx.y][threadIdx.x] = sum;
    __syncthreads();
    if (partial && threadIdx.y == 0 && j < n) {
        float t = 0.f;
        for (int q = 0; q < 8; ++q) t += sums[q][threadIdx.x];
        partial[(int64_t)blockIdx.y * n + j] = t;
    }
}

template <typename T>
__global__ void __launch_bounds__(256) k_slab_sum(int64_t rows, int64_t cols, const float* slab, int64_t ld, int pieces, T* out,
                                                  int64_t ldo, float alpha, const float* alpha_dev,
                                                  const int32_t* targets, int64_t labels) {
    const int64_t n = rows * cols;
    const float a = alpha * (alpha_dev ? *alpha_dev : 1.f);
    for (int64_t e = blockIdx.x * 256ll + threadIdx.x; e < n; e += gridDim.x * 256ll) {
        float t = 0.f;
        const int64_t i = e / cols;
        const float* at = slab + i * ld + (e - i * cols);
        for (int q = 0; q < pieces; ++q) t += at[q * rows * ld];
        t *= a;
        if (targets && !(targets[i] >= 0 && targets[i] < labels)) t = 0.f;
        out[i * ldo + (e - i * cols)] = from_f32<T>(t);
    }
}

__global__ void __launch_bounds__(256) k_join(JoinArgs a) {
    __shared__ double ssum[256], scount[256];
    double sum = 0, count = 0;
    for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < a.m; i += gridDim.x * 256ll) {
        // a block whose sum is 0 (columns beyond the last, or logits of -inf
        // only) has no reference; a sum of NaN counts
        float top = -INFINITY;
        for (int64_t b = 0; b < a.blocks; ++b) {
            const float2 v = a.stats[b * a.stats_ld + i];
            if (v.y != 0.f) top = fmaxf(top, v.x);
        }
        float total = 0.f;
        for (int64_t b = 0; b < a.blocks; ++b) {
            const float2 v = a.stats[b * a.stats_ld + i];
            if (v.y != 0.f) total += v.y * exp2f(v.x - top);
        }
        const float lse = top + log2f(total);
        const int32_t t = a.targets[i];
        const bool has = t >= 0 && t < a.labels;
        const float row = has ? (lse - a.label_logit[i]) * kLn2 : 0.f;
        a.lse[i] = lse;
        if (a.row_loss) a.row_loss[i] = row;
        if (has) {
            sum += row;
            count += 1;
        }
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
        a.partial[2 * blockIdx.x] = ssum[0];
        a.partial[2 * blockIdx.x + 1] = scount[0];
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
        *alpha = any ? (float)(factor / scount[0]) : 0.f;
    }
}

template <typename T>
void dz_typed(int64_t m, int64_t n, const void* z, int64_t ldz, int act, const void* dy, int64_t lddy, void* dz,
              int64_t lddz, float* partial, cudaStream_t s) {
    const int pieces = dz_pieces(m, n);
    const dim3 grid((unsigned)ceil_div(n, 32), pieces);
    note_launches(1);
    auto go = [&](auto kernel) {
        kernel<<<grid, dim3(32, 8), 0, s>>>(m, n, static_cast<const T*>(z), ldz, static_cast<const T*>(dy), lddy,
                                            static_cast<T*>(dz), lddz, partial, ceil_div(m, pieces));
    };
    switch (act) {
        case MSPLAT_ACT_RELU: go(k_dz<T, MSPLAT_ACT_RELU>); break;
        case MSPLAT_ACT_GELU: go(k_dz<T, MSPLAT_ACT_GELU>); break;
        case MSPLAT_ACT_SILU: go(k_dz<T, MSPLAT_ACT_SILU>); break;
        case MSPLAT_ACT_SIGMOID: go(k_dz<T, MSPLAT_ACT_SIGMOID>); break;
        default: go(k_dz<T, MSPLAT_ACT_NONE>); break;
    }
    OPS_CK(cudaGetLastError());
}

}  // namespace

int dz_pieces(int64_t m, int64_t n) {
    // about eight blocks per SM, at least 64 rows each
    const int64_t want = ceil_div(kSMs * 8, ceil_div(n, 32));
    const int64_t most = ceil_div(m, 64);
    return (int)(want < most ? want : most);
}

void launch_dz(int64_t m, int64_t n, const void* z, int64_t ldz, int act, const void* dy, int64_t lddy, void* dz,
               int64_t lddz, float* partial, int dtype, cudaStream_t s) {
    if (dtype == MSPLAT_DTYPE_F32)
        dz_typed<float>(m, n, z, ldz, act, dy, lddy, dz, lddz, partial, s);
    else if (dtype == MSPLAT_DTYPE_F16)
        dz_typed<__half>(m, n, z, ldz, act, dy, lddy, dz, lddz, partial, s);
    else
        dz_typed<__nv_bfloat16>(m, n, z, ldz, act, dy, lddy, dz, lddz, partial, s);
}

void launch_slab_sum(int64_t rows, int64_t cols, const float* slab, int64_t ld, int pieces, void* out, int64_t ldo, float alpha,
                     const float* alpha_dev, const int32_t* targets, int64_t labels, int dtype, cudaStream_t s) {
    const int64_t ctas = ceil_div(rows * cols, 256);
    const unsigned grid = (unsigned)(ctas < kSMs * 8 ? ctas : kSMs * 8);
    note_launches(1);
    if (dtype == MSPLAT_DTYPE_F32)
        k_slab_sum<float><<<grid, 256, 0, s>>>(rows, cols, slab, ld, pieces, static_cast<float*>(out), ldo, alpha,
                                               alpha_dev, targets, labels);
    else if (dtype == MSPLAT_DTYPE_F16)
        k_slab_sum<__half><<<grid, 256, 0, s>>>(rows, cols, slab, ld, pieces, static_cast<__half*>(out), ldo, alpha,
                                                alpha_dev, targets, labels);
    else
        k_slab_sum<__nv_bfloat16><<<grid, 256, 0, s>>>(rows, cols, slab, ld, pieces, static_cast<__nv_bfloat16*>(out),
                                                       ldo, alpha, alpha_dev, targets, labels);
    OPS_CK(cudaGetLastError());
}

int join_blocks(int64_t m) {
    const int64_t b = ceil_div(m, 256);
    return (int)(b < kSMs * 4 ? b : kSMs * 4);
}

void launch_join(const JoinArgs& a, cudaStream_t s) {
    note_launches(1);
    k_join<<<join_blocks(a.m), 256, 0, s>>>(a);
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
