// ops_api.cu — the entry points of include/msplat_ops.h: checks, the layout of
// the caller's workspace, and the order of the launches.
#include <algorithm>
#include <array>
#include <cmath>
#include <map>
#include <mutex>
#include <utility>

#include "ops.cuh"

namespace msplat {
namespace ops {
namespace {

template <typename F>
int guarded(F&& f) {
    try {
        f();
        set_last_error("");
        return MSPLAT_OK;
    } catch (const Error& e) {
        set_last_error(e.what());
        return e.code;
    } catch (const std::exception& e) {
        set_last_error(e.what());
        return MSPLAT_ERR_CUDA;
    }
}

void require(bool ok, const char* what) {
    if (!ok) throw Error(MSPLAT_ERR_ARGUMENT, what);
}

void check_size(int64_t v, int64_t least, const char* name) {
    // tile and element coordinates stay below 2^31 with a tile's overhang
    if (v < least || v > (1 << 30))
        throw Error(MSPLAT_ERR_ARGUMENT, std::string(name) + " must be in [" + std::to_string(least) + ", 2^30]");
}

void check_dtype(int dtype) {
    require(dtype == MSPLAT_DTYPE_F32 || dtype == MSPLAT_DTYPE_F16 || dtype == MSPLAT_DTYPE_BF16,
            "dtype must be MSPLAT_DTYPE_F32, _F16 or _BF16");
}

void check_matrix(const void* p, int64_t rows, int64_t cols, int64_t ld, int elem, const char* name) {
    if (rows == 0) return;
    if (!p) throw Error(MSPLAT_ERR_ARGUMENT, std::string(name) + " is null");
    if (ld < cols) throw Error(MSPLAT_ERR_ARGUMENT, std::string(name) + ": the row stride is below the columns");
    if (ld > INT64_MAX / 8 / rows) throw Error(MSPLAT_ERR_ARGUMENT, std::string(name) + ": the row stride is too large");
    if (reinterpret_cast<uintptr_t>(p) % elem)
        throw Error(MSPLAT_ERR_ARGUMENT, std::string(name) + " is not aligned to its element type");
}

// Lays buffers out in the caller's workspace; without a base it only counts.
struct Arena {
    char* base;
    uint64_t used = 0;
    explicit Arena(void* p) : base(static_cast<char*>(p)) {}
    template <typename T>
    T* take(int64_t count) {
        const uint64_t at = used;
        used += (uint64_t)round_up(count * (int64_t)sizeof(T), 256);
        return base ? reinterpret_cast<T*>(base + at) : nullptr;
    }
};

void check_workspace(const Arena& a, void* workspace, uint64_t bytes) {
    if (a.used == 0) return;
    require(workspace, "workspace is null");
    require(reinterpret_cast<uintptr_t>(workspace) % 256 == 0, "workspace is not aligned to 256 bytes");
    require(bytes >= a.used, "workspace is too small");
}

// Pieces of a long reduction of an M x N result: enough tiles for every SM, in
// pieces of at least 512. The tensor cores truncate when they add, so the pieces,
// whose sums are added with rounding, are no longer than a type's rounding asks
// for as long as they take no more than kSlabBytes: 1024 for 32 bits, 32768 for 16
// (and four times the bytes, since such a piece has so much more to do), whose
// one-signed sums are then off by 2e-4, less than half of half a step of f16.
constexpr int64_t kSlabBytes = 256ll << 20;
struct Split {
    int splits;
    int64_t len;
};
Split plan_split(int64_t M, int64_t N, int64_t R, int dtype) {
    // the share of the SMs' rounds that has work, with as few pieces as come
    // within a twentieth of the best
    const bool exact = dtype == MSPLAT_DTYPE_F32;
    const int64_t tiles = ceil_div(M, 128) * ceil_div(N, exact ? 128 : N > 128 ? 256 : N > 64 ? 128 : 64);
    const int64_t most = std::min<int64_t>(ceil_div(R, 512), std::max<int64_t>(1, 2 * kSMs / tiles));
    int64_t s = 1;
    double best = 0;
    for (int64_t q = 1; q <= most; ++q) {
        const double used = (double)(tiles * q) / (double)(ceil_div(tiles * q, kSMs) * kSMs);
        if (used > best + 0.05) {
            best = used;
            s = q;
        }
    }
    const int64_t room = (exact ? kSlabBytes : 4 * kSlabBytes) / (M * N * 4);
    s = std::max(s, std::min(ceil_div(R, exact ? 1024 : 32768), std::max<int64_t>(1, room)));
    const int64_t len = round_up(ceil_div(R, s), 64);
    return {(int)ceil_div(R, len), len};
}

// ---- linear -----------------------------------------------------------------

void check_act(int act) {
    require(act >= MSPLAT_ACT_NONE && act <= MSPLAT_ACT_SIGMOID, "unknown activation");
}

struct BackwardPlan {
    Split split;
    void* dz = nullptr;
    int64_t lddz = 0;
    float* slab = nullptr;
    float* sums = nullptr;
    int pieces = 0;
    bool rows = false;  // in one pass over the rows
    BackwardPlan(Arena& a, int64_t m, int64_t n, int64_t k, int act, int dtype) {
        rows = fits_rows(m, n, k);
        if (rows) {
            pieces = rows_blocks(m);
            slab = a.take<float>((int64_t)pieces * n * slab_ld(k));
            sums = a.take<float>((int64_t)pieces * n);
            return;
        }
        split = plan_split(n, k, m, dtype);
        pieces = dz_pieces(m, n);
        lddz = round_up(n, 16 / dtype_size(dtype));
        if (act != MSPLAT_ACT_NONE) dz = a.take<char>(m * lddz * dtype_size(dtype));
        slab = a.take<float>((int64_t)split.splits * n * slab_ld(k));
        sums = a.take<float>((int64_t)pieces * n);
    }
};

void check_backward(int64_t m, int64_t n, int64_t k, int act, int dtype) {
    check_size(m, 0, "m");
    check_size(n, 1, "n");
    check_size(k, 1, "k");
    check_act(act);
    check_dtype(dtype);
}

// ---- label loss -------------------------------------------------------------

constexpr int64_t kStatsBytes = 64ll << 20;   // statistics of the column blocks kept at a time
constexpr int64_t kPieceBytes = 256ll << 20;  // softmax gradients kept at a time

struct LossPlan {
    int64_t blocks, stats_rows;        // column blocks; rows per statistics pass
    bool by_rows;                      // gradient pieces are rows of the table's full width, else columns
    int64_t chunk, ldg;
    Split sx, sw;                      // reductions of dx (over labels) and dw (over rows)
    float *label_logit, *alpha;
    float2* norm;
    double* partial;
    float2* stats;
    // x's labelled rows and, when rows of d 16-bit elements are no multiple of 16
    // bytes, w, with rows of ldx elements; a piece of the softmax gradient
    char *x = nullptr, *w = nullptr, *g = nullptr;
    int64_t ldx;
    float *slab_x = nullptr, *slab_w = nullptr;
    bool rows;                         // in one pass over the rows
    LossPlan(Arena& a, int64_t m, int64_t v, int64_t d, bool grad, int dtype) {
        rows = fits_rows(m, v, d);
        if (rows) {
            alpha = a.take<float>(1);
            partial = a.take<double>(2 * rows_blocks(m));
            slab_w = a.take<float>((int64_t)rows_blocks(m) * v * slab_ld(d));
            return;
        }
        blocks = stats_blocks_most(v);
        stats_rows = round_up(std::max<int64_t>(kStatsBytes / (8 * blocks), 1), 256);
        if (stats_rows > m) stats_rows = m;
        alpha = a.take<float>(1);
        norm = a.take<float2>(m);
        label_logit = a.take<float>(m);
        partial = a.take<double>(2 * ceil_div(m, stats_rows) * join_blocks(stats_rows));
        stats = a.take<float2>(blocks * stats_rows);
        const int es = dtype_size(dtype);
        ldx = round_up(d, 16 / es);
        const bool odd = es == 2 && ldx != d;
        if (grad || odd) x = a.take<char>(m * ldx * es);
        if (odd) w = a.take<char>(v * ldx * es);
        if (!grad) return;
        by_rows = m >= v;
        const int64_t other = round_up(by_rows ? v : m, 16 / es), all = by_rows ? m : v;
        chunk = std::min(all, round_up(std::max<int64_t>(kPieceBytes / (other * es), 1), 128));
        ldg = by_rows ? other : round_up(chunk, 16 / es);
        g = a.take<char>((by_rows ? chunk : m) * ldg * es);
        const int64_t rows = by_rows ? chunk : m, cols = by_rows ? v : chunk;
        sx = plan_split(rows, d, cols, dtype);
        sw = plan_split(cols, d, rows, dtype);
        const bool pieces = chunk < all;
        if ((!by_rows && pieces) || sx.splits > 1) slab_x = a.take<float>((int64_t)sx.splits * rows * slab_ld(d));
        if ((by_rows && pieces) || sw.splits > 1) slab_w = a.take<float>((int64_t)sw.splits * cols * slab_ld(d));
    }
};

void check_loss(int64_t m, int64_t v, int64_t d, int dtype) {
    check_size(m, 0, "m");
    check_size(v, 1, "v");
    check_size(d, 1, "d");
    check_dtype(dtype);
}

// One product of the softmax gradients with x or w. With `sums` its result
// adds up over the pieces (through the slab), else each piece has its own rows.
void launch_gradient(Product q, const LossPlan& plan, float* slab, Split split, bool sums, bool first, bool last,
                     void* out, int64_t ldo, int64_t labels, int dtype, cudaStream_t s) {
    q.dtype = dtype;
    q.alpha = 1.f;
    q.alpha_dev = plan.alpha;
    q.labels = labels;
    if (!slab) {
        q.epi = kEpiLinear;
        q.out = out; q.ldo = ldo; q.out_dtype = dtype;
        launch_product(q, s);
        return;
    }
    q.epi = kEpiSlab;
    q.slab = slab;
    q.splits = (int)ceil_div(q.R, split.len);
    q.split_len = split.len;
    q.accumulate = sums && !first;
    launch_product(q, s);
    if (!sums || last)
        launch_slab_sum(q.M, q.N, slab, slab_ld(q.N), sums ? split.splits : q.splits, out, ldo, 1.f, plan.alpha,
                        q.targets, labels, dtype, s);
}

// Makes a stream's device current (the null stream's is).
struct OnDeviceOf {
    int device = 0, before = 0;
    explicit OnDeviceOf(cudaStream_t s) {
        OPS_CK(cudaGetDevice(&before));
        OPS_CK(cudaStreamGetDevice(s, &device));
        if (device != before) OPS_CK(cudaSetDevice(device));
    }
    ~OnDeviceOf() {
        if (device != before) cudaSetDevice(before);
    }
    OnDeviceOf(const OnDeviceOf&) = delete;
};

const char* at(const void* p, int64_t elements, int es) { return static_cast<const char*>(p) + elements * es; }
char* at(void* p, int64_t elements, int es) { return static_cast<char*>(p) + elements * es; }

}  // namespace
}  // namespace ops
}  // namespace msplat

using namespace msplat;
using namespace msplat::ops;

extern "C" {

int msplat_ops_status(void* stream) {
    return guarded([&] {
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        OnDeviceOf on(s);
        unsigned long long id = 0;
        OPS_CK(cudaStreamGetId(s, &id));
        const std::array<unsigned, 3> now = {gave_up_tc16(s), gave_up_tcv(s), gave_up_rows(s)};
        // (a stream that has not asked yet starts from none)
        static std::mutex lock;
        static std::map<std::pair<int, unsigned long long>, std::array<unsigned, 3>> told;
        std::lock_guard<std::mutex> hold(lock);
        std::array<unsigned, 3>& last = told[{on.device, id}];
        const bool more = last != now;
        last = now;
        if (more)
            throw Error(MSPLAT_ERR_CUDA, "a kernel gave up waiting: results since this stream's last call are not valid");
    });
}

int msplat_ops_rehearse_timeout(int32_t kernels, void* stream) {
    return guarded([&] {
        require(kernels >= 0 && kernels <= 2, "kernels must be 0, 1 or 2");
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        OnDeviceOf on(s);
        kernels == 0 ? give_up_tc16(s) : kernels == 1 ? give_up_tcv(s) : give_up_rows(s);
    });
}

int msplat_linear_forward(int64_t m, int64_t n, int64_t k, const void* x, int64_t ldx, const void* w, int64_t ldw,
                          const void* bias, int32_t activation, const void* residual, int64_t ldr, void* preact,
                          int64_t ldz, void* y, int64_t ldy, int32_t dtype, int32_t y_dtype, void* stream) {
    return guarded([&] {
        check_size(m, 0, "m");
        check_size(n, 1, "n");
        check_size(k, 1, "k");
        check_act(activation);
        check_dtype(dtype);
        require(y_dtype == dtype || y_dtype == MSPLAT_DTYPE_F32, "y_dtype must be dtype or MSPLAT_DTYPE_F32");
        if (m == 0) return;
        const int es = dtype_size(dtype), eo = dtype_size(y_dtype);
        check_matrix(x, m, k, ldx, es, "x");
        check_matrix(w, n, k, ldw, es, "w");
        if (bias) check_matrix(bias, 1, n, n, es, "bias");
        if (residual) check_matrix(residual, m, n, ldr, eo, "residual");
        if (preact) check_matrix(preact, m, n, ldz, eo, "preact");
        check_matrix(y, m, n, ldy, eo, "y");
        Product p{};
        p.M = m; p.N = n; p.R = k;
        p.A = x; p.lda = ldx;
        p.B = w; p.ldb = ldw;
        p.dtype = dtype;
        p.epi = kEpiLinear;
        p.bias = bias;
        p.act = activation;
        p.residual = residual; p.ldr = ldr;
        p.preact = preact; p.ldz = ldz;
        p.out = y; p.ldo = ldy; p.out_dtype = y_dtype;
        p.alpha = 1.f;
        launch_product(p, static_cast<cudaStream_t>(stream));
    });
}

int msplat_linear_backward_workspace(int64_t m, int64_t n, int64_t k, int32_t activation, int32_t dtype,
                                     uint64_t* bytes) {
    return guarded([&] {
        check_backward(m, n, k, activation, dtype);
        require(bytes, "bytes is null");
        Arena a(nullptr);
        if (m > 0) BackwardPlan(a, m, n, k, activation, dtype);
        *bytes = a.used;
    });
}

int msplat_linear_backward(int64_t m, int64_t n, int64_t k, const void* x, int64_t ldx, const void* w, int64_t ldw,
                           const void* preact, int64_t ldz, int32_t activation, const void* dy, int64_t lddy,
                           void* dx, int64_t lddx, void* dw, int64_t lddw, void* dbias, int32_t dtype,
                           void* workspace, uint64_t workspace_bytes, void* stream) {
    return guarded([&] {
        check_backward(m, n, k, activation, dtype);
        const int es = dtype_size(dtype);
        if (dw) {
            check_matrix(x, m, k, ldx, es, "x");
            check_matrix(dw, n, k, lddw, es, "dw");
        }
        if (dx) {
            check_matrix(w, n, k, ldw, es, "w");
            check_matrix(dx, m, k, lddx, es, "dx");
        }
        if (dbias) check_matrix(dbias, 1, n, n, es, "dbias");
        check_matrix(dy, m, n, lddy, es, "dy");
        if (activation != MSPLAT_ACT_NONE) check_matrix(preact, m, n, ldz, es, "preact");
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        if (m == 0) {
            if (dw) OPS_CK(cudaMemset2DAsync(dw, lddw * es, 0, k * es, n, s));
            if (dbias) OPS_CK(cudaMemsetAsync(dbias, 0, n * es, s));
            return;
        }
        Arena a(workspace);
        const BackwardPlan plan(a, m, n, k, activation, dtype);
        check_workspace(a, workspace, workspace_bytes);
        if (plan.rows) {
            if (!dx && !dw && !dbias) return;
            launch_rows_layer(m, n, k, x, ldx, w, ldw, preact, ldz, activation, dy, lddy, dx, lddx,
                              dw ? plan.slab : nullptr, dbias ? plan.sums : nullptr, dtype, s);
            if (dw) launch_slab_sum(n, k, plan.slab, slab_ld(k), plan.pieces, dw, lddw, 1.f, nullptr, nullptr, 0, dtype, s);
            if (dbias) launch_slab_sum(1, n, plan.sums, n, plan.pieces, dbias, n, 1.f, nullptr, nullptr, 0, dtype, s);
            return;
        }
        const void* dz = dy;
        int64_t lddz = lddy;
        if (activation != MSPLAT_ACT_NONE || dbias) {
            launch_dz(m, n, preact, ldz, activation, dy, lddy, plan.dz, plan.lddz, dbias ? plan.sums : nullptr, dtype,
                      s);
            if (dbias) launch_slab_sum(1, n, plan.sums, n, plan.pieces, dbias, n, 1.f, nullptr, nullptr, 0, dtype, s);
            if (plan.dz) {
                dz = plan.dz;
                lddz = plan.lddz;
            }
        }
        if (dx) {
            Product p{};
            p.M = m; p.N = k; p.R = n;
            p.A = dz; p.lda = lddz;
            p.B = w; p.ldb = ldw; p.b_mn = true;
            p.dtype = dtype;
            p.epi = kEpiLinear;
            p.out = dx; p.ldo = lddx; p.out_dtype = dtype;
            p.alpha = 1.f;
            launch_product(p, s);
        }
        if (dw) {
            Product p{};
            p.M = n; p.N = k; p.R = m;
            p.A = dz; p.lda = lddz; p.a_mn = true;
            p.B = x; p.ldb = ldx; p.b_mn = true;
            p.dtype = dtype;
            p.epi = kEpiSlab;
            p.slab = plan.slab;
            p.splits = plan.split.splits;
            p.split_len = plan.split.len;
            launch_product(p, s);
            launch_slab_sum(n, k, plan.slab, slab_ld(k), plan.split.splits, dw, lddw, 1.f, nullptr, nullptr, 0, dtype, s);
        }
    });
}

int msplat_dropout(int64_t rows, int64_t cols, const void* x, int64_t ldx, const void* residual, int64_t ldr,
                   void* y, int64_t ldy, float p, uint64_t seed, uint64_t offset, const uint64_t* offset_dev,
                   int32_t dtype, void* stream) {
    return guarded([&] {
        check_size(rows, 0, "rows");
        check_size(cols, 0, "cols");
        check_dtype(dtype);
        require(p >= 0.f && p <= 1.f, "p must be in [0, 1]");
        if (rows == 0 || cols == 0) return;
        const int es = dtype_size(dtype);
        check_matrix(x, rows, cols, ldx, es, "x");
        if (residual) check_matrix(residual, rows, cols, ldr, es, "residual");
        check_matrix(y, rows, cols, ldy, es, "y");
        require(reinterpret_cast<uintptr_t>(offset_dev) % 8 == 0, "offset_dev is not aligned to its type");
        const uint32_t below = (uint32_t)std::floor((double)p * 65536.0 + 0.5);
        const float scale = below < 65536 ? (float)(65536.0 / (65536.0 - below)) : 0.f;
        launch_dropout(rows, cols, x, ldx, residual, ldr, y, ldy, below, scale, seed, offset, offset_dev, dtype,
                       static_cast<cudaStream_t>(stream));
    });
}

int msplat_loss_cross_entropy_workspace(int64_t m, int64_t v, int64_t d, int32_t grad, int32_t dtype,
                                        uint64_t* bytes) {
    return guarded([&] {
        check_loss(m, v, d, dtype);
        require(bytes, "bytes is null");
        Arena a(nullptr);
        if (m > 0) LossPlan(a, m, v, d, grad != 0, dtype);
        *bytes = a.used;
    });
}

int msplat_loss_cross_entropy(int64_t m, int64_t v, int64_t d, const void* x, int64_t ldx, const void* w,
                              int64_t ldw, const int32_t* targets, float logit_scale, float weight, float* loss,
                              float* row_loss, void* dx, int64_t lddx, void* dw, int64_t lddw, int32_t dtype,
                              void* workspace, uint64_t workspace_bytes, void* stream) {
    return guarded([&] {
        check_loss(m, v, d, dtype);
        require(std::isfinite(logit_scale) && std::isfinite(weight), "logit_scale and weight must be finite");
        const int es = dtype_size(dtype);
        check_matrix(x, m, d, ldx, es, "x");
        check_matrix(w, v, d, ldw, es, "w");
        if (m > 0) check_matrix(targets, 1, m, m, 4, "targets");
        if (loss) check_matrix(loss, 1, 1, 1, 4, "loss");
        if (row_loss) check_matrix(row_loss, 1, m, m, 4, "row_loss");
        if (dx) check_matrix(dx, m, d, lddx, es, "dx");
        if (dw) check_matrix(dw, v, d, lddw, es, "dw");
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        if (m == 0) {
            if (loss) OPS_CK(cudaMemsetAsync(loss, 0, sizeof(float), s));
            if (dw) OPS_CK(cudaMemset2DAsync(dw, lddw * es, 0, d * es, v, s));
            return;
        }
        const bool grad = dx || dw;
        Arena a(workspace);
        const LossPlan plan(a, m, v, d, grad, dtype);
        check_workspace(a, workspace, workspace_bytes);

        const float g_scale = dtype == MSPLAT_DTYPE_F16 ? 16384.f : 1.f;
        if (plan.rows) {
            const int blocks = rows_blocks(m);
            launch_count_labels(m, targets, v, plan.partial, blocks, s);
            launch_loss_total(plan.partial, blocks, 0.f, weight * logit_scale / g_scale, nullptr, plan.alpha, s);
            launch_rows_labels(m, v, d, x, ldx, w, ldw, targets, logit_scale, g_scale, plan.alpha, row_loss,
                               plan.partial, dx, lddx, dw ? plan.slab_w : nullptr, dtype, s);
            if (loss) launch_loss_total(plan.partial, blocks, weight, 0.f, loss, nullptr, s);
            if (dw)
                launch_slab_sum(v, d, plan.slab_w, slab_ld(d), blocks, dw, lddw, 1.f, plan.alpha, nullptr, 0, dtype, s);
            return;
        }
        Product logits{};
        logits.M = m; logits.N = v; logits.R = d;
        logits.A = x; logits.lda = ldx;
        logits.B = w; logits.ldb = ldw;
        logits.dtype = dtype;
        logits.targets = targets;
        logits.labels = v;
        logits.logit_scale = logit_scale;
        logits.g_scale = g_scale;

        if (plan.x) {
            launch_labelled_rows(m, d, x, ldx, targets, v, plan.x, plan.ldx, dtype, s);
            logits.A = x = plan.x;
            logits.lda = ldx = plan.ldx;
        }
        if (plan.w && !can_product_tc16(logits)) {
            launch_labelled_rows(v, d, w, ldw, nullptr, 0, plan.w, plan.ldx, dtype, s);
            logits.B = w = plan.w;
            logits.ldb = ldw = plan.ldx;
        }
        int joined = 0;
        for (int64_t r0 = 0; r0 < m; r0 += plan.stats_rows) {
            const int64_t rows = std::min(plan.stats_rows, m - r0);
            Product p = logits;
            p.M = rows;
            p.A = at(x, r0 * ldx, es);
            p.targets = targets + r0;
            p.epi = kEpiStats;
            p.stats = plan.stats; p.stats_ld = plan.stats_rows;
            p.label_logit = plan.label_logit + r0;
            launch_product(p, s);
            JoinArgs j{};
            j.m = rows; j.blocks = stats_blocks(p);
            j.stats = plan.stats; j.stats_ld = plan.stats_rows;
            j.label_logit = plan.label_logit + r0;
            j.targets = targets + r0; j.labels = v;
            j.norm = plan.norm + r0;
            j.row_loss = row_loss ? row_loss + r0 : nullptr;
            j.partial = plan.partial + 2 * joined;
            launch_join(j, s);
            joined += join_blocks(rows);
        }
        launch_loss_total(plan.partial, joined, weight, weight * logit_scale / g_scale, loss, plan.alpha, s);
        if (!grad) return;

        const int64_t all = plan.by_rows ? m : v;
        for (int64_t c0 = 0; c0 < all; c0 += plan.chunk) {
            const int64_t len = std::min(plan.chunk, all - c0);
            const int64_t r0 = plan.by_rows ? c0 : 0, rows = plan.by_rows ? len : m;
            const int64_t l0 = plan.by_rows ? 0 : c0, cols = plan.by_rows ? v : len;
            const bool first = c0 == 0, last = c0 + len >= all;
            Product p = logits;
            p.M = rows; p.N = cols;
            p.A = at(x, r0 * ldx, es);
            p.B = at(w, l0 * ldw, es);
            p.targets = targets + r0;
            p.epi = kEpiGrad;
            p.col0 = l0;
            p.norm = plan.norm + r0;
            p.out = plan.g; p.ldo = plan.ldg; p.out_dtype = dtype;
            launch_product(p, s);
            if (dx) {
                Product q{};
                q.M = rows; q.N = d; q.R = cols;
                q.A = plan.g; q.lda = plan.ldg;
                q.B = p.B; q.ldb = ldw; q.b_mn = true;
                q.targets = p.targets;
                launch_gradient(q, plan, plan.slab_x, plan.sx, !plan.by_rows, first, last, at(dx, r0 * lddx, es),
                                lddx, v, dtype, s);
            }
            if (dw) {
                Product q{};
                q.M = cols; q.N = d; q.R = rows;
                q.A = plan.g; q.lda = plan.ldg; q.a_mn = true;
                q.B = p.A; q.ldb = ldx; q.b_mn = true;
                launch_gradient(q, plan, plan.slab_w, plan.sw, plan.by_rows, first, last, at(dw, l0 * lddw, es),
                                lddw, v, dtype, s);
            }
        }
    });
}

}  // extern "C"
