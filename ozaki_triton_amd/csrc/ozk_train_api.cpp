// ozk_train_api.cpp -- the C entry points of the dense product with its epilogue,
// the router, and gradient norms (include/ozaki_amd.h): argument checks,
// workspace layout, launches.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <initializer_list>
#include <new>

#include "../../include/ozaki_amd.h"
#include "ozk_train.h"

namespace {

bool is_half(int d) { return d == OZK_F16 || d == OZK_BF16; }
bool is_float(int d) { return d == OZK_F32 || is_half(d); }
int64_t round_up(int64_t x, int64_t m) { return (x + m - 1) / m * m; }

int launched(hipError_t e) {
    return e == hipSuccess                     ? OZK_OK
           : e == hipErrorInvalidConfiguration ? OZK_ERR_TOO_LARGE
                                               : OZK_ERR_LAUNCH;
}
// the tile kernels step through up to 256 rows with 31-bit byte offsets
constexpr int64_t kMaxStride = (int64_t)1 << 22;
// no size negative, the product of all within 60 bits (so are byte offsets)
bool sizes_ok(std::initializer_list<int64_t> v) {
    double all = 1.0;
    for (int64_t x : v) {
        if (x < 0) return false;
        all *= x > 1 ? (double)x : 1.0;
    }
    return all < (double)((int64_t)1 << 60);
}
int stride_status(std::initializer_list<int64_t> v) {
    int st = OZK_OK;
    for (int64_t x : v) {
        if (x < 0) return OZK_ERR_SHAPE;
        if (x >= kMaxStride) st = OZK_ERR_TOO_LARGE;
    }
    return st;
}

// ---- dense products ----

// One product and its part of the workspace: copies of operands whose rows are no
// whole 16-byte pieces (where they pay and there is room), then partial sums.
ozk::GroupedParams as_grouped(const ozk::DenseParams &p) {
    ozk::GroupedParams g = {};
    g.A = p.A;
    g.B = p.B;
    g.T = p.M;
    g.K = p.K;
    g.N = p.N;
    g.G = 1;
    g.a_pitch = p.a_pitch;
    g.b_pitch = p.b_pitch;
    g.b_cols = p.b_cols;
    g.a_padded = p.a_padded;
    g.b_padded = p.b_padded;
    return g;
}
ozk::GroupedGradParams as_grad(const ozk::DenseParams &p) {   // K rows of M and of N
    ozk::GroupedGradParams g = {};
    g.A = p.A;
    g.D = p.B;
    g.T = p.K;
    g.K = p.M;
    g.N = p.N;
    g.G = 1;
    g.splits = 1;
    g.a_pitch = p.a_pitch;
    g.d_pitch = p.b_pitch;
    g.a_padded = p.a_padded;
    g.d_padded = p.b_padded;
    return g;
}
ozk::PackedSizes copies(const ozk::DenseParams &p) {
    // few rows go past the tiles
    if (ozk::dense_few(p)) return {0, 0};
    if (p.a_cols) return ozk::plan_grad_pack(as_grad(p));
    ozk::GroupedParams g = as_grouped(p);
    // a grouped product has smaller tiles for fewer than 48 rows, this one does not (us,
    // read as they are / copied: 40 x 6592 x 2861 59 / 25, 40 x 4096 x 4097 28 / 26, but 40 x
    // 8192 x 8190 58 / 69; the rule does not know the K ranges)
    if (g.T > 32 && g.T < 48) g.T = 48;
    return ozk::plan_grouped_pack(g);
}
size_t part_bytes(const ozk::DenseParams &p, int splits) {
    return splits > 1 ? (size_t)round_up((int64_t)splits * p.M * p.N * 4, 16) : 0;
}
// partial sums, then the copies
size_t dense_bytes(const ozk::DenseParams &p) {
    return part_bytes(p, ozk::dense_splits(p)) + copies(p).total();
}
int run_dense(ozk::DenseParams p, int dtype, char *ws, size_t room, hipStream_t st) {
    if (p.M == 0 || p.N == 0) return OZK_OK;
    p.splits = ozk::dense_splits(p);
    const size_t part = part_bytes(p, p.splits);
    if (part > room) return OZK_ERR_WORKSPACE;
    p.part = (float *)ws;
    const ozk::PackedSizes n = copies(p);
    if (n.total() && room - part >= n.total()) {
        char *to = ws + part;
        hipError_t e;
        if (p.a_cols) {
            ozk::GroupedGradParams g = as_grad(p);
            e = ozk::pack_grad(g, n, to, st);
            p.A = g.A;
            p.B = g.D;
            p.a_pitch = g.a_pitch;
            p.b_pitch = g.d_pitch;
            p.a_padded = g.a_padded;
            p.b_padded = g.d_padded;
        } else {
            ozk::GroupedParams g = as_grouped(p);
            e = ozk::pack_grouped(g, n, to, st);
            p.A = g.A;
            p.B = g.B;
            p.a_pitch = g.a_pitch;
            p.b_pitch = g.b_pitch;
            p.a_padded = g.a_padded;
            p.b_padded = g.b_padded;
        }
        if (e != hipSuccess) return launched(e);
    }
    return launched(ozk::launch_dense(p, dtype, st));
}

// x [M, K] and W [N, K] as the forward product reads them
int linear_params(ozk::DenseParams &p, const void *x, int64_t x_stride, const void *W,
                  const int64_t w_strides[2], int64_t M, int64_t N, int64_t K) {
    if (!w_strides) return OZK_ERR_NULL;
    if (!sizes_ok({M, N, K})) return OZK_ERR_SHAPE;
    if (w_strides[0] != 1 && w_strides[1] != 1) return OZK_ERR_SHAPE;
    p = {};
    p.b_cols = w_strides[1] != 1;
    const int64_t w_pitch = p.b_cols ? w_strides[1] : w_strides[0];
    if (int st = stride_status({x_stride, w_pitch})) return st;
    p.A = (const char *)x;
    p.B = (const char *)W;
    p.M = M;
    p.N = N;
    p.K = K;
    p.a_pitch = x_stride * 2;
    p.b_pitch = w_pitch * 2;
    p.splits = 1;
    return OZK_OK;
}

// What a backward call has in its workspace: dz, the bias' partial sums, and what
// the two products need, one after the other.
struct BackwardPlan {
    ozk::DenseParams dx, dw;
    ozk::DenseGradParams d;
    size_t dz, sums, products;
    size_t total() const { return dz + sums + products; }
};
int backward_plan(BackwardPlan &b, const void *dy, int64_t dy_stride, const void *x,
                  int64_t x_stride, const void *W, const int64_t w_strides[2], int activation,
                  int64_t M, int64_t N, int64_t K, int want, const void *ws) {
    ozk::DenseParams f;
    if (int st = linear_params(f, x, x_stride, W, w_strides, M, N, K)) return st;
    if (activation < OZK_ACT_NONE || activation > OZK_ACT_SILU) return OZK_ERR_SHAPE;
    if (want & ~7) return OZK_ERR_SHAPE;
    if (int st = stride_status({dy_stride})) return st;
    const bool act = activation != OZK_ACT_NONE, products = (want & 3) != 0 && M > 0 && N > 0;
    const int64_t padded = round_up(N, 8);
    if (act && M > 1 && padded >= kMaxStride) return OZK_ERR_TOO_LARGE;
    b = {};
    b.d.dy = (const char *)dy;
    b.d.dy_pitch = dy_stride * 2;
    b.d.M = M;
    b.d.N = N;
    b.d.act = activation;
    b.d.rows = ozk::dense_grad_rows(M, N);
    b.dz = act && products ? (size_t)round_up(M * padded * 2, 256) : 0;
    b.sums = (want & 4) && M > 0 ? (size_t)round_up((M + b.d.rows - 1) / b.d.rows * N * 4, 256) : 0;
    const char *dz = act ? (const char *)ws : (const char *)dy;
    const int64_t pitch = M <= 1 ? 0 : act ? padded * 2 : dy_stride * 2;
    // dx = dz W: the contraction runs along N
    b.dx = {};
    b.dx.A = dz;
    b.dx.B = f.B;
    b.dx.M = M;
    b.dx.N = K;
    b.dx.K = N;
    b.dx.a_pitch = pitch;
    b.dx.b_pitch = f.b_pitch;
    b.dx.a_padded = act;
    b.dx.b_cols = !f.b_cols;
    b.dx.splits = 1;
    // dW = dz^T x: along M
    b.dw = {};
    b.dw.A = dz;
    b.dw.B = f.A;
    b.dw.M = N;
    b.dw.N = K;
    b.dw.K = M;
    b.dw.a_pitch = pitch;
    b.dw.b_pitch = f.a_pitch;
    b.dw.a_padded = act;
    b.dw.a_cols = b.dw.b_cols = true;
    b.dw.splits = 1;
    if (want & 1) b.products = dense_bytes(b.dx);
    if (want & 2) b.products = std::max(b.products, dense_bytes(b.dw));
    return OZK_OK;
}

// ---- gradient norms ----

// Partial sums: one to a workgroup, kClipGrid of them shared by the launches by
// their pieces, at least one each
constexpr int64_t kClipGrid = 2048;
size_t clip_bytes(int64_t tensors) { return 8 * (size_t)(kClipGrid + tensors + 1); }

int clip_checks(const void *const *grads, void *const *outs, bool scaled, const int64_t *counts,
                const int *dtypes, int64_t tensors, double &elements, double &bytes) {
    if (tensors < 0) return OZK_ERR_SHAPE;
    if (tensors > (int64_t)1 << 28) return OZK_ERR_TOO_LARGE;
    if (tensors && (!grads || !counts || !dtypes || (scaled && !outs))) return OZK_ERR_NULL;
    elements = bytes = 0;
    for (int64_t i = 0; i < tensors; ++i) {
        if (!is_float(dtypes[i])) return OZK_ERR_DTYPE;
        if (counts[i] < 0 || counts[i] >= (int64_t)1 << 56) return OZK_ERR_SHAPE;
        if (counts[i] && (!grads[i] || (scaled && !outs[i]))) return OZK_ERR_NULL;
        elements += (double)counts[i];
        bytes += (double)counts[i] * (dtypes[i] == OZK_F32 ? 4 : 2);
    }
    return OZK_OK;
}

// No result may lie on another tensor's elements, or beside its own: the workgroups
// take them in any order.
int overlap_checks(const void *const *grads, void *const *outs, const int64_t *counts,
                   const int *dtypes, int64_t tensors) {
    struct Range {
        uintptr_t lo, hi;
        bool out;
    };
    Range *r = new (std::nothrow) Range[2 * (size_t)tensors + 1];
    if (!r) return OZK_ERR_WORKSPACE;
    size_t n = 0;
    for (int64_t i = 0; i < tensors; ++i) {
        const uintptr_t bytes = (uintptr_t)counts[i] * (dtypes[i] == OZK_F32 ? 4 : 2);
        if (!bytes) continue;
        const uintptr_t in = (uintptr_t)grads[i], out = (uintptr_t)outs[i];
        r[n++] = {out, out + bytes, true};
        if (in != out) r[n++] = {in, in + bytes, false};
    }
    std::sort(r, r + n, [](const Range &a, const Range &b) { return a.lo < b.lo; });
    uintptr_t all = 0, outs_to = 0;
    int st = OZK_OK;
    for (size_t i = 0; i < n; ++i) {
        if (r[i].lo < (r[i].out ? all : outs_to)) st = OZK_ERR_SHAPE;
        all = std::max(all, r[i].hi);
        if (r[i].out) outs_to = std::max(outs_to, r[i].hi);
    }
    delete[] r;
    return st;
}

int run_clip(const void *const *grads, void *const *outs, const int64_t *counts, const int *dtypes,
             int64_t tensors, double elements, double bytes, double max_norm, float *norm, double *part,
             hipStream_t st) {
    // pieces of 2^11 to 2^14 elements, at least about 4096 of them where there is enough:
    // larger ones come out uneven over the workgroups
    uint32_t size = 1 << 11;
    while (size < 1 << 14 && elements / (2 * size) >= 4096) size *= 2;
    // more than a launch counts: larger ones
    while (elements / size > (double)((int64_t)1 << 30)) {
        if (size >= 1u << 29) return OZK_ERR_TOO_LARGE;
        size *= 2;
    }
    // every launch's tensors, the same for both passes
    ozk::ClipParams p = {};
    p.size = size;
    p.part = part;
    p.max_norm = max_norm;
    p.past_caches = bytes > 256e6;
    const double whole = elements / size + (double)tensors;   // at least all pieces
    for (int pass = 0; pass < (outs ? 2 : 1); ++pass) {
        uint32_t part0 = 0;
        for (int64_t i = 0; i < tensors;) {
            p.count = 0;
            int64_t pieces = 0;
            for (; i < tensors && p.count < ozk::kClipTensors; ++i) {
                if (!counts[i]) continue;
                const int64_t n = (counts[i] + size - 1) / size;
                if (pieces + n > (int64_t)1 << 31) break;
                p.t[p.count++] = {(const char *)grads[i], outs ? (char *)outs[i] : nullptr, counts[i],
                                  (uint32_t)pieces, dtypes[i]};
                pieces += n;
            }
            if (!p.count) continue;
            p.pieces = (uint32_t)pieces;
            p.part0 = part0;
            const int64_t share = (int64_t)((double)kClipGrid * (double)pieces / whole);
            const uint32_t grid = (uint32_t)(share < 1 ? 1 : share < pieces ? share : pieces);
            if (pass == 0) {
                if (hipError_t e = ozk::launch_square_sums(p, grid, st); e != hipSuccess) return launched(e);
            } else {
                if (hipError_t e = ozk::launch_scale(p, grid, st); e != hipSuccess) return launched(e);
                p.norm = nullptr;
            }
            part0 += grid;
        }
        p.parts = part0;
        p.norm = norm;
        if (!outs || (pass == 1 && p.parts == 0)) return launched(ozk::launch_norm(p, st));
    }
    return OZK_OK;
}

}  // namespace

extern "C" {

int ozk_linear_workspace_bytes(const void *x, int64_t x_stride, const void *W,
                               const int64_t w_strides[2], int64_t M, int64_t N, int64_t K,
                               size_t *bytes_out) {
    if (!bytes_out) return OZK_ERR_NULL;
    ozk::DenseParams p;
    if (int st = linear_params(p, x, x_stride, W, w_strides, M, N, K)) return st;
    *bytes_out = dense_bytes(p);
    return OZK_OK;
}

int ozk_linear(const void *x, int64_t x_stride, const void *W, const int64_t w_strides[2],
               const void *bias, const void *residual, int64_t r_stride, int activation, int64_t M,
               int64_t N, int64_t K, int dtype, void *y, int64_t y_stride, void *z, void *workspace,
               size_t workspace_bytes, void *stream) {
    if (!is_half(dtype)) return OZK_ERR_DTYPE;
    ozk::DenseParams p;
    if (int st = linear_params(p, x, x_stride, W, w_strides, M, N, K)) return st;
    if (activation < OZK_ACT_NONE || activation > OZK_ACT_SILU || r_stride < 0 ||
        (M > 1 && y_stride < N))
        return OZK_ERR_SHAPE;
    if (M == 0 || N == 0) return OZK_OK;
    if (!y || (K > 0 && (!x || !W))) return OZK_ERR_NULL;
    if (workspace && ((uintptr_t)workspace & 15)) return OZK_ERR_WORKSPACE;
    p.C = (char *)y;
    p.c_pitch = y_stride * 2;
    p.bias = (const char *)bias;
    p.res = (const char *)residual;
    p.r_pitch = r_stride * 2;
    p.Z = (char *)z;
    p.act = activation;
    return run_dense(p, dtype, (char *)workspace, workspace ? workspace_bytes : 0, (hipStream_t)stream);
}

int ozk_linear_backward_workspace_bytes(const void *dy, int64_t dy_stride, const void *x,
                                        int64_t x_stride, const void *W, const int64_t w_strides[2],
                                        int activation, int64_t M, int64_t N, int64_t K, int want,
                                        size_t *bytes_out) {
    if (!bytes_out) return OZK_ERR_NULL;
    BackwardPlan b;
    if (int st = backward_plan(b, dy, dy_stride, x, x_stride, W, w_strides, activation, M, N, K,
                               want, nullptr))
        return st;
    *bytes_out = b.total();
    return OZK_OK;
}

int ozk_linear_backward(const void *dy, int64_t dy_stride, const void *z, const void *x,
                        int64_t x_stride, const void *W, const int64_t w_strides[2],
                        int activation, int64_t M, int64_t N, int64_t K, int dtype, void *dx,
                        int64_t dx_stride, void *dW, int64_t dw_stride, void *db, void *workspace,
                        size_t workspace_bytes, void *stream) {
    if (!is_half(dtype)) return OZK_ERR_DTYPE;
    const int want = (dx ? 1 : 0) | (dW ? 2 : 0) | (db ? 4 : 0);
    BackwardPlan b;
    if (int st = backward_plan(b, dy, dy_stride, x, x_stride, W, w_strides, activation, M, N, K,
                               want, workspace))
        return st;
    if ((dx && M > 1 && dx_stride < K) || (dW && N > 1 && dw_stride < K)) return OZK_ERR_SHAPE;
    const bool some = M > 0 && N > 0;
    if (some && (!dy || (activation != OZK_ACT_NONE && !z))) return OZK_ERR_NULL;
    if (some && K > 0 && (((want & 1) && !W) || ((want & 2) && !x))) return OZK_ERR_NULL;
    if (b.total() && (!workspace || workspace_bytes < b.total() || ((uintptr_t)workspace & 255)))
        return OZK_ERR_WORKSPACE;
    char *ws = (char *)workspace;
    const hipStream_t st = (hipStream_t)stream;
    // db's partial sums are added up by workgroups of dW's product where there is one
    const bool in_product = db && b.sums && (want & 2) && N > 0 && K > 0;
    if (N > 0) {
        b.d.z = (const char *)z;
        b.d.dz = b.dz ? ws : nullptr;
        b.d.dz_pitch = round_up(N, 8) * 2;
        b.d.sums = b.sums ? (float *)(ws + b.dz) : nullptr;
        b.d.db = (char *)db;
        if (b.d.dz || b.d.sums)
            if (hipError_t e = ozk::launch_dense_grad(b.d, dtype, st); e != hipSuccess) return launched(e);
        if (db && !in_product)   // (no rows: zeros)
            if (hipError_t e = ozk::launch_dense_bias(b.d, dtype, st); e != hipSuccess) return launched(e);
    }
    char *rest = ws ? ws + b.dz + b.sums : nullptr;
    if (in_product) {
        b.dw.sums = b.d.sums;
        b.dw.db = b.d.db;
        b.dw.db_n = N;
        b.dw.db_blocks = (M + b.d.rows - 1) / b.d.rows;
    }
    if (want & 1) {
        b.dx.C = (char *)dx;
        b.dx.c_pitch = dx_stride * 2;
        if (int r = run_dense(b.dx, dtype, rest, b.products, st)) return r;
    }
    if (want & 2) {
        b.dw.C = (char *)dW;
        b.dw.c_pitch = dw_stride * 2;
        if (int r = run_dense(b.dw, dtype, rest, b.products, st)) return r;
    }
    return OZK_OK;
}

static int route_checks(int64_t T, int64_t E, int64_t k, int64_t stride) {
    if (!sizes_ok({T, E}) || E < 1 || k < 1 || k > E || stride < 0) return OZK_ERR_SHAPE;
    if (E > OZK_MAX_EXPERTS || T >= (int64_t)1 << 31 || T * k >= (int64_t)1 << 31)
        return OZK_ERR_TOO_LARGE;
    return OZK_OK;
}
static ozk::RouteParams route_params(int64_t T, int64_t E, int64_t k) {
    ozk::RouteParams p = {};
    p.T = T;
    p.E = (int)E;
    p.k = (int)k;
    ozk::plan_route(p);
    return p;
}
static size_t route_bytes(const ozk::RouteParams &p) {
    return p.blocks > 1 ? (size_t)p.blocks * p.E * 8 : 0;
}

int ozk_route_workspace_bytes(int64_t T, int64_t E, int64_t k, size_t *bytes_out) {
    if (!bytes_out) return OZK_ERR_NULL;
    if (int st = route_checks(T, E, k, 0)) return st;
    *bytes_out = route_bytes(route_params(T, E, k));
    return OZK_OK;
}

int ozk_route(const void *logits, int dtype, int64_t l_stride, const void *mask, int64_t T, int64_t E,
              int64_t k, int normalize, int32_t *experts, float *weights, int32_t *order,
              int32_t *place, int32_t *offsets, int32_t *counts, float *loss, void *workspace,
              size_t workspace_bytes, void *stream) {
    if (!is_float(dtype)) return OZK_ERR_DTYPE;
    if (int st = route_checks(T, E, k, l_stride)) return st;
    if (!offsets || !counts || !loss) return OZK_ERR_NULL;
    if (T > 0 && (!logits || !experts || !weights || !order || !place)) return OZK_ERR_NULL;
    ozk::RouteParams p = route_params(T, E, k);
    const size_t need = route_bytes(p);
    if (need && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15)))
        return OZK_ERR_WORKSPACE;
    p.logits = (const char *)logits;
    p.mask = (const uint8_t *)mask;
    p.pitch = l_stride;
    p.normalize = normalize != 0;
    p.experts = experts;
    p.weights = weights;
    p.order = order;
    p.place = place;
    p.offsets = offsets;
    p.counts = counts;
    p.loss = loss;
    p.hist = (uint32_t *)workspace;
    p.psum = (float *)(p.hist + (int64_t)p.blocks * p.E);
    return launched(ozk::launch_route(p, dtype, (hipStream_t)stream));
}

int ozk_route_backward(const void *logits, int dtype, int64_t l_stride, const void *mask, int64_t T,
                       int64_t E, int64_t k, int normalize, const int32_t *experts,
                       const float *weights, const int32_t *counts, const float *dweights,
                       const float *dloss, void *dlogits, void *stream) {
    if (!is_float(dtype)) return OZK_ERR_DTYPE;
    if (int st = route_checks(T, E, k, l_stride)) return st;
    if (T == 0) return OZK_OK;
    if (!logits || !dlogits || !counts || (dweights && (!experts || !weights))) return OZK_ERR_NULL;
    ozk::RouteGradParams p = {};
    p.logits = (const char *)logits;
    p.mask = (const uint8_t *)mask;
    p.T = T;
    p.pitch = l_stride;
    p.E = (int)E;
    p.k = (int)k;
    p.normalize = normalize != 0;
    p.experts = experts;
    p.counts = counts;
    p.weights = weights;
    p.dw = dweights;
    p.dloss = dloss;
    p.dlogits = (char *)dlogits;
    return launched(ozk::launch_route_grad(p, dtype, (hipStream_t)stream));
}

int ozk_gradient_norm_workspace_bytes(int64_t tensors, size_t *bytes_out) {
    if (!bytes_out) return OZK_ERR_NULL;
    if (tensors < 0) return OZK_ERR_SHAPE;
    if (tensors > (int64_t)1 << 28) return OZK_ERR_TOO_LARGE;
    *bytes_out = clip_bytes(tensors);
    return OZK_OK;
}

int ozk_gradient_norm(const void *const *grads, const int64_t *counts, const int *dtypes,
                      int64_t tensors, float *norm, void *workspace, size_t workspace_bytes,
                      void *stream) {
    double elements, bytes;
    if (int st = clip_checks(grads, nullptr, false, counts, dtypes, tensors, elements, bytes)) return st;
    if (!norm) return OZK_ERR_NULL;
    if (!workspace || workspace_bytes < clip_bytes(tensors) || ((uintptr_t)workspace & 15))
        return OZK_ERR_WORKSPACE;
    return run_clip(grads, nullptr, counts, dtypes, tensors, elements, bytes, 0.0, norm, (double *)workspace,
                    (hipStream_t)stream);
}

int ozk_clip_gradients(const void *const *grads, void *const *outs, const int64_t *counts,
                       const int *dtypes, int64_t tensors, double max_norm, float *norm,
                       void *workspace, size_t workspace_bytes, void *stream) {
    double elements, bytes;
    if (int st = clip_checks(grads, outs, true, counts, dtypes, tensors, elements, bytes)) return st;
    if (!norm) return OZK_ERR_NULL;
    if (!(max_norm >= 0.0)) return OZK_ERR_SHAPE;
    if (!workspace || workspace_bytes < clip_bytes(tensors) || ((uintptr_t)workspace & 15))
        return OZK_ERR_WORKSPACE;
    if (!tensors)
        return run_clip(grads, nullptr, counts, dtypes, 0, 0.0, 0.0, 0.0, norm, (double *)workspace,
                        (hipStream_t)stream);
    if (int st = overlap_checks(grads, outs, counts, dtypes, tensors)) return st;
    return run_clip(grads, outs, counts, dtypes, tensors, elements, bytes, max_norm, norm,
                    (double *)workspace, (hipStream_t)stream);
}

}  // extern "C"
