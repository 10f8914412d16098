// ozk_linear_api.cpp -- the C entry points of the operators for linear layers
// (include/ozaki_amd.h): argument checks, workspace layout, launches.
#include <hip/hip_runtime.h>

#include <math.h>

#include <initializer_list>

#include "../../include/ozaki_amd.h"
#include "ozk_linear.h"

namespace {

bool is_half(int d) { return d == OZK_F16 || d == OZK_BF16; }
bool is_float(int d) { return d == OZK_F32 || is_half(d); }
int64_t round_up(int64_t x, int64_t m) { return (x + m - 1) / m * m; }

// a launch's status: a grid that does not fit is the caller's size
int launched(hipError_t e) {
    return e == hipSuccess                     ? OZK_OK
           : e == hipErrorInvalidConfiguration ? OZK_ERR_TOO_LARGE
                                               : OZK_ERR_LAUNCH;
}

// the tile kernels step through up to 256 rows with 32-bit offsets
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
// OZK_OK, or why rows cannot lie this far apart
int stride_status(std::initializer_list<int64_t> v) {
    int st = OZK_OK;
    for (int64_t x : v) {
        if (x < 0) return OZK_ERR_SHAPE;
        if (x >= kMaxStride) st = OZK_ERR_TOO_LARGE;
    }
    return st;
}

size_t wgrad_bytes(int64_t T, int64_t K, int64_t N, int64_t G) {
    const int s = ozk::grouped_grad_splits(T, K, N, G);
    return s > 1 ? (size_t)s * (size_t)(G * K * N) * 4 : 0;
}

// workspace of an orthogonalisation, in order: the partial sums, X (twice from
// two steps on), A, B
struct OrthLayout {
    size_t sums, x, a, total;
    int blocks, xs;
    OrthLayout(int64_t batch, int64_t M, int64_t N, int steps) {
        const int64_t m = M < N ? M : N, n = M < N ? N : M;
        blocks = ozk::orth_blocks(batch, M, N);
        xs = steps > 1 ? 2 : 1;
        sums = (size_t)round_up(batch * blocks * 8, 256);
        x = (size_t)(batch * m * ((n + 31) / 32 * 128));
        a = (size_t)(batch * m * ((m + 31) / 32 * 128));
        total = sums + xs * x + 2 * a;
    }
};

// the largest power of two that keeps values up to `bound` within fp16, with
// room for a factor of two
double slice_scale(double bound) {
    if (!(bound > 0.0)) return 1.0;
    const int e = (int)floor(log2(32768.0 / bound));
    return ldexp(1.0, e > 60 ? 60 : e < -60 ? -60 : e);
}
// largest |a + b t + c t^2| sqrt(t) over t in [0, top]
double bound_x(double a, double b, double c, double top) {
    auto f = [&](double t) { return fabs((a + b * t + c * t * t) * sqrt(t)); };
    double best = f(top);
    // where the derivative a + 3 b s^2 + 5 c s^4 is zero
    auto at = [&](double t) {
        if (t > 0 && t < top && f(t) > best) best = f(t);
    };
    if (c != 0) {
        const double d = 9 * b * b - 20 * a * c;
        if (d >= 0) {
            at((-3 * b + sqrt(d)) / (10 * c));
            at((-3 * b - sqrt(d)) / (10 * c));
        }
    } else if (b != 0) {
        at(-a / (3 * b));
    }
    return best;
}
// largest |b t + c t^2| over t in [0, top]
double bound_b(double b, double c, double top) {
    auto f = [&](double t) { return fabs(b * t + c * t * t); };
    double best = f(top);
    if (c != 0) {
        const double t = -b / (2 * c);
        if (t > 0 && t < top && f(t) > best) best = f(t);
    }
    return best;
}

}  // namespace

extern "C" {

int ozk_grouped_matmul(const void *A, int64_t a_stride, const void *B, const int64_t b_strides[3],
                       const void *offsets, int offset_bytes, int64_t T, int64_t K, int64_t N,
                       int64_t G, int dtype, void *C, int64_t c_stride, void *stream) {
    if (!is_half(dtype) || (offset_bytes != 4 && offset_bytes != 8)) return OZK_ERR_DTYPE;
    if (!b_strides) return OZK_ERR_NULL;
    if (!sizes_ok({T, K, N, G})) return OZK_ERR_SHAPE;
    if (b_strides[2] != 1 && b_strides[1] != 1) return OZK_ERR_SHAPE;
    if (T == 0 || N == 0) return OZK_OK;
    if (!C || !offsets || (K > 0 && (!A || (G > 0 && !B)))) return OZK_ERR_NULL;
    const bool cols = b_strides[2] == 1;
    const int64_t b_pitch = cols ? b_strides[1] : b_strides[2];
    if (c_stride < 0 || b_strides[0] < 0) return OZK_ERR_SHAPE;
    if (int st = stride_status({a_stride, b_pitch})) return st;
    ozk::GroupedParams p;
    p.A = (const char *)A;
    p.B = (const char *)B;
    p.C = (char *)C;
    p.offsets = offsets;
    p.T = T;
    p.K = K;
    p.N = N;
    p.G = G;
    p.a_pitch = a_stride * 2;
    p.b_group = b_strides[0] * 2;
    p.b_pitch = b_pitch * 2;
    p.c_pitch = c_stride * 2;
    p.b_cols = cols;
    p.offsets64 = offset_bytes == 8;
    return launched(ozk::launch_grouped(p, dtype, (hipStream_t)stream));
}

int ozk_grouped_matmul_wgrad_workspace_bytes(int64_t T, int64_t K, int64_t N, int64_t G,
                                             size_t *bytes_out) {
    if (!bytes_out) return OZK_ERR_NULL;
    if (!sizes_ok({T, K, N, G})) return OZK_ERR_SHAPE;
    *bytes_out = wgrad_bytes(T, K, N, G);
    return OZK_OK;
}

int ozk_grouped_matmul_wgrad(const void *A, int64_t a_stride, const void *D, int64_t d_stride,
                             const void *offsets, int offset_bytes, int64_t T, int64_t K,
                             int64_t N, int64_t G, int dtype, void *dB,
                             const int64_t db_strides[2], void *workspace,
                             size_t workspace_bytes, void *stream) {
    if (!is_half(dtype) || (offset_bytes != 4 && offset_bytes != 8)) return OZK_ERR_DTYPE;
    if (!db_strides) return OZK_ERR_NULL;
    if (!sizes_ok({T, K, N, G})) return OZK_ERR_SHAPE;
    if (K == 0 || N == 0 || G == 0) return OZK_OK;
    if (!dB || !offsets || (T > 0 && (!A || !D))) return OZK_ERR_NULL;
    if (db_strides[0] < 0 || db_strides[1] < 0) return OZK_ERR_SHAPE;
    if (int st = stride_status({a_stride, d_stride})) return st;
    const size_t need = wgrad_bytes(T, K, N, G);
    if (need && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15)))
        return OZK_ERR_WORKSPACE;
    ozk::GroupedGradParams p;
    p.A = (const char *)A;
    p.D = (const char *)D;
    p.dB = (char *)dB;
    p.offsets = offsets;
    p.T = T;
    p.K = K;
    p.N = N;
    p.G = G;
    p.a_pitch = a_stride * 2;
    p.d_pitch = d_stride * 2;
    p.db_group = db_strides[0] * 2;
    p.db_pitch = db_strides[1] * 2;
    p.offsets64 = offset_bytes == 8;
    p.part = (float *)workspace;
    p.splits = ozk::grouped_grad_splits(T, K, N, G);
    return launched(ozk::launch_grouped_grad(p, dtype, (hipStream_t)stream));
}

static int w4_checks(int64_t N, int64_t K, int group, const void *packed, int64_t packed_stride,
                     const void *scales, int64_t s_stride, const void *zeros, int64_t z_stride) {
    if (group != 32 && group != 64 && group != 128) return OZK_ERR_SHAPE;
    if (!sizes_ok({N, K})) return OZK_ERR_SHAPE;
    if (N == 0 || K == 0) return OZK_OK;
    if (!packed || !scales) return OZK_ERR_NULL;
    if (((uintptr_t)packed & 15) || packed_stride % 16 || packed_stride < (K + 31) / 32 * 16)
        return OZK_ERR_SHAPE;
    if (s_stride < 0 || (zeros && z_stride < 0)) return OZK_ERR_SHAPE;
    return OZK_OK;
}

int ozk_quantize_w4(const void *W, int dtype, int64_t N, int64_t K, int64_t w_stride, int group,
                    void *packed, int64_t packed_stride, void *scales, int64_t s_stride,
                    void *zeros, int64_t z_stride, void *stream) {
    if (!is_float(dtype)) return OZK_ERR_DTYPE;
    if (int st = w4_checks(N, K, group, packed, packed_stride, scales, s_stride, zeros, z_stride))
        return st;
    if (N == 0 || K == 0) return OZK_OK;
    if (!W) return OZK_ERR_NULL;
    if (w_stride < 0) return OZK_ERR_SHAPE;
    ozk::QuantParams p = {};
    p.W = (const char *)W;
    p.packed = (uint8_t *)packed;
    p.scales = (char *)scales;
    p.zeros = (uint8_t *)zeros;
    p.N = N;
    p.K = K;
    p.w_pitch = w_stride;
    p.p_pitch = packed_stride;
    p.s_pitch = s_stride;
    p.z_pitch = z_stride;
    p.group = group;
    return launched(ozk::launch_quantize_w4(p, dtype, (hipStream_t)stream));
}

int ozk_dequantize_w4(const void *packed, int64_t packed_stride, const void *scales,
                      int scale_dtype, int64_t s_stride, const void *zeros, int64_t z_stride,
                      int group, int64_t N, int64_t K, void *W, int dtype, int64_t w_stride,
                      void *stream) {
    if (!is_float(dtype) || (scale_dtype != dtype && scale_dtype != OZK_F32)) return OZK_ERR_DTYPE;
    if (int st = w4_checks(N, K, group, packed, packed_stride, scales, s_stride, zeros, z_stride))
        return st;
    if (N == 0 || K == 0) return OZK_OK;
    if (!W) return OZK_ERR_NULL;
    if (w_stride < 0) return OZK_ERR_SHAPE;
    ozk::QuantParams p = {};
    p.out = (char *)W;
    p.packed = (uint8_t *)const_cast<void *>(packed);
    p.scales = (char *)const_cast<void *>(scales);
    p.zeros = (uint8_t *)const_cast<void *>(zeros);
    p.N = N;
    p.K = K;
    p.w_pitch = w_stride;
    p.p_pitch = packed_stride;
    p.s_pitch = s_stride;
    p.z_pitch = z_stride;
    p.group = group;
    return launched(ozk::launch_dequantize_w4(p, dtype, scale_dtype, (hipStream_t)stream));
}

int ozk_matmul_w4_workspace_bytes(int dtype, int64_t M, int64_t N, int64_t K, int group,
                                  size_t *bytes_out) {
    if (!bytes_out) return OZK_ERR_NULL;
    if (!is_float(dtype)) return OZK_ERR_DTYPE;
    if (!sizes_ok({M, N, K}) || (group != 32 && group != 64 && group != 128)) return OZK_ERR_SHAPE;
    *bytes_out = 0;
    if (M == 0 || N == 0) return OZK_OK;
    ozk::W4Params p = {};
    p.M = M;
    p.N = N;
    p.K = K;
    p.group = group;
    ozk::plan_w4(p, dtype);
    if (p.splits > 1) *bytes_out = (size_t)p.splits * (size_t)(M * N) * 4;
    return OZK_OK;
}

int ozk_matmul_w4(const void *x, int dtype, int64_t x_stride, const void *packed,
                  int64_t packed_stride, const void *scales, int scale_dtype, int64_t s_stride,
                  const void *zeros, int64_t z_stride, int group, int64_t M, int64_t N, int64_t K,
                  void *y, int64_t y_stride, void *workspace, size_t workspace_bytes,
                  void *stream) {
    if (!is_float(dtype) || (scale_dtype != dtype && scale_dtype != OZK_F32)) return OZK_ERR_DTYPE;
    if (!sizes_ok({M, N, K}) || K == 0) return OZK_ERR_SHAPE;
    if (int st = w4_checks(N, K, group, packed, packed_stride, scales, s_stride, zeros, z_stride))
        return st;
    if (M == 0 || N == 0) return OZK_OK;
    if (!x || !y) return OZK_ERR_NULL;
    if (x_stride < 0 || y_stride < 0) return OZK_ERR_SHAPE;
    ozk::W4Params p = {};
    p.x = (const char *)x;
    p.packed = (const uint8_t *)packed;
    p.scales = scales;
    p.zeros = (const uint8_t *)zeros;
    p.y = (char *)y;
    p.M = M;
    p.N = N;
    p.K = K;
    p.x_pitch = x_stride;
    p.w_pitch = packed_stride;
    p.s_pitch = s_stride;
    p.z_pitch = z_stride;
    p.y_pitch = y_stride;
    p.scales32 = scale_dtype == OZK_F32;
    p.group = group;
    ozk::plan_w4(p, dtype);
    if (p.splits > 1) {
        if (!workspace || workspace_bytes < (size_t)p.splits * (size_t)(M * N) * 4 ||
            ((uintptr_t)workspace & 15))
            return OZK_ERR_WORKSPACE;
        p.part = (float *)workspace;
    }
    return launched(ozk::launch_w4(p, dtype, (hipStream_t)stream));
}

int ozk_orthogonalize_workspace_bytes(int64_t batch, int64_t M, int64_t N, int steps,
                                      size_t *bytes_out) {
    if (!bytes_out) return OZK_ERR_NULL;
    if (!sizes_ok({batch, M, N}) || steps < 1) return OZK_ERR_SHAPE;
    if (M >= kMaxStride || N >= kMaxStride || batch > 65535) return OZK_ERR_TOO_LARGE;
    *bytes_out = batch && M && N ? OrthLayout(batch, M, N, steps).total : 0;
    return OZK_OK;
}

int ozk_orthogonalize(const void *G, int dtype, int64_t batch, int64_t M, int64_t N,
                      const int64_t g_strides[2], const double *coefficients, int steps,
                      double eps, void *out, const int64_t o_strides[2], void *workspace,
                      size_t workspace_bytes, void *stream) {
    if (!is_float(dtype)) return OZK_ERR_DTYPE;
    if (!sizes_ok({batch, M, N}) || steps < 1 || steps > 64) return OZK_ERR_SHAPE;
    if (M >= kMaxStride || N >= kMaxStride || batch > 65535) return OZK_ERR_TOO_LARGE;
    if (!coefficients || !g_strides || !o_strides) return OZK_ERR_NULL;
    if (!batch || !M || !N) return OZK_OK;
    if (!G || !out) return OZK_ERR_NULL;
    if (g_strides[0] < 0 || g_strides[1] < 0 || o_strides[0] < 0 || o_strides[1] < 0)
        return OZK_ERR_SHAPE;
    const OrthLayout at(batch, M, N, steps);
    if (!workspace || workspace_bytes < at.total || ((uintptr_t)workspace & 15))
        return OZK_ERR_WORKSPACE;
    ozk::OrthParams p;
    p.G = (const char *)G;
    p.out = (char *)out;
    p.batch = batch;
    p.M = M;
    p.N = N;
    p.g_batch = g_strides[0];
    p.g_row = g_strides[1];
    p.o_batch = o_strides[0];
    p.o_row = o_strides[1];
    p.eps = eps;
    char *ws = (char *)workspace;
    p.sums = (double *)ws;
    p.blocks = at.blocks;
    p.X[0] = ws + at.sums;
    p.X[1] = p.X[0] + (at.xs > 1 ? at.x : 0);
    p.A = p.X[1] + at.x;
    p.B = p.A + at.a;

    // bounds of the singular values, step by step, and the slices' scales
    ozk::OrthStep step[64];
    double bound = 1.0, sx = slice_scale(bound);
    p.start_scale = (float)sx;
    for (int i = 0; i < steps; ++i) {
        const double a = coefficients[3 * i], b = coefficients[3 * i + 1],
                     c = coefficients[3 * i + 2];
        const double top = bound * bound;
        const double sa = slice_scale(top), sb = slice_scale(bound_b(b, c, top));
        bound = 1.001 * bound_x(a, b, c, top);
        const double next = i + 1 < steps ? slice_scale(bound) : 1.0;
        step[i].a_acc = (float)(sa / (sx * sx));
        step[i].b_a = (float)(b * sb / sa);
        step[i].b_acc = (float)(c * sb / (sa * sa));
        step[i].x_x = (float)(a * next / sx);
        step[i].x_acc = (float)(next / (sb * sx));
        sx = next;
    }
    return launched(ozk::launch_orth(p, step, steps, dtype, (hipStream_t)stream));
}

}  // extern "C"
