// ozk_linear_api.cpp -- the C entry points of the operators for linear layers
// (include/ozaki_amd.h): argument checks, workspace layout, launches.
#include <hip/hip_runtime.h>

#include <math.h>

#include <initializer_list>

#include "../../include/ozaki_amd.h"
#include "../../include/ozaki_amd_debug.h"
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

// the tile kernels step through up to 256 rows with 31-bit byte offsets: of two
// bytes an element, and of four in the slices of an orthogonalisation
constexpr int64_t kMaxStride = (int64_t)1 << 22, kMaxOrth = (int64_t)1 << 20;
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

// the largest power of two that keeps values up to `bound` within fp16, with
// room for a factor of two
double slice_scale(double bound) {
    if (!(bound > 0.0)) return 1.0;
    const double e = floor(log2(32768.0 / bound));
    return ldexp(1.0, e > 60 ? 60 : e > -60 ? (int)e : -60);
}
// largest |f(t)| over [0, top], at its end or at the places t[0 .. n) where it
// turns
template <typename F> double largest(F f, double top, const double *t, int n) {
    double best = fabs(f(top)), f0 = fabs(f(0.0));
    if (f0 > best) best = f0;
    for (int i = 0; i < n; ++i)
        if (t[i] > 0 && t[i] < top && fabs(f(t[i])) > best) best = fabs(f(t[i]));
    return best;
}
// Bounds over the eigenvalues t of A, 0 .. top, of what a step with a, b, c makes
struct OrthBounds {
    double x;     // singular values of the next X: |a + b t + c t^2| sqrt(t)
    double b;     // of B: |b t + c t^2|
    double p;     // of P: |a + b t + c t^2|
    double w;     // of P A: the same times t
    double slope; // |b + 2 c t|
    double gain;  // of an error in X: |a + b t + c t^2|, or |a + 3 b t + 5 c t^2| along s
    OrthBounds() = default;
    OrthBounds(double a, double b_, double c, double top) {
        auto poly = [&](double t) { return a + b_ * t + c * t * t; };
        // where (a + b t + c t^2) t^k turns: k a + (k + 1) b t + (k + 2) c t^2 = 0
        auto turns = [&](double k, double (&t)[2]) -> int {
            const double qa = (k + 2) * c, qb = (k + 1) * b_, qc = k * a;
            if (qa == 0) {
                if (qb == 0) return 0;
                t[0] = -qc / qb;
                return 1;
            }
            const double d = qb * qb - 4 * qa * qc;
            if (!(d >= 0)) return 0;
            t[0] = (-qb + sqrt(d)) / (2 * qa);
            t[1] = (-qb - sqrt(d)) / (2 * qa);
            return 2;
        };
        double t[2];
        int n = turns(0.5, t);
        x = 1.001 * largest([&](double u) { return poly(u) * sqrt(u); }, top, t, n);
        n = turns(0, t);
        b = largest([&](double u) { return b_ * u + c * u * u; }, top, t, n);
        p = largest(poly, top, t, n);
        n = turns(1, t);
        w = largest([&](double u) { return poly(u) * u; }, top, t, n);
        slope = largest([&](double u) { return b_ + 2 * c * u; }, top, t, 0);
        t[0] = c != 0 ? -3 * b_ / (10 * c) : 0;
        gain = largest([&](double u) { return a + 3 * b_ * u + 5 * c * u * u; }, top, t, 1);
        if (p > gain) gain = p;
    }
};

// Worst-case error of a result, to first order, from what the slices round:
// 2^-22 of a matrix' bound, each time one is made.
struct OrthErrors {
    static constexpr double e = 0x1p-22;
    const OrthBounds *at;
    const double *bound;   // of X before each step
    // Steps by themselves: an error d in X leaves a step as gain d, and the step
    // adds what the slices of A, B and the new X round.
    double own(int steps) const {
        double d = e;
        for (int i = 0; i < steps; ++i) {
            const double top = bound[i] * bound[i];
            d = at[i].gain * d + bound[i] * e * (at[i].slope * top + at[i].b) + e * bound[i + 1];
        }
        return d;
    }
    // The last j steps on A alone: with W = P A and A' = W P errors go from A to
    // P by P's slope, from both to W and A', and from every P to Q.
    double chain(int steps, int j) const {
        const int from = steps - j;
        double d = own(from), dA = e * bound[from] * bound[from], dP = 0, q = 1, dQ = 0;
        for (int i = from; i < steps; ++i) {
            d *= at[i].gain;
            if (i > from) {
                const OrthBounds &k = at[i - 1];
                const double dW = k.p * dA + bound[i - 1] * bound[i - 1] * dP + e * k.w;
                dA = k.p * dW + k.w * dP + e * bound[i] * bound[i];
            }
            dP = at[i].slope * dA + e * at[i].p;
            dQ = at[i].p * dQ + q * dP + (i > from ? e * q * at[i].p : 0);
            q *= at[i].p;
        }
        return d + dQ * bound[from];
    }
};

// The slices' scales come from the bounds where each is within this: values of
// order 1 then keep 22 bits (2^-25 of 2^14 / 2^10) in sums of up to 2^13 of them.
constexpr double kOrthTight = 1024;

bool chain_pays(int64_t m, int64_t n) { return n >= 2 * m; }   // see plan_orth

// The products of an orthogonalisation (X [m, n], m <= n).
//
// One step by itself is A = X X^T, B = b A + c A A, X' = a X + B X, one
// symmetric and one full product of X.  The last j steps can go without X in
// between: with P = a I + b A + c A A, X' = P X and so A' = P A P, and all of
// these are polynomials in A, symmetric and commuting.  Then A = X X^T and Q X
// are paid once, Q the product of the P's, and a step is P, P A, (P A) P and P Q,
// four symmetric products of [m, m]: less where n is at least 2 m (measured, a
// step by itself / one of these, 2048 x 8192: 323 / 145 us, 2048 x 4096: 193 /
// 145, 2048 x 2048: 120 / 145).  What it costs
// is accuracy: A's rounding is amplified by P^2 a step and by P's slope into
// every P.  So j is the most whose worst case (OrthErrors) is within 1.5 times that
// of the steps by themselves, and the result is as near as theirs.  With the
// coefficients 3.4445, -4.775, 2.0315 that is 2 of 5 steps; error before the last
// rounding on matrices of 64 x 200 with singular values over four decades, for j =
// 1 .. 5: 3.7e-6, 3.7e-6, 6.4e-6, 3.7e-5, 7.7e-5 (plain fp32 4.6e-6).  For fp32
// results every step runs by itself: products more of 22 bits show there (4 steps
// of 1.5, -0.5, 0: 1.0e-7, with j = 2 1.6e-7).
//
// The bounds are over whole intervals, each step's over all that the one before
// may give, and can grow far past every value (published triples from 8.29, -23.6,
// 17.3 to 1.875, -1.25, 0.375: to 1e89 in seven steps that take all of [0, 1] to
// within 2; slices on that scale are zeros).  Where a bound is past kOrthTight, every
// step runs by itself on scales that are measured: A of X / |X| has entries within
// 1, and B and the next X are written as fp32 values first (two launches more each).
void plan_orth(ozk::OrthPlan &plan, int64_t m, int64_t n, const double *co, int steps, int dtype) {
    double bound[65] = {1.0};
    OrthBounds at[64];
    for (int i = 0; i < steps; ++i) {
        at[i] = OrthBounds(co[3 * i], co[3 * i + 1], co[3 * i + 2], bound[i] * bound[i]);
        bound[i + 1] = at[i].x;
    }
    plan.measured = false;
    for (int i = 0; i < steps; ++i)
        if (!(bound[i] * bound[i] <= kOrthTight && at[i].b <= kOrthTight)) plan.measured = true;
    int j = 1;
    if (chain_pays(m, n) && dtype != OZK_F32 && !plan.measured) {
        const OrthErrors err = {at, bound};
        double q = at[steps - 1].p;
        while (j < steps && (q *= at[steps - 1 - j].p) <= kOrthTight &&
               err.chain(steps, j + 1) <= 1.5 * err.own(steps))
            ++j;
    }
    auto push = [&](int kind, int L, int R, int Y, int D, double f_acc, double f_y, double f_i) {
        plan.op[plan.ops++] = {kind, L, R, Y, D, (float)f_acc, (float)f_y, (float)f_i};
        if (D + 1 > plan.squares) plan.squares = D + 1;
    };
    constexpr int none = -9;
    plan.ops = plan.squares = 0;
    plan.xs = steps - j > 0 ? 2 : 1;
    double sx = slice_scale(1.0);
    plan.start_scale = (float)sx;
    if (plan.measured) {
        for (int i = 0; i < steps; ++i) {
            const double a = co[3 * i], b = co[3 * i + 1], c = co[3 * i + 2];
            const bool last = i + 1 == steps;
            push(ozk::kOrthXX, -1, -1, none, 0, 1 / sx, 0, 0);
            push(ozk::kOrthNewB, 0, 0, 0, 0, c / (sx * sx), b / sx, 0);
            push(last ? ozk::kOrthLast : ozk::kOrthNewX, 0, -1, -1, last ? none : -1,
                 1 / (sx * sx), a / sx, 0);
        }
        plan.squares = 2;                         // and one for B's fp32 values
        return;
    }
    int x = -1;                                   // X's buffer
    const int own = j > 1 ? steps - j : steps;    // steps by themselves
    for (int i = 0; i < own; ++i) {
        const double a = co[3 * i], b = co[3 * i + 1], c = co[3 * i + 2];
        const bool last = i + 1 == steps;
        const double sa = slice_scale(bound[i] * bound[i]), sb = slice_scale(at[i].b);
        const double next = last ? 1.0 : slice_scale(bound[i + 1]);
        push(ozk::kOrthXX, x, x, none, 0, sa / (sx * sx), 0, 0);
        push(ozk::kOrthSym, 0, 0, 0, 1, c * sb / (sa * sa), b * sb / sa, 0);
        push(last ? ozk::kOrthLast : ozk::kOrthX, 1, x, x, last ? none : -3 - x, next / (sb * sx),
             a * next / sx, 0);
        sx = next;
        x = -3 - x;                               // -1 and -2 in turn
    }
    if (j == 1) return;
    double sa = slice_scale(bound[own] * bound[own]), sp = 1, sq = 1, all = 1;
    int P = -1, Q = -1;
    push(ozk::kOrthXX, x, x, none, 0, sa / (sx * sx), 0, 0);
    for (int i = own; i < steps; ++i) {
        const double a = co[3 * i], b = co[3 * i + 1], c = co[3 * i + 2];
        if (i > own) {
            const double sw = slice_scale(at[i - 1].w), na = slice_scale(bound[i] * bound[i]);
            push(ozk::kOrthSym, P, 0, none, 2, sw / (sp * sa), 0, 0);
            push(ozk::kOrthSym, 2, P, none, 0, na / (sw * sp), 0, 0);
            sa = na;
        }
        const OrthBounds &k = at[i];
        sp = slice_scale(k.p);
        all *= k.p;
        P = Q == 1 ? 3 : 1;
        push(ozk::kOrthSym, 0, 0, 0, P, c * sp / (sa * sa), b * sp / sa, a * sp);
        if (i == own) {
            Q = P;
            sq = sp;
        } else {
            const double ns = slice_scale(all);
            const int to = P != 3 && Q != 3 ? 3 : P != 4 && Q != 4 ? 4 : 1;
            push(ozk::kOrthSym, P, Q, none, to, ns / (sp * sq), 0, 0);
            Q = to;
            sq = ns;
        }
    }
    push(ozk::kOrthLast, Q, x, none, none, 1.0 / (sq * sx), 0, 0);
}

// workspace of an orthogonalisation, in order: the partial sums and the norms of
// X and B, X (twice where steps run by themselves), the square matrices.  The size covers every plan.
struct OrthLayout {
    size_t norms, sums, x, a, total;
    int blocks;
    OrthLayout(int64_t batch, int64_t M, int64_t N, int xs, int squares) {
        const int64_t m = M < N ? M : N, n = M < N ? N : M;
        blocks = ozk::orth_blocks(batch, M, N);
        norms = (size_t)(batch * blocks * 8);
        sums = (size_t)round_up((int64_t)norms + 2 * batch * 8, 256);
        x = (size_t)(batch * m * ((n + 31) / 32 * 128));
        a = (size_t)(batch * m * ((m + 31) / 32 * 128));
        total = sums + xs * x + squares * a;
    }
};
// what any plan of so many steps takes: all steps by themselves two square
// matrices, the last ones together five
OrthLayout orth_most(int64_t batch, int64_t M, int64_t N, int steps) {
    const int64_t m = M < N ? M : N, n = M < N ? N : M;
    return OrthLayout(batch, M, N, steps > 1 ? 2 : 1,
                      steps > 1 && chain_pays(m, n) ? ozk::kOrthSquares : 2);
}

}  // namespace

extern "C" {

static int grouped_params(ozk::GroupedParams &p, const void *A, int64_t a_stride, const void *B,
                          const int64_t b_strides[3], int64_t T, int64_t K, int64_t N, int64_t G) {
    if (!b_strides) return OZK_ERR_NULL;
    if (!sizes_ok({T, K, N, G})) return OZK_ERR_SHAPE;
    if (b_strides[2] != 1 && b_strides[1] != 1) return OZK_ERR_SHAPE;
    const bool cols = b_strides[2] == 1;
    const int64_t b_pitch = cols ? b_strides[1] : b_strides[2];
    if (b_strides[0] < 0) return OZK_ERR_SHAPE;
    if (int st = stride_status({a_stride, b_pitch})) return st;
    p = {};
    p.A = (const char *)A;
    p.B = (const char *)B;
    p.T = T;
    p.K = K;
    p.N = N;
    p.G = G;
    p.a_pitch = a_stride * 2;
    p.b_group = b_strides[0] * 2;
    p.b_pitch = b_pitch * 2;
    p.b_cols = cols;
    return OZK_OK;
}

int ozk_grouped_matmul_workspace_bytes(const void *A, int64_t a_stride, const void *B,
                                       const int64_t b_strides[3], int64_t T, int64_t K, int64_t N,
                                       int64_t G, size_t *bytes_out) {
    if (!bytes_out) return OZK_ERR_NULL;
    ozk::GroupedParams p;
    if (int st = grouped_params(p, A, a_stride, B, b_strides, T, K, N, G)) return st;
    *bytes_out = ozk::plan_grouped_pack(p).total();
    return OZK_OK;
}

int ozk_grouped_matmul(const void *A, int64_t a_stride, const void *B, const int64_t b_strides[3],
                       const void *offsets, int offset_bytes, int64_t T, int64_t K, int64_t N,
                       int64_t G, int dtype, void *C, int64_t c_stride, void *workspace,
                       size_t workspace_bytes, void *stream) {
    if (!is_half(dtype) || (offset_bytes != 4 && offset_bytes != 8)) return OZK_ERR_DTYPE;
    ozk::GroupedParams p;
    if (int st = grouped_params(p, A, a_stride, B, b_strides, T, K, N, G)) return st;
    if (c_stride < 0) return OZK_ERR_SHAPE;
    if (T == 0 || N == 0) return OZK_OK;
    if (!C || !offsets || (K > 0 && (!A || (G > 0 && !B)))) return OZK_ERR_NULL;
    p.C = (char *)C;
    p.offsets = offsets;
    p.c_pitch = c_stride * 2;
    p.offsets64 = offset_bytes == 8;
    const hipStream_t st = (hipStream_t)stream;
    const ozk::PackedSizes n = ozk::plan_grouped_pack(p);
    if (n.total() && workspace && workspace_bytes >= n.total()) {
        if ((uintptr_t)workspace & 15) return OZK_ERR_WORKSPACE;
        if (hipError_t e = ozk::pack_grouped(p, n, (char *)workspace, st); e != hipSuccess)
            return launched(e);
    }
    return launched(ozk::launch_grouped(p, dtype, st));
}

static int grad_params(ozk::GroupedGradParams &p, const void *A, int64_t a_stride, const void *D,
                       int64_t d_stride, int64_t T, int64_t K, int64_t N, int64_t G) {
    if (!sizes_ok({T, K, N, G})) return OZK_ERR_SHAPE;
    if (int st = stride_status({a_stride, d_stride})) return st;
    p = {};
    p.A = (const char *)A;
    p.D = (const char *)D;
    p.T = T;
    p.K = K;
    p.N = N;
    p.G = G;
    p.a_pitch = a_stride * 2;
    p.d_pitch = d_stride * 2;
    p.splits = ozk::grouped_grad_splits(T, K, N, G);
    return OZK_OK;
}
// the partial sums, in whole 16 bytes, then the copies
static size_t part_bytes(const ozk::GroupedGradParams &p) {
    return p.splits > 1 ? (size_t)round_up((int64_t)p.splits * p.G * p.K * p.N * 4, 16) : 0;
}

int ozk_grouped_matmul_wgrad_workspace_bytes(const void *A, int64_t a_stride, const void *D,
                                             int64_t d_stride, int64_t T, int64_t K, int64_t N,
                                             int64_t G, size_t *bytes_out) {
    if (!bytes_out) return OZK_ERR_NULL;
    ozk::GroupedGradParams p;
    if (int st = grad_params(p, A, a_stride, D, d_stride, T, K, N, G)) return st;
    *bytes_out = part_bytes(p) + ozk::plan_grad_pack(p).total();
    return OZK_OK;
}

int ozk_grouped_matmul_wgrad(const void *A, int64_t a_stride, const void *D, int64_t d_stride,
                             const void *offsets, int offset_bytes, int64_t T, int64_t K,
                             int64_t N, int64_t G, int dtype, void *dB,
                             const int64_t db_strides[2], void *workspace,
                             size_t workspace_bytes, void *stream) {
    if (!is_half(dtype) || (offset_bytes != 4 && offset_bytes != 8)) return OZK_ERR_DTYPE;
    if (!db_strides) return OZK_ERR_NULL;
    ozk::GroupedGradParams p;
    if (int st = grad_params(p, A, a_stride, D, d_stride, T, K, N, G)) return st;
    if (db_strides[0] < 0 || db_strides[1] < 0) return OZK_ERR_SHAPE;
    if (K == 0 || N == 0 || G == 0) return OZK_OK;
    if (!dB || !offsets || (T > 0 && (!A || !D))) return OZK_ERR_NULL;
    const size_t part = part_bytes(p);
    if (part && (!workspace || workspace_bytes < part)) return OZK_ERR_WORKSPACE;
    if (workspace && ((uintptr_t)workspace & 15)) return OZK_ERR_WORKSPACE;
    p.dB = (char *)dB;
    p.offsets = offsets;
    p.db_group = db_strides[0] * 2;
    p.db_pitch = db_strides[1] * 2;
    p.offsets64 = offset_bytes == 8;
    p.part = (float *)workspace;
    const hipStream_t st = (hipStream_t)stream;
    const ozk::PackedSizes n = ozk::plan_grad_pack(p);
    if (n.total() && workspace && workspace_bytes >= part + n.total())
        if (hipError_t e = ozk::pack_grad(p, n, (char *)workspace + part, st); e != hipSuccess)
            return launched(e);
    return launched(ozk::launch_grouped_grad(p, dtype, st));
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
    if (K >= (int64_t)1 << 30) return OZK_ERR_TOO_LARGE;
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
    if (K >= (int64_t)1 << 30) return OZK_ERR_TOO_LARGE;
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
    if (M >= kMaxOrth || N >= kMaxOrth || batch > 65535) return OZK_ERR_TOO_LARGE;
    *bytes_out = batch && M && N ? orth_most(batch, M, N, steps).total : 0;
    return OZK_OK;
}

int ozk_orthogonalize(const void *G, int dtype, int64_t batch, int64_t M, int64_t N,
                      const int64_t g_strides[2], const double *coefficients, int steps,
                      double eps, void *out, const int64_t o_strides[2], void *workspace,
                      size_t workspace_bytes, void *stream) {
    if (!is_float(dtype)) return OZK_ERR_DTYPE;
    if (!sizes_ok({batch, M, N}) || steps < 1 || steps > 64) return OZK_ERR_SHAPE;
    if (M >= kMaxOrth || N >= kMaxOrth || batch > 65535) return OZK_ERR_TOO_LARGE;
    if (!coefficients || !g_strides || !o_strides) return OZK_ERR_NULL;
    if (!batch || !M || !N) return OZK_OK;
    if (!G || !out) return OZK_ERR_NULL;
    if (g_strides[0] < 0 || g_strides[1] < 0 || o_strides[0] < 0 || o_strides[1] < 0)
        return OZK_ERR_SHAPE;
    const OrthLayout at = orth_most(batch, M, N, steps);
    if (!workspace || workspace_bytes < at.total || ((uintptr_t)workspace & 15))
        return OZK_ERR_WORKSPACE;
    ozk::OrthPlan plan;
    plan_orth(plan, M < N ? M : N, M < N ? N : M, coefficients, steps, dtype);
    if (at.sums + plan.xs * at.x + plan.squares * at.a > at.total) return OZK_ERR_WORKSPACE;
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
    p.norms = plan.measured ? (double *)(ws + at.norms) : nullptr;
    p.start_scale = plan.start_scale;
    p.X[0] = ws + at.sums;
    p.X[1] = p.X[0] + (plan.xs > 1 ? at.x : 0);
    for (int i = 0; i < ozk::kOrthSquares; ++i) p.S[i] = p.X[1] + at.x + i * at.a;
    return launched(ozk::launch_orth(p, plan, dtype, (hipStream_t)stream));
}

int ozk_debug_orth_plan(int64_t m, int64_t n, const double *coefficients, int steps, int dtype,
                        int *buffers, float *factors, float *start_scale, int *ops) {
    if (!coefficients || !buffers || !factors || !start_scale || !ops) return OZK_ERR_NULL;
    if (!is_float(dtype)) return OZK_ERR_DTYPE;
    if (m > n || steps < 1 || steps > 64) return OZK_ERR_SHAPE;
    ozk::OrthPlan plan;
    plan_orth(plan, m, n, coefficients, steps, dtype);
    for (int i = 0; i < plan.ops; ++i) {
        const ozk::OrthOp &op = plan.op[i];
        for (int b : {op.kind, op.L, op.R, op.Y, op.D}) *buffers++ = b;
        for (float f : {op.f_acc, op.f_y, op.f_i}) *factors++ = f;
    }
    *start_scale = plan.start_scale;
    *ops = plan.ops;
    return OZK_OK;
}

}  // extern "C"
