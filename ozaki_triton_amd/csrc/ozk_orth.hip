// ozk_orth.hip -- orthogonalisation of a matrix by Newton-Schulz products.
//
//   X0 = G / (|G|_F + eps);   A = X X^T,  B = b A + c A A,  X <- a X + B X
//
// Each step moves every singular value s of X to s (a + b s^2 + c s^4).  What
// a step rounds, later steps amplify (by a for the smallest singular values),
// so the products are fp32-grade: every matrix is kept as two fp16 slices
// h + l of one power-of-two scale (22 bits), and a product sums the slice
// pairs hh, hl, lh in fp32.  On a Gaussian 512 x 512 matrix and 5 steps the
// result is 2.2e-6 off, as with fp32 products; with one fp16 slice 1.8e-3,
// with bf16 matrices 2.3e-2.  The scales come from the host, which bounds the
// singular values of X, A and B step by step from the coefficients, so no
// entry leaves fp16's range.  Where these bounds grow far past what a matrix does,
// its entries would keep few bits, or none: there B and X are written as fp32
// values, and their slices are those of B / |B|_F and X / |X|_F.
//
// A and B are symmetric: only tiles on and below the diagonal are computed,
// each stored twice.
#include "ozk_linear.h"
#include "ozk_tile.h"

namespace ozk {

// bytes of a slice row of n columns: 64 of h and 64 of l for every 32 columns
__host__ __device__ inline int64_t slice_pitch(int64_t n) { return (n + 31) / 32 * 128; }

OZK_DEV double block_sum(double v) {   // of 256 lanes, in every lane
    __shared__ double part[4];
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    return part[0] + part[1] + part[2] + part[3];
}

// 16 bytes of a row
template <typename T> struct OrthPiece {
    static constexpr int E = 16 / (int)sizeof(T);
    i32x4 raw;
    OZK_DEV float at(int e) const {
        if constexpr (sizeof(T) == 4) return __int_as_float(raw[e]);
        else return from_bits16((uint16_t)((uint32_t)raw[e / 2] >> (16 * (e & 1))), T{});
    }
};
template <typename T> OZK_DEV bool orth_wide(const OrthParams &p, const char *G) {
    return (((uintptr_t)G | (uintptr_t)(p.g_row * (int64_t)sizeof(T))) & 15) == 0;
}

// Sums of squares, in fp64 (no overflow, whatever the gradient's scale), of
// the rows blockIdx.x, + blocks, .. of matrix blockIdx.y.  Bound by its loads,
// 16 bytes a lane where the rows allow (2048 x 8192 bf16: 9 us, 19 one by one)
template <typename T> __global__ __launch_bounds__(256) void orth_norm_kernel(OrthParams p) {
    const char *G = p.G + (int64_t)blockIdx.y * p.g_batch * (int64_t)sizeof(T);
    double sum = 0.0;
    constexpr int E = OrthPiece<T>::E;
    const int64_t whole = orth_wide<T>(p, G) ? p.N / E : 0;   // pieces of a row
    for (int64_t r = blockIdx.x; r < p.M; r += p.blocks) {
        const char *row = G + r * p.g_row * (int64_t)sizeof(T);
#pragma unroll 4
        for (int64_t i = threadIdx.x; i < whole; i += 256) {
            OrthPiece<T> x;
            x.raw = *(const i32x4 *)(row + i * 16);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const double v = x.at(e);
                sum += v * v;
            }
        }
        for (int64_t c = whole * E + threadIdx.x; c < p.N; c += 256) {
            const double v = load_value<T>(row, c);
            sum += v * v;
        }
    }
    sum = block_sum(sum);
    if (threadIdx.x == 0) p.sums[(int64_t)blockIdx.y * p.blocks + blockIdx.x] = sum;
}

OZK_DEV void put_slices(char *at, float v) {
    const _Float16 h = (_Float16)v;
    const _Float16 l = (_Float16)(v - (float)h);
    *(_Float16 *)at = h;
    *(_Float16 *)(at + 64) = l;
}

// X0's slices, 32 columns x 64 rows of X a workgroup: 8 columns a lane where G's
// rows are X's and allow wide loads (2048 x 8192 bf16: 25 us, 38 one by one),
// else through the LDS, which transposes them where M > N.  G is on its way while
// the partial sums are added.
// norm_out: takes the norm, or with `first` a 1 (X0's own, whose norm is 1).
template <typename T>
__global__ __launch_bounds__(256) void orth_start_kernel(OrthParams p, double *norm_out, bool first) {
    const bool flip = p.M > p.N;
    const int64_t m = flip ? p.N : p.M, n = flip ? p.M : p.N;
    const int64_t b = blockIdx.z, r0 = (int64_t)blockIdx.y * 64, c0 = (int64_t)blockIdx.x * 32;
    const char *G = p.G + b * p.g_batch * (int64_t)sizeof(T);
    char *X = p.X[0] + b * m * slice_pitch(n);
    const bool wide = !flip && orth_wide<T>(p, G) && c0 + 32 <= n;

    __shared__ float tile[64][33];
    float v[8];
    if (wide) {
        const int64_t row = r0 + threadIdx.x / 4;
        constexpr int E = OrthPiece<T>::E;
        OrthPiece<T> x[8 / E] = {};
        if (row < m)
#pragma unroll
            for (int i = 0; i < 8 / E; ++i)
                x[i].raw = *(const i32x4 *)(G + (row * p.g_row + c0 + threadIdx.x % 4 * 8 + i * E) *
                                                    (int64_t)sizeof(T));
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = x[e / E].at(e % E);
    } else {
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            // consecutive lanes along G's rows
            const int r = flip ? threadIdx.x % 64 : threadIdx.x / 32 + 8 * q;
            const int c = flip ? threadIdx.x / 64 + 4 * q : threadIdx.x % 32;
            const int64_t row = r0 + r, col = c0 + c;
            v[q] = 0.f;
            if (row < m && col < n) v[q] = load_value<T>(G, flip ? col * p.g_row + row : row * p.g_row + col);
        }
    }
    double sum = 0.0;
    for (int i = threadIdx.x; i < p.blocks; i += 256) sum += p.sums[b * p.blocks + i];
    const double root = sqrt(block_sum(sum)), norm = root + p.eps;
    if (norm_out && blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0)
        norm_out[b] = first ? 1.0 : root;
    const double f = norm == 0.0 ? 0.0 : (double)p.start_scale / norm;   // zero stays zero
#pragma unroll
    for (int q = 0; q < 8; ++q) v[q] = (float)((double)v[q] * f);

    if (wide) {
        const int64_t row = r0 + threadIdx.x / 4;
        if (row >= m) return;
        _Float16 h[8], l[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            h[e] = (_Float16)v[e];
            l[e] = (_Float16)(v[e] - (float)h[e]);
        }
        i32x4 u[2];
        __builtin_memcpy(&u[0], h, 16);
        __builtin_memcpy(&u[1], l, 16);
        char *to = X + row * slice_pitch(n) + c0 * 4 + threadIdx.x % 4 * 16;
        *(i32x4 *)to = u[0];
        *(i32x4 *)(to + 64) = u[1];
        return;
    }
#pragma unroll
    for (int q = 0; q < 8; ++q) {
        const int r = flip ? threadIdx.x % 64 : threadIdx.x / 32 + 8 * q;
        const int c = flip ? threadIdx.x / 64 + 4 * q : threadIdx.x % 32;
        tile[r][c] = v[q];
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 8; ++q) {
        const int r = threadIdx.x / 32 + 8 * q, c = threadIdx.x % 32;
        if (r0 + r < m) put_slices(X + (r0 + r) * slice_pitch(n) + c0 * 4 + c * 2, tile[r][c]);
    }
}

struct OrthGemm {
    const char *L, *R, *Y;       // left and right operand, what is added or null
    char *D;
    int64_t m, n;                // of X
    int64_t l_batch, r_batch, y_batch, d_batch;   // bytes
    int64_t d_row;               // kOrthLast: elements
    float f_acc, f_y, f_i;
    const double *norm_x, *norm_b;   // kOrthLast: the slices' measured scales, or null
    int64_t tiles_m, tiles_n;
    uint32_t total;
    int flip;
};

// the largest r with r (r + 1) / 2 <= t
OZK_DEV uint32_t triangle_row(uint32_t t) {
    uint32_t r = (uint32_t)((sqrtf(8.f * (float)t + 1.f) - 1.f) * 0.5f);
    while ((uint64_t)r * (r + 1) / 2 > t) --r;
    while ((uint64_t)(r + 1) * (r + 2) / 2 <= t) ++r;
    return (uint32_t)uniform((int)r);
}

OZK_DEV i32x2 pack_half(const _Float16 (&v)[4]) {
    i32x2 u;
    __builtin_memcpy(&u, v, 8);
    return u;
}

template <typename T, int KIND, typename Sh>
__global__ __launch_bounds__(Sh::THREADS, Sh::PER_SIMD) void orth_gemm_kernel(OrthGemm p) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    constexpr int BM = Sh::BM, BN = Sh::BN;
    constexpr bool kSym = KIND == kOrthXX || KIND == kOrthSym;
    static_assert(!kSym || BM == BN, "symmetric products run on square tiles");
    const int64_t tile = xcd_tile(blockIdx.x, p.total);
    if (tile < 0) return;
    const uint32_t each = kSym ? (uint32_t)(p.tiles_m * (p.tiles_m + 1) / 2)
                               : (uint32_t)(p.tiles_m * p.tiles_n);
    const uint32_t b = (uint32_t)tile / each, in = (uint32_t)tile - b * each;
    uint32_t tm, tn;
    if (kSym) {
        // on and below the diagonal, in blocks of 512 x 512 (row of blocks by row
        // of blocks, inside one column by column): an XCD's workgroups share the
        // rows of a block, not those of a whole row of tiles
        constexpr uint32_t SB = 512 / BM;
        const uint32_t r0 = triangle_row(in) / SB * SB, rest = in - r0 * (r0 + 1) / 2;
        const uint32_t left = (uint32_t)p.tiles_m - r0, h = left < SB ? left : SB;
        const uint32_t J = rest / (h * SB) * SB;
        if (J < r0) {
            const uint32_t t = rest - J * h;
            tn = J + t / h;
            tm = r0 + t - (t / h) * h;
        } else {
            const uint32_t t = rest - r0 * h, r = triangle_row(t);
            tm = r0 + r;
            tn = r0 + t - r * (r + 1) / 2;
        }
    } else {
        // 8 tile rows at a time, column by column
        const uint32_t first = in / (uint32_t)p.tiles_n / 8 * 8;
        const uint32_t left = (uint32_t)p.tiles_m - first, high = left < 8 ? left : 8;
        const uint32_t at = in - first * (uint32_t)p.tiles_n;
        tn = at / high;
        tm = first + at - tn * high;
    }
    const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BN;
    const int64_t lp = KIND == kOrthXX ? slice_pitch(p.n) : slice_pitch(p.m);
    const int64_t rp = KIND == kOrthSym ? slice_pitch(p.m) : slice_pitch(p.n);
    const int64_t cols_all = kSym ? p.m : p.n;
    const int rows = (int)(p.m - m0 < BM ? p.m - m0 : BM);
    const int cols = (int)(cols_all - n0 < BN ? cols_all - n0 : BN);

    TileLoop<_Float16, Sh, true> t;
    const char *L = p.L + (int64_t)b * p.l_batch, *R = p.R + (int64_t)b * p.r_batch;
    const TileSrc A = {L + m0 * lp, lp, rows, lp, L};
    const int row = (int)(rp - n0 * 4 < BN * 4 ? rp - n0 * 4 : BN * 4);
    const TileSrc B = Sh::BCOLS ? TileSrc{R + n0 * 4, rp, row, p.m, R}
                                : TileSrc{R + n0 * rp, rp, cols, rp, R};
    if (!t.run(A, B, smem)) return;

    const int64_t dp = kSym ? slice_pitch(p.m) : slice_pitch(p.n);   // of D's and Y's slices
    const int cols_up = (cols + 31) / 32 * 32, rows_up = (rows + 31) / 32 * 32;   // with the zeros
    const char *Y = p.Y ? p.Y + (int64_t)b * p.y_batch : nullptr;
    char *D = p.D + (int64_t)b * p.d_batch;
    const int g = (threadIdx.x >> 4) & 3, q = threadIdx.x & 3;
    const bool diagonal = KIND == kOrthSym && tm == tn && p.f_i != 0.f;
    float f_acc = p.f_acc, f_y = p.f_y;
    if (KIND == kOrthLast && p.norm_x) {
        const double x = p.norm_x[b];
        if (p.norm_b) {        // of B and X, and of X
            f_acc = (float)(f_acc * p.norm_b[b] * x);
            f_y = (float)(f_y * x);
        } else {               // of A twice, and of A
            f_acc = (float)(f_acc * x * x * x * x);
            f_y = (float)(f_y * x * x);
        }
    }
    // 32 columns at a time: a line of D's slices
    t.each_pair([&](int mi, int ni, f32x4 lo, f32x4 hi) {
        const int n32 = ni - 4 * g;
        if (n32 >= cols_up) return;
        const int64_t m = m0 + mi, n = n0 + ni;
        const int64_t line = m * dp + (n0 + n32) * 4;
        float v[2][4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[0][e] = lo[e] * f_acc;
            v[1][e] = hi[e] * f_acc;
        }
        if (KIND != kOrthXX && Y) {
            i32x4 y[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
            if (mi < rows) {
                y[0] = *(const i32x4 *)(Y + line + pair_column(g) * 2);
                y[1] = *(const i32x4 *)(Y + line + pair_column(g) * 2 + 64);
            }
            i32x2 h[2], l[2];
            split_pair(y[0], h[0], h[1]);
            split_pair(y[1], l[0], l[1]);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                _Float16 hv[4], lv[4];
                __builtin_memcpy(hv, &h[u], 8);
                __builtin_memcpy(lv, &l[u], 8);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[u][e] += ((float)hv[e] + (float)lv[e]) * f_y;
            }
        }
        if (diagonal)
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (mi == ni + 16 * u + e && mi < rows) v[u][e] += p.f_i;
        if constexpr (KIND == kOrthLast) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int c = ni + 16 * u;
                if constexpr (sizeof(T) == 2) {
                    uint16_t e[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) e[i] = to_bits16(v[u][i], T{});
                    i32x2 w;
                    __builtin_memcpy(&w, e, 8);
                    int64_t at = m * p.d_row + n0 + c;
                    bool whole = mi < rows && c + 4 <= cols;
                    if (p.flip) {
                        // four rows of the result, four of its columns
                        w = transpose_quad(w);
                        __builtin_memcpy(e, &w, 8);
                        at = (n0 + c + q) * p.d_row + m - q;
                        whole = mi - q + 4 <= rows && c + q < cols;
                    }
                    char *to = D + at * 2;
                    if (whole && ((uintptr_t)to & 7) == 0) {
                        *(i32x2 *)to = w;
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (p.flip ? mi - q + i < rows && c + q < cols : mi < rows && c + i < cols)
                                ((uint16_t *)to)[i] = e[i];
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (mi < rows && c + i < cols)
                            ((float *)D)[p.flip ? (n0 + c + i) * p.d_row + m
                                                : m * p.d_row + n0 + c + i] = v[u][i];
                }
            }
        } else {
            i32x2 h[2], l[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                _Float16 hv[4], lv[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    hv[e] = (_Float16)v[u][e];
                    lv[e] = (_Float16)(v[u][e] - (float)hv[e]);
                }
                h[u] = pack_half(hv);
                l[u] = pack_half(lv);
            }
            const i32x4 hj = join_pair(h[0], h[1]), lj = join_pair(l[0], l[1]);
            if (mi < rows) {
                char *to = D + line + pair_column(g) * 2;
                *(i32x4 *)to = hj;
                *(i32x4 *)(to + 64) = lj;
            }
            if (kSym && tm != tn) {
                // the mirrored tile: four lanes' values of a column, a row there
                const int m4 = mi - q;
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const i32x2 ht = transpose_quad(h[u]), lt = transpose_quad(l[u]);
                    if (m4 < rows_up && ni + 16 * u + q < cols) {
                        char *to = D + (n + 16 * u + q) * dp + (m0 + m4) / 32 * 128 + (m0 + m4) % 32 * 2;
                        *(i32x2 *)to = ht;
                        *(i32x2 *)(to + 64) = lt;
                    }
                }
            }
        }
    });
}

namespace {

template <typename T, int KIND, int BM, int WM, int WN, int NST, int KW = 1>
hipError_t orth_gemm(OrthGemm q, int64_t batch, hipStream_t st) {
    using Sh = TileShape<2, false, KIND >= kOrthX, BM, BM, WM, WN, NST, KW>;
    q.tiles_m = (q.m + BM - 1) / BM;
    q.tiles_n = ((KIND >= kOrthX ? q.n : q.m) + BM - 1) / BM;
    const int64_t tiles = batch * (KIND >= kOrthX ? q.tiles_m * q.tiles_n
                                                  : q.tiles_m * (q.tiles_m + 1) / 2);
    if (tiles >= (int64_t)1 << 31) return hipErrorInvalidConfiguration;
    q.total = (uint32_t)tiles;
    if (hipError_t e = allow_lds<&orth_gemm_kernel<T, KIND, Sh>>(Sh::LDS_BYTES); e != hipSuccess)
        return e;
    orth_gemm_kernel<T, KIND, Sh><<<dim3((uint32_t)((tiles + 7) / 8 * 8)), Sh::THREADS,
                                    Sh::LDS_BYTES, st>>>(q);
    return hipGetLastError();
}

template <typename T, int KIND>
hipError_t orth_product(const OrthGemm &q, int64_t batch, hipStream_t st) {
    // A CU has one workgroup, whatever the tile: the tile is the one whose rounds of
    // workgroups over the 256 CUs take the shortest.  A round takes (us, K in 1024s,
    // fitted to what follows; R by rows / by columns):
    //     256 x 256, 8 waves               31 + 46 K / 31 + 60 K
    //     128 x 128, 2 x 8 waves           16 + 15 K / 12 + 18 K
    //     96 x 96, 2 x 6 waves, 3 stages   11 + 12 K /  4 + 15 K (never the shortest)
    //     64 x 64, 2 x 4 waves, 4 stages    7 +  5 K /  3 +  7 K
    // Measured (us, X X^T / A A / B X of 2048 x 8192, then of 1400 x 2000, of two
    // 1024 x 4096, of 8 matrices 512 x 1024, of 8 256 x 512):
    //     256   424 / 129 / 165     - /  - /  -     - /  - /  -     - /  - /  -    44 /  36 /  38
    //     128   141 /  46 / 195     - /  - / 33    72 / 34 / 59    25 / 19 / 19    17 /  14 /  11
    //     96    109 /  35 / 275    26 / 22 / 44    47 / 19 / 77    18 / 14 / 33     - /   - /   -
    //     64    155 /  52 / 280    20 / 18 / 41    53 / 22 / 82    20 / 16 / 29   8.8 / 7.2 / 7.6
    // (A A of 2048 in tiles of 96 with two stages: 41 us, in one group of waves 38)
    constexpr bool cols = KIND >= kOrthX;
    const double k = (double)(KIND == kOrthXX ? q.n : q.m) / 1024;
    auto time = [&](int64_t bm, double fixed, double slope) {
        const int64_t tm = (q.m + bm - 1) / bm, tn = ((cols ? q.n : q.m) + bm - 1) / bm;
        const int64_t tiles = batch * (cols ? tm * tn : tm * (tm + 1) / 2);
        return (double)((tiles + 255) / 256) * (fixed + slope * k);
    };
    const double t256 = cols ? time(256, 31, 60) : time(256, 31, 46);
    const double t128 = cols ? time(128, 12, 18) : time(128, 16, 15);
    const double t64 = cols ? time(64, 3, 7) : time(64, 7, 5);
    if constexpr (!cols) {
        const double t96 = time(96, 11, 12);
        if (t96 < t256 && t96 < t128 && t96 < t64)
            return orth_gemm<T, KIND, 96, 2, 3, 3, 2>(q, batch, st);
    }
    if (t256 <= t128 && t256 <= t64) return orth_gemm<T, KIND, 256, 2, 4, 2>(q, batch, st);
    if (t128 <= t64) return orth_gemm<T, KIND, 128, 2, 4, 2, 2>(q, batch, st);
    return orth_gemm<T, KIND, 64, 2, 2, 4, 2>(q, batch, st);
}

// p.G's slices over its norm into p.X[0]
template <typename T>
hipError_t orth_slices(const OrthParams &p, double *norm_out, bool first, hipStream_t st) {
    const int64_t m = p.M > p.N ? p.N : p.M, n = p.M > p.N ? p.M : p.N;
    orth_norm_kernel<T><<<dim3((uint32_t)p.blocks, (uint32_t)p.batch), 256, 0, st>>>(p);
    orth_start_kernel<T><<<dim3((uint32_t)((n + 31) / 32), (uint32_t)((m + 63) / 64),
                                (uint32_t)p.batch), 256, 0, st>>>(p, norm_out, first);
    return hipGetLastError();
}

// A product into `fp32` [m, n], and from there its slices over its norm, which
// goes to norm_out, into `to`.  (The partial sums have room: orth_blocks grows
// with either side.)
hipError_t orth_measured(const OrthParams &p, OrthGemm q, char *fp32, char *to, double *norm_out,
                         hipStream_t st) {
    q.flip = 0;
    q.D = fp32;
    q.d_batch = q.m * slice_pitch(q.n);
    q.d_row = slice_pitch(q.n) / 4;
    if (hipError_t e = orth_product<float, kOrthLast>(q, p.batch, st); e != hipSuccess) return e;
    OrthParams s = p;
    s.G = fp32;
    s.M = q.m;
    s.N = q.n;
    s.g_batch = q.d_batch / 4;
    s.g_row = q.d_row;
    s.eps = 0;
    s.blocks = orth_blocks(p.batch, q.m, q.n);
    s.X[0] = to;
    return orth_slices<float>(s, norm_out, false, st);
}

template <typename T>
hipError_t orth_run(const OrthParams &p, const OrthPlan &plan, hipStream_t st) {
    const bool flip = p.M > p.N;
    const int64_t m = flip ? p.N : p.M, n = flip ? p.M : p.N;
    const int64_t xb = m * slice_pitch(n), ab = m * slice_pitch(m);
    double *norm_x = p.norms, *norm_b = p.norms ? p.norms + p.batch : nullptr;
    hipError_t e = orth_slices<T>(p, norm_x, true, st);
    auto buffer = [&](int id, int64_t &bytes) -> char * {
        bytes = id >= 0 ? ab : xb;
        return id >= 0 ? p.S[id] : id >= -2 ? p.X[-1 - id] : nullptr;
    };
    for (int i = 0; i < plan.ops && e == hipSuccess; ++i) {
        const OrthOp &op = plan.op[i];
        OrthGemm q;
        q.m = m;
        q.n = n;
        q.flip = flip;
        q.d_row = p.o_row;
        q.f_acc = op.f_acc;
        q.f_y = op.f_y;
        q.f_i = op.f_i;
        q.norm_x = norm_x;
        q.norm_b = norm_b;
        q.L = buffer(op.L, q.l_batch);
        q.R = buffer(op.R, q.r_batch);
        q.Y = buffer(op.Y, q.y_batch);
        q.D = buffer(op.D, q.d_batch);
        switch (op.kind) {
        case kOrthXX: e = orth_product<T, kOrthXX>(q, p.batch, st); break;
        case kOrthSym: e = orth_product<T, kOrthSym>(q, p.batch, st); break;
        case kOrthX: e = orth_product<T, kOrthX>(q, p.batch, st); break;
        case kOrthNewB:
            q.n = m;
            q.norm_b = nullptr;
            e = orth_measured(p, q, p.S[1], q.D, norm_b, st);
            break;
        case kOrthNewX: e = orth_measured(p, q, p.X[1], q.D, norm_x, st); break;
        default:
            q.D = p.out;
            q.d_batch = p.o_batch * (int64_t)sizeof(T);
            e = orth_product<T, kOrthLast>(q, p.batch, st);
        }
    }
    return e;
}

}  // namespace

// Partial sums of a matrix; each workgroup of the next kernel adds all of them
// (2048 x 8192 bf16: with 2048 of them it takes 32 us, with 512 25)
int orth_blocks(int64_t batch, int64_t M, int64_t N) {
    int64_t b = 512 / (batch > 0 ? batch : 1);
    if (b > M) b = M;
    if (b > M * N / 1024) b = M * N / 1024;
    return (int)(b < 1 ? 1 : b);
}

hipError_t launch_orth(const OrthParams &p, const OrthPlan &plan, int dtype, hipStream_t st) {
    if (dtype == 1) return orth_run<float>(p, plan, st);
    return dtype == 2 ? orth_run<_Float16>(p, plan, st) : orth_run<__bf16>(p, plan, st);
}

}  // namespace ozk
