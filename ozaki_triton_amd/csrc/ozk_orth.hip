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
// entry leaves fp16's range.
//
// A and B are symmetric: only tiles on and below the diagonal are computed,
// each stored twice.
#include "ozk_linear.h"
#include "ozk_tile.h"

namespace ozk {

// bytes of a slice row of n columns: 64 of h and 64 of l for every 32 columns
__host__ __device__ inline int64_t slice_pitch(int64_t n) { return (n + 31) / 32 * 128; }

template <typename T> OZK_DEV float orth_load(const char *p, int64_t i) {
    if constexpr (sizeof(T) == 4) return ((const float *)p)[i];
    else return from_bits16(((const uint16_t *)p)[i], T{});
}
template <typename T> OZK_DEV void orth_store(char *p, int64_t i, float v) {
    if constexpr (sizeof(T) == 4) ((float *)p)[i] = v;
    else ((uint16_t *)p)[i] = to_bits16(v, T{});
}

OZK_DEV double block_sum(double v) {   // of 256 lanes, in every lane
    __shared__ double part[4];
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    return part[0] + part[1] + part[2] + part[3];
}

// Sums of squares, in fp64 (no overflow, whatever the gradient's scale), of
// the rows blockIdx.x, + blocks, .. of matrix blockIdx.y
template <typename T> __global__ __launch_bounds__(256) void orth_norm_kernel(OrthParams p) {
    const char *G = p.G + (int64_t)blockIdx.y * p.g_batch * (int64_t)sizeof(T);
    double sum = 0.0;
    for (int64_t r = blockIdx.x; r < p.M; r += p.blocks)
        for (int64_t c = threadIdx.x; c < p.N; c += 256) {
            const double v = orth_load<T>(G, r * p.g_row + c);
            sum += v * v;
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

// X0's slices, 32 columns x 64 rows of X a workgroup, transposed through the
// LDS where M > N
template <typename T> __global__ __launch_bounds__(256) void orth_start_kernel(OrthParams p) {
    const bool flip = p.M > p.N;
    const int64_t m = flip ? p.N : p.M, n = flip ? p.M : p.N;
    const int64_t b = blockIdx.z, r0 = (int64_t)blockIdx.y * 64, c0 = (int64_t)blockIdx.x * 32;
    double sum = 0.0;
    for (int i = threadIdx.x; i < p.blocks; i += 256) sum += p.sums[b * p.blocks + i];
    const double f = (double)p.start_scale / (sqrt(block_sum(sum)) + p.eps);
    const char *G = p.G + b * p.g_batch * (int64_t)sizeof(T);
    char *X = p.X[0] + b * m * slice_pitch(n);

    __shared__ float tile[64][33];
#pragma unroll
    for (int q = 0; q < 8; ++q) {
        // consecutive lanes along G's rows
        const int r = flip ? threadIdx.x % 64 : threadIdx.x / 32 + 8 * q;
        const int c = flip ? threadIdx.x / 64 + 4 * q : threadIdx.x % 32;
        const int64_t row = r0 + r, col = c0 + c;
        float v = 0.f;
        if (row < m && col < n)
            v = (float)((double)orth_load<T>(G, flip ? col * p.g_row + row : row * p.g_row + col) * f);
        tile[r][c] = v;
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 8; ++q) {
        const int r = threadIdx.x / 32 + 8 * q, c = threadIdx.x % 32;
        if (r0 + r < m) put_slices(X + (r0 + r) * slice_pitch(n) + c0 * 4 + c * 2, tile[r][c]);
    }
}

enum OrthKind { kOrthA = 0, kOrthB = 1, kOrthX = 2, kOrthLast = 3 };

struct OrthGemm {
    const char *L, *R, *Y;       // left and right operand, what is added (slices)
    char *D;
    int64_t m, n;                // of X
    int64_t l_batch, r_batch, y_batch, d_batch;   // bytes
    int64_t d_row;               // kOrthLast: elements
    float f_y, f_acc;
    int64_t tiles_m, tiles_n;
    uint32_t total;
    int flip;
};

template <typename T, int KIND, typename Sh>
__global__ __launch_bounds__(Sh::THREADS, Sh::PER_SIMD) void orth_gemm_kernel(OrthGemm p) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    constexpr int BM = Sh::BM, BN = Sh::BN;
    constexpr bool kSym = KIND == kOrthA || KIND == kOrthB;
    static_assert(!kSym || BM == BN, "symmetric products run on square tiles");
    const int64_t tile = xcd_tile(blockIdx.x, p.total);
    if (tile < 0) return;
    const uint32_t each = kSym ? (uint32_t)(p.tiles_m * (p.tiles_m + 1) / 2)
                               : (uint32_t)(p.tiles_m * p.tiles_n);
    const uint32_t b = (uint32_t)tile / each, in = (uint32_t)tile - b * each;
    uint32_t tm, tn;
    if (kSym) {
        tm = (uint32_t)((sqrtf(8.f * (float)in + 1.f) - 1.f) * 0.5f);
        while ((uint64_t)tm * (tm + 1) / 2 > in) --tm;
        while ((uint64_t)(tm + 1) * (tm + 2) / 2 <= in) ++tm;
        tm = (uint32_t)uniform((int)tm);
        tn = in - tm * (tm + 1) / 2;
    } else {
        // 8 tile rows at a time, column by column
        const uint32_t first = in / (uint32_t)p.tiles_n / 8 * 8;
        const uint32_t left = (uint32_t)p.tiles_m - first, high = left < 8 ? left : 8;
        const uint32_t at = in - first * (uint32_t)p.tiles_n;
        tn = at / high;
        tm = first + at - tn * high;
    }
    const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BN;
    const int64_t lp = KIND == kOrthA ? slice_pitch(p.n) : slice_pitch(p.m);
    const int64_t rp = KIND == kOrthB ? slice_pitch(p.m) : slice_pitch(p.n);
    const int64_t cols_all = kSym ? p.m : p.n;
    const int rows = (int)(p.m - m0 < BM ? p.m - m0 : BM);
    const int cols = (int)(cols_all - n0 < BN ? cols_all - n0 : BN);

    TileLoop<_Float16, Sh, true> t;
    const char *L = p.L + (int64_t)b * p.l_batch, *R = p.R + (int64_t)b * p.r_batch;
    const TileSrc A = {L + m0 * lp, lp, rows, lp};
    const TileSrc B = Sh::BCOLS ? TileSrc{R + n0 * 4, rp, (int)(rp - n0 * 4 < BN * 4 ? rp - n0 * 4 : BN * 4), p.m}
                                : TileSrc{R + n0 * rp, rp, cols, rp};
    t.run(A, B, smem);

    const int64_t dp = kSym ? slice_pitch(p.m) : slice_pitch(p.n);   // of D's slices
    const int cols_up = (cols + 31) / 32 * 32, rows_up = (rows + 31) / 32 * 32;   // with the zeros
    const char *Y = p.Y + (int64_t)b * p.y_batch;
    char *D = p.D + (int64_t)b * p.d_batch;
    t.each([&](int mi, int ni, f32x4 acc) {
        if (ni >= cols_up) return;
        const int64_t m = m0 + mi, n = n0 + ni;
        float v[4];
        if constexpr (KIND == kOrthA) {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = acc[e] * p.f_acc;
        } else {
            _Float16 h[4] = {0, 0, 0, 0}, l[4] = {0, 0, 0, 0};
            if (mi < rows) {
                const char *at = Y + m * dp + n / 32 * 128 + n % 32 * 2;
                __builtin_memcpy(h, at, 8);
                __builtin_memcpy(l, at + 64, 8);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
                v[e] = __builtin_fmaf(acc[e], p.f_acc, ((float)h[e] + (float)l[e]) * p.f_y);
        }
        if constexpr (KIND == kOrthLast) {
            if (mi >= rows) return;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (ni + e < cols)
                    orth_store<T>(D, p.flip ? (n + e) * p.d_row + m : m * p.d_row + n + e, v[e]);
        } else {
            _Float16 h[4], l[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                h[e] = (_Float16)v[e];
                l[e] = (_Float16)(v[e] - (float)h[e]);
            }
            if (mi < rows) {
                char *at = D + m * dp + n / 32 * 128 + n % 32 * 2;
                __builtin_memcpy(at, h, 8);
                __builtin_memcpy(at + 64, l, 8);
            }
            if (kSym && tm != tn && mi < rows_up) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (ni + e < cols) {
                        char *at = D + (n + e) * dp + m / 32 * 128 + m % 32 * 2;
                        *(_Float16 *)at = h[e];
                        *(_Float16 *)(at + 64) = l[e];
                    }
            }
        }
    });
}

namespace {

template <typename T, int KIND, int BM, int WM, int WN, int NST>
hipError_t orth_gemm(OrthGemm q, int64_t batch, hipStream_t st) {
    using Sh = TileShape<2, false, KIND >= kOrthX, BM, BM, WM, WN, NST>;
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
    const int64_t cols = KIND >= kOrthX ? q.n : q.m;
    auto tiles = [&](int64_t bm) {
        const int64_t tm = (q.m + bm - 1) / bm, tn = (cols + bm - 1) / bm;
        return batch * (KIND >= kOrthX ? tm * tn : tm * (tm + 1) / 2);
    };
    // the largest tile that still gives the CUs enough workgroups; where each has
    // one at most, more stages in flight.  Measured (us, A = X X^T / B X of
    // 2048 x 8192, then of 1024 x 1024, then of 8 matrices 256 x 512):
    //     256 x 256                452 / 200    76 / 84    44 / 38
    //     128 x 128                265 / 200    41 / 44    21 / 16
    //     64 x 64, two stages      168 / 249    23 / 24    11 / 8.4
    //     64 x 64, four stages     205 / 274    16 / 17    10 / 8.1
    if (tiles(256) >= 192) return orth_gemm<T, KIND, 256, 2, 4, 2>(q, batch, st);
    if (tiles(128) >= 256) return orth_gemm<T, KIND, 128, 2, 2, 2>(q, batch, st);
    if (tiles(64) >= 384) return orth_gemm<T, KIND, 64, 2, 2, 2>(q, batch, st);
    return orth_gemm<T, KIND, 64, 2, 2, 4>(q, batch, st);
}

template <typename T>
hipError_t orth_run(const OrthParams &p, const OrthStep *steps, int count, hipStream_t st) {
    const bool flip = p.M > p.N;
    const int64_t m = flip ? p.N : p.M, n = flip ? p.M : p.N;
    const int64_t xb = m * slice_pitch(n), ab = m * slice_pitch(m);
    orth_norm_kernel<T><<<dim3((uint32_t)p.blocks, (uint32_t)p.batch), 256, 0, st>>>(p);
    orth_start_kernel<T><<<dim3((uint32_t)((n + 31) / 32), (uint32_t)((m + 63) / 64),
                                (uint32_t)p.batch), 256, 0, st>>>(p);
    hipError_t e = hipGetLastError();
    OrthGemm q;
    q.m = m;
    q.n = n;
    q.flip = flip;
    q.d_row = p.o_row;
    for (int i = 0; i < count && e == hipSuccess; ++i) {
        const char *X = p.X[i & 1];
        q.L = q.R = q.Y = X;
        q.l_batch = q.r_batch = q.y_batch = xb;
        q.D = p.A;
        q.d_batch = ab;
        q.f_y = 0.f;
        q.f_acc = steps[i].a_acc;
        e = orth_product<T, kOrthA>(q, p.batch, st);
        if (e != hipSuccess) break;
        q.L = q.R = q.Y = p.A;
        q.l_batch = q.r_batch = q.y_batch = ab;
        q.D = p.B;
        q.f_y = steps[i].b_a;
        q.f_acc = steps[i].b_acc;
        e = orth_product<T, kOrthB>(q, p.batch, st);
        if (e != hipSuccess) break;
        q.L = p.B;
        q.R = q.Y = X;
        q.r_batch = q.y_batch = xb;
        q.f_y = steps[i].x_x;
        q.f_acc = steps[i].x_acc;
        if (i + 1 < count) {
            q.D = p.X[(i + 1) & 1];
            q.d_batch = xb;
            e = orth_product<T, kOrthX>(q, p.batch, st);
        } else {
            q.D = p.out;
            q.d_batch = p.o_batch * (int64_t)sizeof(T);
            e = orth_product<T, kOrthLast>(q, p.batch, st);
        }
    }
    return e;
}

}  // namespace

int orth_blocks(int64_t batch, int64_t M, int64_t N) {
    int64_t b = 2048 / (batch > 0 ? batch : 1);
    if (b > M) b = M;
    if (b > M * N / 1024) b = M * N / 1024;
    return (int)(b < 1 ? 1 : b);
}

hipError_t launch_orth(const OrthParams &p, const OrthStep *steps, int count, int dtype,
                       hipStream_t st) {
    if (dtype == 1) return orth_run<float>(p, steps, count, st);
    return dtype == 2 ? orth_run<_Float16>(p, steps, count, st) : orth_run<__bf16>(p, steps, count, st);
}

}  // namespace ozk
