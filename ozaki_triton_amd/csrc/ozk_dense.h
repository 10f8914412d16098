// ozk_dense.h -- the product of a linear layer, y = act(x W^T + b) + r, and
// what its gradients need beside products.  Part of the unit of the grouped
// products (ozk_grouped.hip), whose tiles and copies it shares: included there, and
// nowhere else.
//
// Three kernels compute the sums: tiles on the matrix cores (ozk_tile.h) with
// the epilogue in them, the same with K cut into ranges whose fp32 sums a second
// launch joins, and one for a few rows, which is bound by reading W.
#pragma once

#include "../../include/ozaki_amd.h"
#include "ozk_train.h"
#include "ozk_tile.h"

namespace ozk {

// ---------------------------------------------------------------------------
// Activations.  Results are rounded to 8 or 11 bits: exp2 and the reciprocal of the
// hardware (1 ulp each) and the roundings of exp2's argument stay far below that.  The
// latter are worth 2^-24 of the argument's size each, which grows with z in silu, with
// z^2 in gelu and z^3 in gelu_tanh: up to 7e-6, 8e-6 and 1.7e-5 of the smallest normal
// results (fp32 steps against 64 bits, 2e6 values of z each).
// ---------------------------------------------------------------------------
constexpr float kLog2e = 1.44269504f, kGelu2 = 1.59576912f /* 2 sqrt(2 / pi) */, kGelu3 = 0.044715f;

// Far below 0 the exponentials leave fp32's normal range, where exp2 and the reciprocal
// give 0, before the results do (bf16 has that range, too; silu(-88) is -5.3e-37): they
// are 2^64 times as large there, and the results brought back last.
struct Scaled {
    float v, by;   // v * by, by 1 or 2^-64
};
template <bool FAR = true> OZK_DEV Scaled sigmoid(float z) {   // 1 / (1 + e^-z); FAR: of any z
    const float t = -kLog2e * z;
    const bool far = FAR && t > 96.f;
    return {__builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(far ? t - 64.f : t)), far ? 0x1p-64f : 1.f};
}
// Phi(-a) of the normal distribution for a = |z| is e^(-a a / 2) times something
// smooth, here a polynomial in t = 1 / (1 + 0.3 a) fitted to it over 0 .. 14 (beyond,
// e^(-a a / 2) is below every result): relative error 2.2e-6 in fp32.  The
// coefficients are a weighted least-squares fit to 0.5 erfcx(a / sqrt 2).
OZK_DEV float tail_factor(float z) {
    const float t = __builtin_amdgcn_rcpf(fmaf(0.3f, fabsf(z), 1.f));
    float q = -0.08459325134754181f;
    q = fmaf(q, t, 0.24057289958000183f);
    q = fmaf(q, t, -0.048644598573446274f);
    q = fmaf(q, t, 0.1647646278142929f);
    q = fmaf(q, t, 0.1067044585943222f);
    q = fmaf(q, t, 0.12127471715211868f);
    return fmaf(q, t, -7.979064685059711e-05f);
}
// (gelu itself: where e^(-z z / 2) is 0 here it is below 2^-127; its derivative is not)
OZK_DEV float gauss(float z) { return __builtin_amdgcn_exp2f(-0.5f * kLog2e * z * z); }
OZK_DEV Scaled gauss_scaled(float z) {
    const float t = -0.5f * kLog2e * z * z;
    const bool far = t < -96.f;
    return {__builtin_amdgcn_exp2f(far ? t + 64.f : t), far ? 0x1p-64f : 1.f};
}
// |z| and z within 1e4, where every formula below has reached its limit and no
// infinity is left to be multiplied with 0; a NaN is carried by the other factors
OZK_DEV float near_abs(float z) { return fminf(fabsf(z), 1e4f); }
OZK_DEV float near(float z) { return __builtin_amdgcn_fmed3f(z, -1e4f, 1e4f); }

// FAR: of any z; else of z from far_below on, with the same bits
template <int ACT> constexpr float far_below = ACT == OZK_ACT_SILU ? -64.f : -9.f;   // sigmoid's t < 96 behind it
template <int ACT, bool FAR> OZK_DEV float activation(float z) {
    if constexpr (ACT == OZK_ACT_RELU) return z < 0.f ? 0.f : z;   // NaN stays
    if constexpr (ACT == OZK_ACT_SILU) {
        const Scaled s = sigmoid<FAR>(z);
        return z * s.v * s.by;
    }
    if constexpr (ACT == OZK_ACT_GELU_TANH) {   // (1 + tanh u) / 2 = sigmoid(2u)
        const Scaled s = sigmoid<FAR>(kGelu2 * fmaf(kGelu3 * z * z, z, z));
        return z * s.v * s.by;
    }
    if constexpr (ACT == OZK_ACT_GELU)                             // z Phi(z)
        return fmaf(-near_abs(z), tail_factor(z) * gauss(z), fmaxf(z, 0.f));
    return z;
}
// Its derivative.  1 - s of a sigmoid s is off by 2^-24, which its factors leave far
// below dy's own rounding.
template <int ACT> OZK_DEV float derivative(float z) {
    if constexpr (ACT == OZK_ACT_RELU) return z > 0.f ? 1.f : z <= 0.f ? 0.f : z;   // NaN stays
    if constexpr (ACT == OZK_ACT_SILU) {
        const Scaled s = sigmoid(z);
        return s.v * fmaf(near(z), 1.f - s.v * s.by, 1.f) * s.by;
    }
    if constexpr (ACT == OZK_ACT_GELU_TANH) {
        const float c = near(z), zz = kGelu3 * c * c;
        const Scaled s = sigmoid(kGelu2 * fmaf(zz, z, z));
        return s.v * fmaf(c * (1.f - s.v * s.by), kGelu2 * fmaf(3.f, zz, 1.f), 1.f) * s.by;
    }
    if constexpr (ACT == OZK_ACT_GELU) {   // Phi(z) + z phi(z): d below 0, 1 - d above
        const Scaled s = gauss_scaled(z);
        const float d = s.v * fmaf(-0.398942280f, near_abs(z), tail_factor(z)) * s.by;
        return z < 0.f ? d : 1.f - d;
    }
    return 1.f;
}
template <typename F> OZK_DEV void with_act(int act, F &&f) {
    switch (act) {
    case OZK_ACT_RELU: f(std::integral_constant<int, OZK_ACT_RELU>{}); break;
    case OZK_ACT_GELU: f(std::integral_constant<int, OZK_ACT_GELU>{}); break;
    case OZK_ACT_GELU_TANH: f(std::integral_constant<int, OZK_ACT_GELU_TANH>{}); break;
    case OZK_ACT_SILU: f(std::integral_constant<int, OZK_ACT_SILU>{}); break;
    default: break;
    }
}

// ---------------------------------------------------------------------------
// 8 consecutive 16-bit values of a row, of which `n` exist
// ---------------------------------------------------------------------------
typedef int i32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef int i32x4_words __attribute__((ext_vector_type(4), aligned(4)));
OZK_DEV i32x4 load8(const char *p, int n) {
    i32x4 v = {0, 0, 0, 0};
    if (n >= 8) {
        __builtin_memcpy(&v, p, 16);   // of any alignment
    } else {
#pragma unroll 1
        for (int i = n - 1; i >= 0; --i) push16(v, ((const uint16_t *)p)[i]);
    }
    return v;
}
// all 8, past the caches: read once, and what is written meanwhile is read again soon
OZK_DEV i32x4 load8_once(const char *p) { return __builtin_nontemporal_load((const i32x4_any *)p); }
OZK_DEV void store8(char *p, int n, i32x4 v) {
    if (n >= 8) {
        __builtin_memcpy(p, &v, 16);
    } else {
#pragma unroll 1
        for (int i = 0; i < n; ++i) {
            ((uint16_t *)p)[i] = (uint16_t)v.x;
            v = i32x4{(int)__builtin_amdgcn_alignbit((uint32_t)v.y, (uint32_t)v.x, 16),
                      (int)__builtin_amdgcn_alignbit((uint32_t)v.z, (uint32_t)v.y, 16),
                      (int)__builtin_amdgcn_alignbit((uint32_t)v.w, (uint32_t)v.z, 16),
                      (int)((uint32_t)v.w >> 16)};
        }
    }
}
template <typename ST> OZK_DEV void unpack8(i32x4 v, float (&f)[8]) {
    uint16_t e[8];
    __builtin_memcpy(e, &v, 16);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = from_bits16(e[i], ST{});
}
template <typename ST> OZK_DEV i32x4 pack8(const float (&f)[8]) {
    uint16_t e[8];
    i32x4 v;
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = to_bits16(f[i], ST{});
    __builtin_memcpy(&v, e, 16);
    return v;
}

// The epilogue of 8 sums of row m from column n on, `left` columns to N
template <typename ST>
OZK_DEV void finish8(const DenseParams &p, float (&v)[8], const float (&bias)[8], i32x4 res,
                     int64_t m, int64_t n, int left) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] += bias[i];
    if (p.Z) {
        // z is kept in 16 bits for the backward pass: act' moves by at most 0.32 2^-9
        // (bf16) with it, as much as dy's own rounding.  Where relu's side depends on
        // it, a z that underflows keeps its own.
        i32x4 z = pack8<ST>(v);
        if (p.act == OZK_ACT_RELU) {
            uint16_t e[8];
            __builtin_memcpy(e, &z, 16);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if ((e[i] & 0x7FFF) == 0 && v[i] != 0.f) e[i] |= 1;
            __builtin_memcpy(&z, e, 16);
        }
        char *to = p.Z + (m * p.N + n) * 2;
        if (left == 8) __builtin_nontemporal_store((i32x4_any)z, (i32x4_any *)to);   // not read soon
        else store8(to, left, z);
    }
    with_act(p.act, [&](auto act) {
        constexpr int ACT = decltype(act)::value;
        if constexpr (ACT == OZK_ACT_SILU || ACT == OZK_ACT_GELU_TANH) {
            // hardly ever; always, it costs (4096 x 4096 x 1024, tanh gelu) 1.1 us of 40
            float least = v[0];
#pragma unroll
            for (int i = 1; i < 8; ++i) least = fminf(least, v[i]);
            if (least < far_below<ACT>) {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = activation<ACT, true>(v[i]);
                return;
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = activation<ACT, false>(v[i]);
    });
    if (p.res) {
        float r[8];
        unpack8<ST>(res, r);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += r[i];
    }
    store8(p.C + m * p.c_pitch + n * 2, left, pack8<ST>(v));
}
template <typename ST>
OZK_DEV void bias_at(const DenseParams &p, int64_t n, int left, float (&bias)[8]) {
    unpack8<ST>(p.bias && left > 0 ? load8(p.bias + n * 2, left) : i32x4{0, 0, 0, 0}, bias);
}
template <typename ST>
OZK_DEV i32x4 res_at(const DenseParams &p, int64_t m, int64_t n, int left) {
    return p.res ? load8(p.res + m * p.r_pitch + n * 2, left) : i32x4{0, 0, 0, 0};
}

// A wave's part of a tile through the LDS, so that a lane has 8 columns of a row:
// the epilogue's code is there once, not once per accumulator (128 values a lane
// in the largest tile), its columns' bias stays in registers, and residual, Z and
// C are read and written in whole lines.
template <typename ST, typename Sh, typename Loop>
OZK_DEV void finish_tile(const Loop &t, const DenseParams &p, char *smem, int64_t m0, int64_t n0) {
    constexpr int MI = Sh::MI, NI = Sh::NI, CHUNKS = NI * 4;   // 16-byte pieces of an LDS row
    constexpr int ROOM = Sh::LDS_BYTES / Sh::WAVES / (NI * 1024);
    constexpr auto most = [](int room) {
        int c = MI < room ? MI : room;
        while (MI % c) --c;
        return c;
    };
    constexpr int CI = most(ROOM);          // blocks of 16 rows at a time
    constexpr int LANES = NI * 2, RPI = 64 / LANES;   // lanes of a row, rows of a wave's step
    static_assert(ROOM >= 1 && (NI == 1 || NI == 2 || NI == 4) && CI * 16 >= RPI, "");
    const int lane = threadIdx.x & 63, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    m0 += wave / Sh::WN * MI * 16;
    n0 += wave % Sh::WN * NI * 16 + lane % LANES * 8;
    const int64_t over = p.N - n0;
    const int left = over < 8 ? (int)(over < 0 ? 0 : over) : 8;
    float bias[8];
    bias_at<ST>(p, n0, left, bias);
    f32x4 *buf = (f32x4 *)(smem + wave * CI * NI * 1024);
    // 16-byte pieces XORed with the row: neither the writes (16 rows of one column)
    // nor the reads (8 lanes to 256 bytes) meet in a bank
    auto at = [&](int row, int chunk) {
        const int x = NI == 4 ? row & 15 : NI == 2 ? (row >> 1) & 7 : (row >> 2) & 3;
        return row * CHUNKS + (chunk ^ x);
    };
    auto settle = [] {   // LDS writes of the other lanes before reads, and back
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    };
#pragma unroll
    for (int c = 0; c < MI / CI; ++c) {
        if (c) settle();
#pragma unroll
        for (int i = 0; i < CI; ++i)
#pragma unroll
            for (int j = 0; j < NI; ++j)
                buf[at(i * 16 + (lane & 15), j * 4 + g)] = t.acc[c * CI + i][j];
        settle();
#pragma unroll 2
        for (int r = 0; r < CI * 16; r += RPI) {
            const int row = r + lane / LANES;
            const int64_t m = m0 + c * CI * 16 + row;
            const f32x4 lo = buf[at(row, lane % LANES * 2)], hi = buf[at(row, lane % LANES * 2 + 1)];
            if (m < p.M && left > 0) {
                float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
                finish8<ST>(p, v, bias, res_at<ST>(p, m, n0, left), m, n0, left);
            }
        }
    }
}

// db for 16 columns: the partial sums' rows over groups of 16 lanes, added in 64 bits
template <typename ST> OZK_DEV void add_bias(const DenseParams &p, int64_t block, int threads, double (*join)[16]) {
    const int64_t c = block * 16 + threadIdx.x % 16;
    const int groups = threads / 16, of = threadIdx.x / 16;   // 32 groups at most
    double v = 0.0;
    if (c < p.db_n)
#pragma unroll 4
        for (int64_t b = of; b < p.db_blocks; b += groups) v += (double)p.sums[b * p.db_n + c];
    join[of][threadIdx.x % 16] = v;
    __syncthreads();
    if (threadIdx.x < 16 && c < p.db_n) {
        v = 0.0;
        for (int i = 0; i < groups; ++i) v += join[i][threadIdx.x];
        store_value<ST>(p.db, c, (float)v);
    }
}

template <typename ST, typename Sh, bool DMA>
__global__ __launch_bounds__(Sh::THREADS, Sh::PER_SIMD) void dense_kernel(DenseParams p) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    constexpr int BM = Sh::BM, BN = Sh::BN;
    const uint32_t tiles_m = (uint32_t)((p.M + BM - 1) / BM), tiles_n = (uint32_t)((p.N + BN - 1) / BN);
    const uint32_t each = tiles_m * tiles_n;
    if constexpr (Sh::ACOLS) {   // a weight's gradient: the bias' with it
        const uint32_t own = (each * (uint32_t)p.splits + 7) / 8 * 8;
        if (blockIdx.x >= own) {
            add_bias<ST>(p, blockIdx.x - own, Sh::THREADS, (double(*)[16])smem);
            return;
        }
    }
    const int64_t tile = xcd_tile(blockIdx.x, each * (uint32_t)p.splits);
    if (tile < 0) return;
    // 8 tile rows at a time, column by column: the workgroups of an XCD share a
    // square block of both operands in its L2
    const uint32_t s = (uint32_t)tile / each, in = (uint32_t)tile - s * each;
    const uint32_t first = in / tiles_n / 8 * 8;
    const uint32_t high = tiles_m - first < 8 ? tiles_m - first : 8, ahead = in - first * tiles_n;
    const uint32_t tn = ahead / high, tm = first + ahead - tn * high;
    const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BN;
    const int rows = (int)(p.M - m0 < BM ? p.M - m0 : BM);
    const int cols = (int)(p.N - n0 < BN ? p.N - n0 : BN);
    // the s-th range of K, whole stages each
    int64_t k0 = 0, k1 = p.K;
    if (p.splits > 1) {
        const int64_t stages = (p.K + Sh::KS - 1) / Sh::KS;
        const int64_t per = (stages + p.splits - 1) / p.splits * Sh::KS;
        k0 = per * s < p.K ? per * s : p.K;
        k1 = p.K - k0 < per ? p.K : k0 + per;
    }
    auto bytes = [](int64_t n, bool padded) { return padded ? (n + 7) / 8 * 16 : n * 2; };
    auto source = [&](const char *base, int64_t pitch, bool cols_, bool padded, int64_t at, int n) {
        return cols_ ? TileSrc{base + k0 * pitch + at * 2, pitch, (int)bytes(n, padded), k1 - k0, base}
                     : TileSrc{base + at * pitch + k0 * 2, pitch, n, bytes(k1 - k0, padded), base};
    };
    TileLoop<ST, Sh, DMA> t;
    const TileSrc A = source(p.A, p.a_pitch, Sh::ACOLS, p.a_padded, m0, rows);
    const TileSrc B = source(p.B, p.b_pitch, Sh::BCOLS, p.b_padded, n0, cols);
    const bool mine = t.run(A, B, smem);
    if (p.splits > 1) {
        if (!mine) return;
        float *P = p.part + (int64_t)s * p.M * p.N + m0 * p.N + n0;
        t.each([&](int m, int n, f32x4 v) {
            if (m >= rows) return;
            if (n + 4 <= cols) {
                __builtin_memcpy(P + (int64_t)m * p.N + n, &v, 16);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (n + i < cols) P[(int64_t)m * p.N + n + i] = v[i];
            }
        });
        return;
    }
    if constexpr (Sh::ACOLS) {   // a weight's gradient: nothing but the sums
        if (mine) store_tile<ST>(t, p.C + m0 * p.c_pitch + n0 * 2, p.c_pitch, rows, cols);
    } else {
        __syncthreads();         // every wave has read its last stage
        if (mine) finish_tile<ST, Sh>(t, p, smem, m0, n0);
    }
}

// The K ranges' sums, added in order, and the epilogue: 8 columns a lane
template <typename ST>
__global__ __launch_bounds__(256) void dense_join_kernel(DenseParams p) {
    const int64_t pieces = (p.N + 7) / 8, all = p.M * pieces, each = p.M * p.N;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
        const int64_t m = i / pieces, n = (i - m * pieces) * 8;
        const int left = p.N - n < 8 ? (int)(p.N - n) : 8;
        float v[8] = {}, bias[8];
        const float *P = p.part + m * p.N + n;
        for (int s = 0; s < p.splits; ++s, P += each) {
            if (left == 8) {
                f32x4 lo, hi;
                __builtin_memcpy(&lo, P, 16);
                __builtin_memcpy(&hi, P + 4, 16);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    v[e] += lo[e];
                    v[e + 4] += hi[e];
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (e < left) v[e] += P[e];
            }
        }
        bias_at<ST>(p, n, left, bias);
        finish8<ST>(p, v, bias, res_at<ST>(p, m, n, left), m, n, left);
    }
}

// ---------------------------------------------------------------------------
// A few rows (dense_few says how many): bound by reading W, once for every 16 of them,
// which are a row of the grid.  A wave takes a range of K; operands go from memory into
// the matrix cores' registers.  A block of 16 x 16 sums is R = 16 / P rows of x by R
// rows of W, each with P parts of K: index i of either operand is part i / R of row
// i % R, and of the sums those of equal parts count.  A load then reads P 64-byte
// pieces of R rows one behind another, which DRAM serves faster than pieces of 16 rows,
// and few rows of W still fill the chip.  The waves' sums and the parts are added in
// order in the LDS.
// Loads off a 4-byte address take two to three times as long, so rows of odd
// addresses (WORDS false) are read as the words that hold them and shifted (1 x 4096
// x 4097: 16.0 -> 11.7 us, 16 rows 27 -> 16).
// ---------------------------------------------------------------------------
template <typename ST, int P, int WAVES, int U, bool WORDS>
__global__ __launch_bounds__(64 * WAVES) void dense_few_kernel(DenseParams p) {
    constexpr int R = 16 / P;
    __shared__ __attribute__((aligned(16))) float join[WAVES][16][20];   // [x's index][W's index]
    const int lane = threadIdx.x & 63, g = lane >> 4, i16 = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t n0 = (int64_t)blockIdx.x * R;
    // rows past the last read the last one, and are not stored
    const int64_t m0 = (int64_t)blockIdx.y * 16, n = n0 + i16 % R, m = m0 + i16 % R;
    const int in = (i16 / R) * 128 + g * 16;   // the lane's first piece in a step of P 128 bytes
    const char *W = p.B + (n < p.N ? n : p.N - 1) * p.b_pitch + in;
    const char *X = p.A + (m < p.M ? m : p.M - 1) * p.a_pitch + in;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    const int64_t bytes = p.K * 2;
    constexpr int STEP = P * 128;
    auto piece = [&](const char *row, const char *first, int64_t at, bool whole) -> i32x4 {
        i32x4 v;
        if (whole && WORDS) {
            __builtin_memcpy(&v, row + at, 16);
            return v;
        }
        if (whole) {
            const uintptr_t p = (uintptr_t)(row + at);
            const uint32_t *w = (const uint32_t *)(p & ~(uintptr_t)3);
            const uint32_t by = (uint32_t)(p & 2) * 8, e = w[4];
            i32x4_words u = *(const i32x4_words *)w;
            return i32x4{(int)__builtin_amdgcn_alignbit((uint32_t)u.y, (uint32_t)u.x, by),
                         (int)__builtin_amdgcn_alignbit((uint32_t)u.z, (uint32_t)u.y, by),
                         (int)__builtin_amdgcn_alignbit((uint32_t)u.w, (uint32_t)u.z, by),
                         (int)__builtin_amdgcn_alignbit(e, (uint32_t)u.w, by)};
        }
        const int64_t left = bytes - at - in;
        return load_piece(row + (left > 0 ? at : 0), left < 16 ? (int)(left < 0 ? 0 : left) : 16, first);
    };
    // UU steps: all loads, then the products
    auto steps = [&](int64_t at, auto u_, auto whole_) {
        constexpr int UU = decltype(u_)::value;
        constexpr bool whole = decltype(whole_)::value;
        i32x4 w[UU][2], x[UU][2];
#pragma unroll
        for (int u = 0; u < UU; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                w[u][h] = piece(W, p.B, at + u * STEP + 64 * h, whole);
                x[u][h] = piece(X, p.A, at + u * STEP + 64 * h, whole);
            }
#pragma unroll
        for (int u = 0; u < UU; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h) acc = mfma16(w[u][h], x[u][h], acc, ST{});
    };
    using std::integral_constant;
    const int64_t per = ((bytes + STEP - 1) / STEP + WAVES - 1) / WAVES * STEP;
    int64_t at = per * wave;
    const int64_t end = at + per < bytes ? at + per : bytes;
    // (the word behind a shifted piece has to exist)
    const int64_t whole = WORDS || end + 4 <= bytes ? end : bytes - 4;
    for (; at + U * STEP <= whole; at += U * STEP) steps(at, integral_constant<int, U>{}, std::true_type{});
    for (; at + STEP <= whole; at += STEP) steps(at, integral_constant<int, 1>{}, std::true_type{});
    for (; at < end; at += STEP) steps(at, integral_constant<int, 1>{}, std::false_type{});

    *(f32x4 *)&join[wave][i16][4 * g] = acc;
    __syncthreads();
    // 8 columns of a row to a lane (R where that is less)
    constexpr int C = R < 8 ? R : 8, GROUPS = R / C;
    if (threadIdx.x < R * GROUPS) {
        const int row = threadIdx.x / GROUPS, c0 = threadIdx.x % GROUPS * C;
        float v[8] = {};
#pragma unroll
        for (int w = 0; w < WAVES; ++w)
#pragma unroll
            for (int q = 0; q < P; ++q)
#pragma unroll
                for (int e = 0; e < C; ++e) v[e] += join[w][q * R + row][q * R + c0 + e];
        const int64_t col = n0 + c0;
        const int left = p.N - col < C ? (int)(p.N - col) : C;
        if (m0 + row < p.M && left > 0) {
            float bias[8];
            bias_at<ST>(p, col, left, bias);
            finish8<ST>(p, v, bias, res_at<ST>(p, m0 + row, col, left), m0 + row, col, left);
        }
    }
}

// ---------------------------------------------------------------------------
// dz = dy act'(z), rounded to 16 bits as the matrix cores take it, and its column
// sums (of the unrounded values) over the rows of a workgroup: p.lanes lanes with 8
// columns each, 256 / lanes rows at a time.  Bound by memory, 6 bytes an element: with
// many rows a row is read up to 4 KB at a time.
// ---------------------------------------------------------------------------
template <typename ST> __global__ __launch_bounds__(256) void dense_grad_kernel(DenseGradParams p) {
    __shared__ __attribute__((aligned(16))) float join[256 * 8];
    const int lanes = p.lanes, step = 256 / lanes;
    const int in = threadIdx.x & (lanes - 1), of = threadIdx.x / lanes;
    const int64_t n0 = (int64_t)blockIdx.x * lanes * 8, n = n0 + in * 8;
    const int64_t m0 = (int64_t)blockIdx.y * p.rows;
    const int64_t m1 = p.M - m0 < p.rows ? p.M : m0 + p.rows;
    const int left = p.N - n < 8 ? (int)(p.N - n < 0 ? 0 : p.N - n) : 8;
    float sum[8] = {};
    auto add = [&](auto act_, auto whole_, i32x4 dyv, i32x4 zv, int64_t m) {
        constexpr int ACT = decltype(act_)::value;
        constexpr bool whole = decltype(whole_)::value;
        float d[8];
        unpack8<ST>(dyv, d);
        if constexpr (ACT != OZK_ACT_NONE) {
            float z[8];
            unpack8<ST>(zv, z);
#pragma unroll
            for (int i = 0; i < 8; ++i) d[i] *= whole || i < left ? derivative<ACT>(z[i]) : 0.f;
            if (p.dz) {
                const i32x4 v = pack8<ST>(d);
                __builtin_memcpy(p.dz + m * p.dz_pitch + n * 2, &v, 16);   // zeros behind N
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) sum[i] += d[i];
    };
    auto run = [&](auto act_) {
        constexpr int ACT = decltype(act_)::value;
        const char *dy = p.dy + n * 2, *z = p.z + n * 2;
        int64_t m = m0 + of;
        if (left == 8) {
            constexpr int U = 4;   // rows on their way at once
            for (; m + (U - 1) * step < m1; m += U * step) {
                i32x4 dv[U], zv[U] = {};
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    dv[u] = load8_once(dy + (m + u * step) * p.dy_pitch);
                    if constexpr (ACT != OZK_ACT_NONE) zv[u] = load8_once(z + (m + u * step) * p.N * 2);
                }
#pragma unroll
                for (int u = 0; u < U; ++u) add(act_, std::true_type{}, dv[u], zv[u], m + u * step);
            }
            for (; m < m1; m += step)
                add(act_, std::true_type{}, load8_once(dy + m * p.dy_pitch),
                    ACT != OZK_ACT_NONE ? load8_once(z + m * p.N * 2) : i32x4{}, m);
        } else if (left > 0) {
            for (; m < m1; m += step)
                add(act_, std::false_type{}, load8(dy + m * p.dy_pitch, left),
                    ACT != OZK_ACT_NONE ? load8(z + m * p.N * 2, left) : i32x4{}, m);
        }
    };
    if (p.act == OZK_ACT_NONE) run(std::integral_constant<int, OZK_ACT_NONE>{});
    else with_act(p.act, run);
    if (!p.sums) return;
    *(f32x4 *)&join[threadIdx.x * 8] = f32x4{sum[0], sum[1], sum[2], sum[3]};
    *(f32x4 *)&join[threadIdx.x * 8 + 4] = f32x4{sum[4], sum[5], sum[6], sum[7]};
    __syncthreads();
    const int columns = lanes * 8;
    for (int c = threadIdx.x; c < columns && n0 + c < p.N; c += 256) {
        float v = 0.f;
        for (int r = 0; r < step; ++r) v += join[r * columns + c];
        p.sums[(int64_t)blockIdx.y * p.N + n0 + c] = v;
    }
}
template <typename ST> __global__ __launch_bounds__(256) void dense_bias_kernel(DenseParams p) {
    __shared__ double join[16][16];
    add_bias<ST>(p, blockIdx.x, 256, join);
}

namespace {

bool pieces(const DenseParams &p) {
    return whole_pieces(p.A, p.a_pitch, 0, p.a_cols ? p.M : p.K, p.a_padded) &&
           whole_pieces(p.B, p.b_pitch, 0, p.b_cols ? p.N : p.K, p.b_padded);
}
int64_t tiles(const DenseParams &p, int64_t bm, int64_t bn) {
    return ((p.M + bm - 1) / bm) * ((p.N + bn - 1) / bn);
}

template <typename ST, typename Sh, bool DMA>
hipError_t dense_go(const DenseParams &p, hipStream_t st) {
    const int64_t all = tiles(p, Sh::BM, Sh::BN) * p.splits;
    if (all >= (int64_t)1 << 31) return hipErrorInvalidConfiguration;
    if (hipError_t e = allow_lds<&dense_kernel<ST, Sh, DMA>>(Sh::LDS_BYTES); e != hipSuccess) return e;
    const int64_t blocks = (all + 7) / 8 * 8 + (Sh::ACOLS && p.db ? (p.db_n + 15) / 16 : 0);
    dense_kernel<ST, Sh, DMA><<<dim3((uint32_t)blocks), Sh::THREADS, Sh::LDS_BYTES, st>>>(p);
    return hipGetLastError();
}
template <typename ST, int P, int WAVES, int U> hipError_t few_go(const DenseParams &p, hipStream_t st) {
    const int64_t blocks = (p.N + 16 / P - 1) / (16 / P);
    if (blocks >= (int64_t)1 << 31) return hipErrorInvalidConfiguration;
    const dim3 grid((uint32_t)blocks, (uint32_t)((p.M + 15) / 16));
    if ((((uintptr_t)p.A | (uintptr_t)p.B | (uintptr_t)p.a_pitch | (uintptr_t)p.b_pitch) & 3) == 0)
        dense_few_kernel<ST, P, WAVES, U, true><<<grid, 64 * WAVES, 0, st>>>(p);
    else
        dense_few_kernel<ST, P, WAVES, U, false><<<grid, 64 * WAVES, 0, st>>>(p);
    return hipGetLastError();
}
// Parts of K: as few as give three quarters of the CUs a workgroup.  Measured (us,
// M x N x K, one part / two / four):
//     1 x 4096 x 4096    8.9 / 10.0 / 12.2      1 x 1024 x 8192   12.2 / 8.0 / 6.4
//     1 x 8192 x 8192   25.0 / 27.0 / 30.2      1 x 1000 x 2048    5.7 / 4.6 / 4.5
template <typename ST> hipError_t few_plan(const DenseParams &p, hipStream_t st) {
    int parts = 1;
    while (parts < 4 && p.M * parts <= 8 && p.N * parts < 16 * 192) parts *= 2;
    if (parts == 1) return few_go<ST, 1, 8, 8>(p, st);
    if (parts == 2) return few_go<ST, 2, 8, 8>(p, st);
    return few_go<ST, 4, 8, 4>(p, st);
}

// The tile and the K ranges of the shortest time: rounds of workgroups, so many at
// once, by a round's time, `fixed` + `slope` K / 1024 us (fitted to 477 shapes of 32
// to 8192 rows and columns, K = 512 to 4096; operands along N have the times of those
// along K); partial sums cost a launch and their way through memory.  Chosen so,
// products of those shapes take longer than with the best tile of each, on average / at
// worst, of operands along K 0.6 / 10%, along N 1.7 / 41% (32 rows: 32 x 16 tiles read 32
// bytes of a row), of a weight's gradient 1.9 / 18%.
// Measured (us, M x N x K, operands along K, gelu; 32 x 16 / 32 x 32 / 64 x 32 / 64 x 64 in
// two groups of waves / 64 x 64 / 128 x 128 of 4 stages / 128 x 128 / 128 x 256 / 256 x
// 256):
//     32 x 4096 x 4096      12 / 14 / 15 / 20 / 33 / 31 / 60 / 51 / 96
//     128 x 4096 x 4096     34 / 24 / 18 / 23 / 34 / 42 / 64 / 61 / 103
//     512 x 4096 x 4096    124 / 86 / 61 / 42 / 39 / 40 / 63 / 59 / 111
//     1024 x 4096 x 1024   122 / 70 / 48 / 30 / 23 / 16 / 19 / 23 / 38
//     2048 x 4096 x 2048   303 / 206 / 139 / 93 / 76 / 48 / 45 / 42 / 66
//     4096 x 4096 x 2048   588 / 369 / 275 / 183 / 147 / 93 / 84 / 77 / 69
// and a weight's gradient of 8192 rows, 4096 x 2048, in its training step: 128 x 128
// 404 us a step, 128 x 256 413, 256 x 256 431.
struct TileCost {
    int bm, bn, at_once;
    float fixed[2], slope[2];   // of operands along K, of a weight's gradient
};
constexpr TileCost kTiles[] = {
    {32, 16, 256, {2.0f, 1.8f}, {1.45f, 2.4f}},     {32, 32, 256, {2.0f, 1.8f}, {2.25f, 3.3f}},
    {64, 32, 256, {2.7f, 2.2f}, {2.85f, 3.25f}},    {64, 64, 256, {2.7f, 2.1f}, {3.7f, 4.05f}},
    {64, 64, 512, {2.2f, 1.6f}, {6.5f, 7.2f}},      {128, 128, 256, {3.9f, 3.1f}, {7.4f, 7.8f}},
    {128, 128, 512, {6.0f, 1.8f}, {12.6f, 13.1f}},  {128, 256, 256, {6.1f, 4.7f}, {12.2f, 14.2f}},
    {256, 256, 256, {7.7f, 5.4f}, {21.5f, 21.0f}},
};
struct DensePlan {
    int tile, splits;
};
DensePlan plan_tiles(const DenseParams &p) {
    DensePlan best = {0, 1};
    double least = 0;
    for (int splits = 1; splits <= 16; splits *= 2) {
        // ranges of 8 stages at least, sums that stay in the caches
        if (splits > 1 && (p.K < 512 * splits || (double)splits * p.M * p.N > 1 << 24)) break;
        const double join = splits > 1 ? 3.0 + 2e-6 * splits * p.M * p.N : 0.0;
        for (int i = 0; i < (int)(sizeof kTiles / sizeof *kTiles); ++i) {
            const TileCost &t = kTiles[i];
            const double n = (double)tiles(p, t.bm, t.bn) * splits;
            const double time = join + ceil(n / t.at_once) * (t.fixed[p.a_cols] + t.slope[p.a_cols] *
                                                              (double)p.K / splits / 1024);
            if ((i == 0 && splits == 1) || time < least) {
                least = time;
                best = {i, splits};
            }
        }
    }
    return best;
}

template <typename ST, bool AC, bool BC> hipError_t tile_plan(const DenseParams &p, hipStream_t st) {
    if (!pieces(p)) {   // through registers (and with plan_tiles' K ranges, which know the others)
        if (p.M <= 32) return dense_go<ST, TileShape<1, AC, BC, 32, 64, 1, 4, 2>, false>(p, st);
        return dense_go<ST, TileShape<1, AC, BC, 128, 128, 2, 2, 2>, false>(p, st);
    }
    switch (plan_tiles(p).tile) {
    case 0: return dense_go<ST, TileShape<1, AC, BC, 32, 16, 1, 1, 4, 4>, true>(p, st);
    case 1: return dense_go<ST, TileShape<1, AC, BC, 32, 32, 1, 2, 4, 4>, true>(p, st);
    case 2: return dense_go<ST, TileShape<1, AC, BC, 64, 32, 2, 1, 3, 4>, true>(p, st);
    case 3: return dense_go<ST, TileShape<1, AC, BC, 64, 64, 2, 2, 4, 2>, true>(p, st);
    case 4: return dense_go<ST, TileShape<1, AC, BC, 64, 64, 2, 2, 2, 2>, true>(p, st);
    case 5: return dense_go<ST, TileShape<1, AC, BC, 128, 128, 2, 4, 4>, true>(p, st);
    case 6: return dense_go<ST, TileShape<1, AC, BC, 128, 128, 2, 4, 2>, true>(p, st);
    case 7: return dense_go<ST, TileShape<1, AC, BC, 128, 256, 2, 4, 3>, true>(p, st);
    default: return dense_go<ST, TileShape<1, AC, BC, 256, 256, 2, 4, 2>, true>(p, st);
    }
}
template <typename ST> hipError_t dense_plan(const DenseParams &p, hipStream_t st) {
    if (dense_few(p)) return few_plan<ST>(p, st);
    hipError_t e = p.a_cols ? tile_plan<ST, true, true>(p, st)
                 : p.b_cols ? tile_plan<ST, false, true>(p, st)
                            : tile_plan<ST, false, false>(p, st);
    if (e != hipSuccess || p.splits == 1) return e;
    const int64_t blocks = (p.M * ((p.N + 7) / 8) + 255) / 256;
    dense_join_kernel<ST><<<dim3((uint32_t)(blocks < 4096 ? blocks : 4096)), 256, 0, st>>>(p);
    return hipGetLastError();
}

}  // namespace

// Up to 4 rows; of those that the tiles' DMA cannot take up to 32, and up to 128 where
// W, read once for 16 of them, is small (us, this / tiles: 4 x 4096 x 4096 9.7 / 9.4, 16
// x 4096 x 4096 11.5 / 9.6; then this / tiles through registers / tiles on copies: 32 x
// 4096 x 4097 24 / 45 / 22, 48 x 4096 x 4097 34 / 27 / 26, 40 x 3648 x 1810 12 / 39 / 16, 96 x
// 3648 x 1810 18 / 39 / 18, 128 x 1024 x 1001 8 / 24 / 11).  Of a large W that costs: 32 x 8192 x
// 8190 75 / 109 / 64, 32 x 16384 x 4095 116 / 64 / 65.
bool dense_few(const DenseParams &p) {
    if (p.a_cols || p.b_cols) return false;
    if (p.M <= 4) return true;
    const int64_t groups = (p.M + 15) / 16;
    return (groups <= 2 || (groups <= 8 && (double)groups * p.N * p.K <= 35e6)) && !pieces(p);
}
int dense_splits(const DenseParams &p) {
    return dense_few(p) || p.M == 0 || p.N == 0 ? 1 : plan_tiles(p).splits;
}

hipError_t launch_dense(const DenseParams &p, int dtype, hipStream_t st) {
    return dtype == OZK_F16 ? dense_plan<_Float16>(p, st) : dense_plan<__bf16>(p, st);
}

// (us, lanes as below / 32: 8192 x 4096 bf16 41.4 / 43.0; 1999 x 520 fp16 with 32 5.7,
// with 128 8.2)
int dense_grad_lanes(int64_t M, int64_t N) {
    int lanes = 32;
    while (lanes < 256 && lanes * 8 < N && (M / 16) * (N / (lanes * 16)) >= 512) lanes *= 2;
    return lanes;
}
int64_t dense_grad_rows(int64_t M, int64_t N) {
    // about 1024 workgroups, of 16 to 128 rows
    const int64_t columns = dense_grad_lanes(M, N) * 8, across = (N + columns - 1) / columns;
    int64_t rows = 128;
    while (rows > 16 && ((M + rows - 1) / rows) * across < 768) rows /= 2;
    while ((M + rows - 1) / rows >= 32768) rows *= 2;
    return rows;
}
hipError_t launch_dense_grad(const DenseGradParams &q, int dtype, hipStream_t st) {
    DenseGradParams p = q;
    p.lanes = dense_grad_lanes(p.M, p.N);
    const int64_t columns = p.lanes * 8;
    const dim3 grid((uint32_t)((p.N + columns - 1) / columns), (uint32_t)((p.M + p.rows - 1) / p.rows));
    if (dtype == OZK_F16) dense_grad_kernel<_Float16><<<grid, 256, 0, st>>>(p);
    else dense_grad_kernel<__bf16><<<grid, 256, 0, st>>>(p);
    return hipGetLastError();
}
hipError_t launch_dense_bias(const DenseGradParams &p, int dtype, hipStream_t st) {
    DenseParams q = {};
    q.sums = p.sums;
    q.db = p.db;
    q.db_n = p.N;
    q.db_blocks = (p.M + p.rows - 1) / p.rows;
    const dim3 grid((uint32_t)((p.N + 15) / 16));
    if (dtype == OZK_F16) dense_bias_kernel<_Float16><<<grid, 256, 0, st>>>(q);
    else dense_bias_kernel<__bf16><<<grid, 256, 0, st>>>(q);
    return hipGetLastError();
}

}  // namespace ozk
