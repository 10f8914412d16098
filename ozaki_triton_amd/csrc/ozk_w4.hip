// ozk_w4.hip -- products with 4-bit weights in groups with scales, and the
// kernels that make and undo the format.
//
//   y[m, n] = sum_g s[n, g] (sum_{k in g} x[m, k] (16 + q[n, k])
//                            - (16 + z[n, g]) sum_{k in g} x[m, k])
//
// q is a whole number of 0 .. 15, so 16 + q is one OR away from its 4 bits in
// fp16 and bf16 (the exponent of 16, q in the mantissa's upper bits), the
// matrix cores multiply it by x exactly, and the scale and the zero point come
// in fp32 once per group: no weight is rounded.  fp32 x goes in as three bf16
// slices h + m + l = x; h is summed apart from m and l: a sum of h (16 + q) has
// few bits and stays all but exact, where one that takes up m and l is rounded
// at 5 times the result's size before the zero point comes off (1.5e-6 off
// against 3e-7 at K = 2048).  (A row of x with an
// infinity gives NaN: the two sums cancel.)
//
// Both sums are up to 31 times the sum of |x|, so where x has fp32's exponents
// they and all that follows are kept times 2^-12 until the result is stored:
// 128 of 31 times the largest float then stay within it, and no finite x gives
// NaN.  (Values of x below 2^-100 or so lose their last bits instead.)
//
// Few rows of x make this a read of the weights: they go straight from memory
// to registers, 16 bytes (32 weights) of a row per lane, several loads ahead;
// x waits in the LDS.
#include "ozk_linear.h"
#include "ozk_tile.h"

namespace ozk {

template <typename XT> struct W4Type;   // matrix-core type of x, slices of it
template <> struct W4Type<_Float16> { using M = _Float16; static constexpr int SL = 1; };
template <> struct W4Type<__bf16> { using M = __bf16; static constexpr int SL = 1; };
template <> struct W4Type<float> { using M = __bf16; static constexpr int SL = 3; };

// what the sums are kept times
template <typename M> constexpr float kW4Down = std::is_same<M, __bf16>::value ? 0x1p-12f : 1.f;

// the 8 weights of a word as 16 + q, times kW4Down: element order 0, 4, 1, 5, 2, 6,
// 3, 7
OZK_DEV i32x4 unpack_w4(uint32_t w, _Float16) {   // q << 6 beside fp16's 16.0
    return i32x4{(int)(((w << 6) & 0x03C003C0u) | 0x4C004C00u),
                 (int)(((w << 2) & 0x03C003C0u) | 0x4C004C00u),
                 (int)(((w >> 2) & 0x03C003C0u) | 0x4C004C00u),
                 (int)(((w >> 6) & 0x03C003C0u) | 0x4C004C00u)};
}
OZK_DEV i32x4 unpack_w4(uint32_t w, __bf16) {     // q << 3 beside bf16's 2^-8
    return i32x4{(int)(((w << 3) & 0x00780078u) | 0x3B803B80u),
                 (int)(((w >> 1) & 0x00780078u) | 0x3B803B80u),
                 (int)(((w >> 5) & 0x00780078u) | 0x3B803B80u),
                 (int)(((w >> 9) & 0x00780078u) | 0x3B803B80u)};
}

// Lane group j's word i against lane group i's word j: lane group g held 32
// weights of block g of a chunk, afterwards word j holds 8 weights of block j
// in every lane group.
OZK_DEV void transpose_words(uint32_t (&r)[4]) {
    auto swap32 = [](uint32_t &a, uint32_t &b) {
        const auto t = __builtin_amdgcn_permlane32_swap(a, b, false, false);
        a = t[0];
        b = t[1];
    };
    auto swap16 = [](uint32_t &a, uint32_t &b) {
        const auto t = __builtin_amdgcn_permlane16_swap(a, b, false, false);
        a = t[0];
        b = t[1];
    };
    swap32(r[0], r[2]);
    swap32(r[1], r[3]);
    swap16(r[0], r[1]);
    swap16(r[2], r[3]);
}

OZK_DEV void push32(i32x4 &lo, i32x4 &hi, int e) {
    hi = i32x4{lo.w, hi.x, hi.y, hi.z};
    lo = i32x4{e, lo.x, lo.y, lo.z};
}

// 8 scales and zero points of a row of W, of which the first n exist
struct SPiece {
    i32x4 s[2];      // fp32, or 16 bits in the first
    i32x2 z;
    OZK_DEV void load(const W4Params &p, int64_t row, int64_t g, int n) {
        const int64_t at = row * p.s_pitch + g;
        const uint8_t *zf = p.zeros ? p.zeros + row * p.z_pitch + g : nullptr;
        z = i32x2{0, 0};
        if (n >= 8) {
            if (p.scales32) __builtin_memcpy(s, (const float *)p.scales + at, 32);
            else __builtin_memcpy(s, (const uint16_t *)p.scales + at, 16);
            if (zf) __builtin_memcpy(&z, zf, 8);
        } else {
            s[0] = s[1] = i32x4{0, 0, 0, 0};
#pragma unroll 1
            for (int i = n - 1; i >= 0; --i) {
                if (p.scales32) push32(s[0], s[1], ((const int *)p.scales)[at + i]);
                else push16(s[0], ((const uint16_t *)p.scales)[at + i]);
                if (zf) {
                    z.y = (int)__builtin_amdgcn_alignbit((uint32_t)z.y, (uint32_t)z.x, 24);
                    z.x = (int)(((uint32_t)z.x << 8) | zf[i]);
                }
            }
        }
    }
    OZK_DEV float2 at(const W4Params &p, int i, int dtype16) const {   // (s, 16 + z)
        float f;
        if (p.scales32) {
            f = __int_as_float(s[i >> 2][i & 3]);
        } else {
            const uint16_t u = (uint16_t)((uint32_t)s[0][i >> 1] >> (16 * (i & 1)));
            f = dtype16 == 2 ? (float)__builtin_bit_cast(_Float16, u) : bf16_bits_to_f32(u);
        }
        const uint32_t q = ((uint32_t)z[i >> 2] >> (8 * (i & 3))) & 255u;
        return float2{f, p.zeros ? 16.f + (float)q : 24.f};
    }
};

// the sum over 4, 8 or 16 consecutive lanes, in each of them
template <int CTRL> OZK_DEV float dpp_add(float v) {
    return v + __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xF, 0xF, true));
}
template <int N> OZK_DEV float sum_lanes(float v) {
    v = dpp_add<0xB1>(v);                      // lane ^ 1
    v = dpp_add<0x4E>(v);                      // lane ^ 2
    if constexpr (N > 4) v = dpp_add<0x141>(v);   // the other four of 8
    if constexpr (N > 8) v = dpp_add<0x140>(v);   // the other eight of 16
    return v;
}

// 8 values of a row of x, of which the first n exist
template <typename XT> struct XPiece {
    static constexpr int W = sizeof(XT) / 2;   // 16-byte words
    i32x4 raw[W];
    OZK_DEV void load(const char *from, int n) {
        if (n >= 8) {
            __builtin_memcpy(raw, from, sizeof(raw));   // rows of any alignment
            return;
        }
#pragma unroll
        for (int w = 0; w < W; ++w) raw[w] = i32x4{0, 0, 0, 0};
#pragma unroll 1
        for (int i = n - 1; i >= 0; --i) {
            if constexpr (W == 2) push32(raw[0], raw[1], ((const int *)from)[i]);
            else push16(raw[0], ((const uint16_t *)from)[i]);
        }
    }
    OZK_DEV void values(float (&v)[8]) const {
        if constexpr (W == 2) {
            __builtin_memcpy(v, raw, 32);
        } else {
            uint16_t e[8];
            __builtin_memcpy(e, raw, 16);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = from_bits16(e[i], XT{});
        }
    }
};

// Waves: WN along n, WK along the chunks of K; a wave has RT blocks of 16 n
// and TT blocks of 16 rows of x; GPC groups per chunk of 128 k.  The LDS holds
// x, its sums over the groups, and scale and zero point of the workgroup's
// rows of W, for p.held of K.  The loads of x, then of the scales, then of the
// wave's first U chunks of W are all on their way before the first is used.
template <typename XT, int WN, int WK, int RT, int TT, int GPC>
__global__ __launch_bounds__(64 * WN * WK) void w4_kernel(W4Params p) {
    using MT = typename W4Type<XT>::M;
    constexpr int SL = W4Type<XT>::SL, NT = 64 * WN * WK, U = 8 / RT, NR = 16 * RT * WN;
    constexpr int AC = SL > 1 ? 2 : 1;   // sums of the first slice and of the others, apart
    constexpr int D16 = std::is_same<XT, _Float16>::value ? 2 : 3;
    // pieces of x and scales a lane loads at once, before its first chunks of W:
    // loads return in order, so one issued behind W's waits for W
    constexpr int XB = SL > 1 ? 4 : TT > 1 ? 8 : 4, SB = 1;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wn = wave / WK, wk = wave % WK, g = lane >> 4, i16 = lane & 15;

    const int64_t n0 = (int64_t)blockIdx.x * NR;
    const int64_t nb = n0 + wn * 16 * RT;
    const int64_t m0 = (int64_t)blockIdx.y * (16 * TT);
    const int rows = (int)(p.M - m0 < 16 * TT ? p.M - m0 : 16 * TT);
    const int64_t kbeg = (int64_t)blockIdx.z * p.range;
    const int64_t kend = kbeg + p.range < p.K ? kbeg + p.range : p.K;

    // x [slice][row][k]; its sums [AC][group][16 TT rows]; (s, 16 + z) [row][group]
    const int pitch = p.held * 2 + 16;
    const int slice_bytes = rows * pitch;
    const int gheld = p.held / p.group, sums_each = gheld * 16 * TT;
    float *sums = (float *)(smem + SL * slice_bytes);
    float2 *scales = (float2 *)(sums + AC * sums_each);
    const int spitch = gheld + 1;

    const uint8_t *wrow[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        const int64_t n = nb + 16 * r + i16;
        wrow[r] = p.packed + (n < p.N ? n : p.N - 1) * p.w_pitch;
    }
    f32x4 acc[RT][TT];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int t = 0; t < TT; ++t) acc[r][t] = f32x4{0.f, 0.f, 0.f, 0.f};

    const int64_t pieces = (p.K + 31) / 32;          // 16-byte pieces of a row of W
    const int64_t groups = (p.K + p.group - 1) / p.group;
    struct Chunk {
        i32x4 w[RT];
    };
    auto load = [&](int64_t c, Chunk &ch) {          // chunk c: k from 128 c on
        const int64_t piece = c * 4 + g;
#pragma unroll
        for (int r = 0; r < RT; ++r)
            ch.w[r] = piece < pieces ? *(const i32x4 *)(wrow[r] + piece * 16) : i32x4{0, 0, 0, 0};
    };

    for (int64_t k0 = kbeg; k0 < kend; k0 += p.held) {
        const int64_t kstop = k0 + p.held < kend ? k0 + p.held : kend;
        // the wave's chunk t: pairs of chunks (a 128-byte line of each row) in turn
        const int64_t c0 = k0 / 128, c1 = (kstop + 127) / 128;
        auto chunk = [&](int t) { return c0 + ((t >> 1) * WK + wk) * 2 + (t & 1); };

        // x: pieces of 8 of whole chunks, zeros past K
        const int per_row = (int)((kstop - k0 + 127) / 128 * 16), all = rows * per_row;
        const int gcount = (int)((kstop - k0 + p.group - 1) / p.group);
        const int gpieces = (gcount + 7) / 8, sall = NR * gpieces;
        const float x_rcp = 1.f / (float)per_row, s_rcp = 1.f / (float)gpieces;
        XPiece<XT> xp[XB];
        SPiece sp[SB];
        auto load_x = [&](int i, XPiece<XT> &x) {
            const int row = i < all ? part_of(i, per_row, x_rcp) : 0;
            const int at = i < all ? i - row * per_row : 0;
            const int64_t k = k0 + at * 8;
            const int64_t n = i < all ? p.K - k : 0;
            x.load(p.x + ((m0 + row) * p.x_pitch + k) * (int64_t)sizeof(XT),
                   n < 0 ? 0 : n < 8 ? (int)n : 8);
        };
        auto put_x = [&](int i, const XPiece<XT> &x) {
            const int row = i < all ? part_of(i, per_row, x_rcp) : 0;
            const int at = i < all ? i - row * per_row : 0;
            float v[8], sum[AC] = {};
            x.values(v);
            if constexpr (SL == 1) {
                uint16_t h[8];
                __builtin_memcpy(h, x.raw, 16);
                // in the order of the unpacked weights
                const uint16_t o[8] = {h[0], h[4], h[1], h[5], h[2], h[6], h[3], h[7]};
                i32x4 u;
                __builtin_memcpy(&u, o, 16);
                if (i < all) *(i32x4 *)(smem + row * pitch + at * 16) = u;
#pragma unroll
                for (int e = 0; e < 8; ++e) sum[0] = __builtin_fmaf(v[e], kW4Down<MT>, sum[0]);
            } else {
                // 8, 8 and 8 bits of the 24: a slice is the upper half of what is left
#pragma unroll
                for (int s = 0; s < SL; ++s) {
                    i32x4 u;
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        u[e] = (int)__builtin_amdgcn_perm(__float_as_uint(v[e + 4]),
                                                          __float_as_uint(v[e]), 0x07060302u);
                    if (i < all) *(i32x4 *)(smem + s * slice_bytes + row * pitch + at * 16) = u;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float h = __uint_as_float(__float_as_uint(v[e]) & 0xFFFF0000u);
                        if (s + 1 < SL) v[e] -= h;
                        if (s == 0) {
                            sum[0] = __builtin_fmaf(h, kW4Down<MT>, sum[0]);
                            sum[AC - 1] = __builtin_fmaf(v[e], kW4Down<MT>, sum[AC - 1]);
                        }
                    }
                }
            }
#pragma unroll
            for (int a = 0; a < AC; ++a) {
                const float t = sum_lanes<16 / GPC>(sum[a]);
                if (i < all && at % (16 / GPC) == 0)
                    sums[a * sums_each + at / (16 / GPC) * 16 * TT + row] = t;
            }
        };
        auto load_s = [&](int i, SPiece &s) {
            if (i >= sall) return;
            const int row = part_of(i, gpieces, s_rcp), at = (i - row * gpieces) * 8;
            const int64_t n = n0 + row < p.N ? n0 + row : p.N - 1, gi = k0 / p.group + at;
            s.load(p, n, gi, (int)(groups - gi < 8 ? groups - gi : 8));
        };
        auto put_s = [&](int i, const SPiece &s) {
            if (i >= sall) return;
            const int row = part_of(i, gpieces, s_rcp), at = (i - row * gpieces) * 8;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (at + e < gcount) scales[row * spitch + at + e] = s.at(p, e, D16);
        };

#pragma unroll
        for (int u = 0; u < XB; ++u) load_x(threadIdx.x + u * NT, xp[u]);
#pragma unroll
        for (int u = 0; u < SB; ++u) load_s(threadIdx.x + u * NT, sp[u]);
        Chunk cur[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (chunk(u) < c1) load(chunk(u), cur[u]);

        if (k0 != kbeg) __syncthreads();             // the last part of x has been read
#pragma unroll
        for (int u = 0; u < XB; ++u) put_x(threadIdx.x + u * NT, xp[u]);
#pragma unroll
        for (int u = 0; u < SB; ++u) put_s(threadIdx.x + u * NT, sp[u]);
        for (int i = threadIdx.x + XB * NT; i < (all + NT - 1) / NT * NT; i += XB * NT) {
#pragma unroll
            for (int u = 0; u < XB; ++u) load_x(i + u * NT, xp[u]);
#pragma unroll
            for (int u = 0; u < XB; ++u) put_x(i + u * NT, xp[u]);
        }
        for (int i = threadIdx.x + SB * NT; i < sall; i += SB * NT) {
#pragma unroll
            for (int u = 0; u < SB; ++u) load_s(i + u * NT, sp[u]);
#pragma unroll
            for (int u = 0; u < SB; ++u) put_s(i + u * NT, sp[u]);
        }
        __syncthreads();

        for (int t0 = 0; chunk(t0) < c1; t0 += U) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t cu = chunk(t0 + u);
                if (cu >= c1) break;
                const int kl = (int)(cu * 128 - k0);   // of the chunk, in the LDS
                uint32_t w[RT][4];
#pragma unroll
                for (int r = 0; r < RT; ++r) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) w[r][j] = (uint32_t)cur[u].w[r][j];
                    transpose_words(w[r]);
                }
                // the registers are free again: the chunk U rounds on
                if (chunk(t0 + u + U) < c1) load(chunk(t0 + u + U), cur[u]);
#pragma unroll
                for (int q = 0; q < GPC; ++q) {
                    f32x4 part[AC][RT][TT];
#pragma unroll
                    for (int a = 0; a < AC; ++a)
#pragma unroll
                        for (int r = 0; r < RT; ++r)
#pragma unroll
                            for (int t = 0; t < TT; ++t) part[a][r][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int j = q * (4 / GPC); j < (q + 1) * (4 / GPC); ++j) {
                        i32x4 wf[RT];
#pragma unroll
                        for (int r = 0; r < RT; ++r) wf[r] = unpack_w4(w[r][j], MT{});
#pragma unroll
                        for (int t = 0; t < TT; ++t)
#pragma unroll
                            for (int s = 0; s < SL; ++s) {
                                const int row = 16 * t + i16 < rows ? 16 * t + i16 : rows - 1;
                                const i32x4 xf = *(const i32x4 *)(smem + s * slice_bytes +
                                                                  row * pitch +
                                                                  (kl + 32 * j + 8 * g) * 2);
#pragma unroll
                                for (int r = 0; r < RT; ++r)
                                    part[s > 0][r][t] = mfma16(xf, wf[r], part[s > 0][r][t], MT{});
                            }
                    }
                    const int gl = kl / 128 * GPC + q;
                    float2 sz[RT];
#pragma unroll
                    for (int r = 0; r < RT; ++r)
                        sz[r] = scales[(wn * 16 * RT + 16 * r + i16) * spitch +
                                       (gl < gcount ? gl : gcount - 1)];
#pragma unroll
                    for (int t = 0; t < TT; ++t) {
                        const float *xs = sums + gl * 16 * TT + 16 * t + 4 * g;
                        const f32x4 x0 = *(const f32x4 *)xs;
                        f32x4 x1 = x0;
                        if constexpr (AC > 1) x1 = *(const f32x4 *)(xs + sums_each);
#pragma unroll
                        for (int r = 0; r < RT; ++r)
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                float v = __builtin_fmaf(-sz[r].y, x0[e], part[0][r][t][e]);
                                if constexpr (AC > 1)
                                    v += __builtin_fmaf(-sz[r].y, x1[e], part[1][r][t][e]);
                                acc[r][t][e] = __builtin_fmaf(sz[r].x, v, acc[r][t][e]);
                            }
                    }
                }
            }
        }
    }

    // the waves along K, summed in order through the LDS
    if constexpr (WK > 1) {
        f32x4 *to = (f32x4 *)smem;
        __syncthreads();
        if (wk > 0)
#pragma unroll
            for (int r = 0; r < RT; ++r)
#pragma unroll
                for (int t = 0; t < TT; ++t)
                    to[(((wk - 1) * WN + wn) * RT * TT + r * TT + t) * 64 + lane] = acc[r][t];
        __syncthreads();
        if (wk > 0) return;
#pragma unroll
        for (int w = 1; w < WK; ++w)
#pragma unroll
            for (int r = 0; r < RT; ++r)
#pragma unroll
                for (int t = 0; t < TT; ++t) {
                    const f32x4 v = to[(((w - 1) * WN + wn) * RT * TT + r * TT + t) * 64 + lane];
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[r][t][e] += v[e];
                }
    }
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        const int64_t n = nb + 16 * r + i16;
        if (n >= p.N) continue;
#pragma unroll
        for (int t = 0; t < TT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int row = 16 * t + 4 * g + e;
                if (row >= rows) continue;
                const float v = acc[r][t][e] * (1.f / kW4Down<MT>);
                if (p.splits > 1) {
                    p.part[((int64_t)blockIdx.z * p.M + m0 + row) * p.N + n] = acc[r][t][e];
                } else if constexpr (sizeof(XT) == 4) {
                    ((float *)p.y)[(m0 + row) * p.y_pitch + n] = v;
                } else {
                    ((uint16_t *)p.y)[(m0 + row) * p.y_pitch + n] = to_bits16(v, XT{});
                }
            }
    }
}

template <typename XT> __global__ __launch_bounds__(256) void w4_join_kernel(W4Params p) {
    const int64_t all = p.M * p.N;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all;
         i += (int64_t)gridDim.x * 256) {
        float v = 0.f;
        for (int s = 0; s < p.splits; ++s) v += p.part[s * all + i];
        v *= 1.f / kW4Down<typename W4Type<XT>::M>;
        const int64_t m = i / p.N, n = i - m * p.N;
        if constexpr (sizeof(XT) == 4) ((float *)p.y)[m * p.y_pitch + n] = v;
        else ((uint16_t *)p.y)[m * p.y_pitch + n] = to_bits16(v, XT{});
    }
}

// ---------------------------------------------------------------------------
// The format.  Symmetric: s = fl(max |w| fl(1 / 7)), z = 8; with zero points: s =
// fl((max(w, 0) - min(w, 0)) fl(1 / 15)) (the two multiplied first where their
// difference is past fp32), z = rint(-min(w, 0) / s).  q = rint(w / s) + z within 0
// .. 15; a group of zeros has s = 0 and q = z.  NaN counts as 0.
// ---------------------------------------------------------------------------
template <typename T> OZK_DEV float rounded(float v) {
    if constexpr (sizeof(T) == 4) return v;
    else return from_bits16(to_bits16(v, T{}), T{});
}

// smallest and largest over 4, 8 or 16 consecutive lanes, in each of them (of a
// number and NaN the number)
template <int CTRL> OZK_DEV void dpp_range(float &lo, float &hi) {
    lo = fminf(lo, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(lo), CTRL, 0xF, 0xF, true)));
    hi = fmaxf(hi, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(hi), CTRL, 0xF, 0xF, true)));
}

// bytes of a packed row: those up to its distance are not the format's
__host__ __device__ inline int64_t packed_bytes_of(int64_t K) { return (K + 31) / 32 * 16; }

// 8 weights a lane: a group is 4, 8 or 16 lanes, a wave 512 weights of a row.
// The divisions and roundings bound it (8192 x 8192 bf16: 64 us with v / s and
// rint per weight), so a group divides once, y = fl(1 / s), and each quotient is
// corrected twice by its exact remainder, which gives fl(v / s) (Markstein,
// 1990: one correction of a quotient within a unit does where y is fl(1 / s));
// adding 1.5 2^23 rounds it to a whole number, ties to even.
template <typename T> __global__ __launch_bounds__(256) void quantize_w4_kernel(QuantParams p) {
    const int64_t row_bytes = packed_bytes_of(p.K);
    const uint32_t per_row = (uint32_t)((row_bytes * 2 + 511) / 512);
    const uint32_t part = blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    const int64_t n = part / per_row, k = (int64_t)(part - (uint32_t)n * per_row) * 512 + lane * 8;
    if (n >= p.N) return;
    XPiece<T> x;
    x.load(p.W + (n * p.w_pitch + k) * (int64_t)sizeof(T),
           k + 8 <= p.K ? 8 : k < p.K ? (int)(p.K - k) : 0);
    float v[8], lo = 0.f, hi = 0.f;
    x.values(v);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        lo = fminf(lo, v[e]);
        hi = fmaxf(hi, v[e]);
    }
    dpp_range<0xB1>(lo, hi);                           // lane ^ 1
    dpp_range<0x4E>(lo, hi);                           // lane ^ 2
    if (p.group >= 64) dpp_range<0x141>(lo, hi);       // the other four of 8
    if (p.group == 128) dpp_range<0x140>(lo, hi);      // the other eight of 16
    float s, z = 8.f;
    if (p.zeros) {
        const float range = hi - lo;
        s = rounded<T>(__builtin_isinf(range) ? hi * (1.f / 15.f) - lo * (1.f / 15.f)
                                              : range * (1.f / 15.f));
        z = s > 0.f ? fminf(fmaxf(rintf(-lo / s), 0.f), 15.f) : 0.f;
    } else {
        s = rounded<T>(fmaxf(hi, -lo) * (1.f / 7.f));
    }
    uint32_t word = 0;
    bool nan = false;
#pragma unroll
    for (int e = 0; e < 8; e += 2) nan = nan || __builtin_isunordered(v[e], v[e + 1]);
    // remainders stay clear of the subnormals
    if (s > 0x1p-90f && s < 0x1p90f && !nan) {
        const float y = 1.f / s;
        const int zi = (int)z - 0x4B400000;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            float q = v[e] * y;
            q = __builtin_fmaf(__builtin_fmaf(-q, s, v[e]), y, q);
            q = __builtin_fmaf(__builtin_fmaf(-q, s, v[e]), y, q);
            const int i = __float_as_int(q + 12582912.f) + zi;
            word |= (uint32_t)(i < 0 ? 0 : i > 15 ? 15 : i) << (4 * e);
        }
    } else {
#pragma unroll 1
        for (int e = 7; e >= 0; --e) {
            float q = s > 0.f ? rintf(v[7] / s) : 0.f;
            if (q != q) q = 0.f;
            word = (word << 4) | (uint32_t)(int)fminf(fmaxf(q + z, 0.f), 15.f);
#pragma unroll
            for (int i = 7; i > 0; --i) v[i] = v[i - 1];
        }
    }
    if (k < p.K && k % p.group == 0) {
        const int64_t g = k / p.group;
        store_value<T>(p.scales, n * p.s_pitch + g, s);
        if (p.zeros) p.zeros[n * p.z_pitch + g] = (uint8_t)(int)z;
    }
    if (k / 2 < row_bytes) *(uint32_t *)(p.packed + n * p.p_pitch + k / 2) = word;
}

// 8 weights a lane, a wave 512 of a row; bound by its stores (8192 x 8192 bf16: 27 us, 6.3
// TB/s; where a row started off 16 bytes 8 stores a lane took 9.7 us for 1000 x 2047 fp32, the
// wide ones of any alignment 5.6)
template <typename T, typename ST>
__global__ __launch_bounds__(256) void dequantize_w4_kernel(QuantParams p) {
    const uint32_t per_row = (uint32_t)((p.K + 511) / 512);
    const uint32_t part = blockIdx.x * 4 + (threadIdx.x >> 6), row = part / per_row;
    const int64_t n = row, k = (int64_t)(part - row * per_row) * 512 + (threadIdx.x & 63) * 8;
    if (n >= p.N || k >= p.K) return;
    const int64_t g = k >> (31 - __builtin_clz((uint32_t)p.group));
    const uint32_t word = *(const uint32_t *)(p.packed + n * p.p_pitch + k / 2);
    const float s = load_value<ST>(p.scales, n * p.s_pitch + g);
    const float z = p.zeros ? (float)p.zeros[n * p.z_pitch + g] : 8.f;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = ((float)((word >> (4 * e)) & 15u) - z) * s;
    char *to = p.out + (n * p.w_pitch + k) * (int64_t)sizeof(T);
    if (k + 8 <= p.K) {   // rows of any alignment
        i32x4 u[sizeof(T) / 2];
        if constexpr (sizeof(T) == 4) {
            __builtin_memcpy(u, v, 32);
        } else {
            uint16_t h[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) h[e] = to_bits16(v[e], T{});
            __builtin_memcpy(u, h, 16);
        }
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) __builtin_memcpy(to + 16 * i, &u[i], 16);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (k + e < p.K) store_value<T>(to, e, v[e]);
    }
}

namespace {

// Waves along n and K, blocks of n and of rows of x per wave; bytes of the LDS
// for x and the scales.  Few rows of x: one block of 16 n and its whole K to a
// workgroup, nothing to join.  More rows of x: more n to a workgroup, since
// each stages x for itself, and K cut to have a workgroup per CU.  Measured
// (us, HIP graph of 40 calls on several weights, M x N x K, group):
//     1 x 4096 x 4096, 128    {1,8,1,1} 7.7   {2,4,2,1} 10.2   {8,1,2,2} > 11
//     1 x 16384 x 4096, 128   {1,8,1,1} 16.8  {2,4,2,1} 14.3   {4,2,2,1} 17.0
//     2 x 8192 x 8192, 32     {1,8,1,1} 21.0  {2,4,2,1} 21.7   {4,2,2,1} 23.4
//     16 x 8192 x 8192, 128   {4,2,2,1} 22.6  {8,1,2,2} 21.4
//     32 x 8192 x 8192, 128   {4,2,2,2} 26.0  {8,1,2,2} 21.9   {8,1,2,4} 24.8
//     64 x 8192 x 8192, 128   {4,2,2,4} > 40  {8,1,2,2} 35.3   {8,1,2,4} 31.6
struct W4Shape {
    int wn, wk, rt, tt, lds;
};
constexpr W4Shape kW4Shapes[] = {
    {1, 8, 1, 1, 64 << 10}, {2, 4, 2, 1, 64 << 10}, {8, 1, 2, 2, 128 << 10}, {8, 1, 2, 4, 150 << 10}};
int w4_shape(const W4Params &p, int slices) {
    if (p.M <= 16 && p.N <= (p.M <= 4 ? 8192 : 4096)) return 0;
    if (p.M <= 4) return 1;
    return p.M <= 32 || slices > 1 ? 2 : 3;   // (3 with three slices of x leaves no registers)
}
int64_t w4_rows(const W4Params &p, const W4Shape &s) { return p.M < 16 * s.tt ? p.M : 16 * s.tt; }
int lds_of(const W4Params &p, const W4Shape &s, int slices) {
    const int groups = p.held / p.group;
    const int64_t x = slices * w4_rows(p, s) * (p.held * 2 + 16);
    const int64_t sums = (int64_t)groups * 16 * s.tt * 4 * (slices > 1 ? 2 : 1);
    const int64_t scales = (int64_t)16 * s.rt * s.wn * (groups + 1) * 8;
    const int64_t join = (int64_t)(s.wk - 1) * s.wn * s.rt * s.tt * 64 * 16;
    return (int)(x + sums + scales > join ? x + sums + scales : join);
}

template <typename XT, int I, int GPC> hipError_t w4_start(const W4Params &p, hipStream_t st) {
    constexpr W4Shape s = kW4Shapes[I];
    const int lds = lds_of(p, s, W4Type<XT>::SL);
    if (hipError_t e = allow_lds<&w4_kernel<XT, s.wn, s.wk, s.rt, s.tt, GPC>>(lds); e != hipSuccess)
        return e;
    // a launch counts 65535 blocks of rows (so many fill the GPU without K ranges)
    constexpr int64_t rows = 65535 * 16 * s.tt;
    for (int64_t m = 0; m < p.M; m += rows) {
        W4Params q = p;
        q.x += m * p.x_pitch * (int64_t)sizeof(XT);
        q.y += m * p.y_pitch * (int64_t)sizeof(XT);
        q.M = p.M - m < rows ? p.M - m : rows;
        const dim3 grid((uint32_t)((p.N + 16 * s.rt * s.wn - 1) / (16 * s.rt * s.wn)),
                        (uint32_t)((q.M + 16 * s.tt - 1) / (16 * s.tt)), (uint32_t)p.splits);
        w4_kernel<XT, s.wn, s.wk, s.rt, s.tt, GPC><<<grid, 64 * s.wn * s.wk, lds, st>>>(q);
        if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    }
    return hipSuccess;
}

template <typename XT, int I> hipError_t w4_go(const W4Params &p, hipStream_t st) {
    const hipError_t e = p.group == 32   ? w4_start<XT, I, 4>(p, st)
                         : p.group == 64 ? w4_start<XT, I, 2>(p, st)
                                         : w4_start<XT, I, 1>(p, st);
    if (e != hipSuccess || p.splits == 1) return e;
    const int64_t blocks = (p.M * p.N + 255) / 256;
    w4_join_kernel<XT><<<dim3((uint32_t)(blocks < 1024 ? blocks : 1024)), 256, 0, st>>>(p);
    return hipGetLastError();
}

template <typename XT> hipError_t w4_run(const W4Params &p, hipStream_t st) {
    switch (w4_shape(p, W4Type<XT>::SL)) {
    case 0: return w4_go<XT, 0>(p, st);
    case 1: return w4_go<XT, 1>(p, st);
    case 2: return w4_go<XT, 2>(p, st);
    }
    if constexpr (W4Type<XT>::SL == 1) return w4_go<XT, 3>(p, st);
    return hipErrorInvalidConfiguration;
}

}  // namespace

void plan_w4(W4Params &p, int dtype) {
    const int slices = dtype == 1 ? 3 : 1;
    const W4Shape s = kW4Shapes[w4_shape(p, slices)];
    const int64_t blocks = (p.N + 16 * s.rt * s.wn - 1) / (16 * s.rt * s.wn) *
                           ((p.M + 16 * s.tt - 1) / (16 * s.tt));
    const int64_t chunks = (p.K + 127) / 128;
    // workgroups for the CUs, two chunks of work per wave at least
    int64_t splits = 1;
    while (splits < 32 && blocks * splits < 160 && chunks / (2 * splits) >= 2 * s.wk) splits *= 2;
    const int64_t per = (chunks + splits - 1) / splits;
    p.range = (int)(per * 128);
    p.splits = (int)((chunks + per - 1) / per);
    p.part = nullptr;
    // as much of K as the LDS takes, in whole rounds of the waves
    const int step = 128 * s.wk;
    p.held = step;
    while (p.held < p.range) {
        p.held += step;
        if (lds_of(p, s, slices) > s.lds) {
            p.held -= step;
            break;
        }
    }
    if (p.held > p.range) p.held = p.range;
}

hipError_t launch_w4(const W4Params &p, int dtype, hipStream_t st) {
    if (dtype == 1) return w4_run<float>(p, st);
    return dtype == 2 ? w4_run<_Float16>(p, st) : w4_run<__bf16>(p, st);
}

hipError_t launch_quantize_w4(const QuantParams &p, int dtype, hipStream_t st) {
    const int64_t parts = p.N * ((packed_bytes_of(p.K) * 2 + 511) / 512);
    const int64_t blocks = (parts + 3) / 4;
    if (parts >= (int64_t)1 << 31) return hipErrorInvalidConfiguration;
    auto *k = dtype == 1   ? quantize_w4_kernel<float>
              : dtype == 2 ? quantize_w4_kernel<_Float16>
                           : quantize_w4_kernel<__bf16>;
    k<<<dim3((uint32_t)blocks), 256, 0, st>>>(p);
    return hipGetLastError();
}

hipError_t launch_dequantize_w4(const QuantParams &p, int dtype, int sd, hipStream_t st) {
    const int64_t parts = p.N * ((p.K + 511) / 512);
    if (parts >= (int64_t)1 << 31) return hipErrorInvalidConfiguration;
    const dim3 grid((uint32_t)((parts + 3) / 4));
    auto *k = dtype == 1   ? dequantize_w4_kernel<float, float>
              : dtype == 2 ? (sd == 1 ? dequantize_w4_kernel<_Float16, float>
                                      : dequantize_w4_kernel<_Float16, _Float16>)
                           : (sd == 1 ? dequantize_w4_kernel<__bf16, float>
                                      : dequantize_w4_kernel<__bf16, __bf16>);
    k<<<grid, 256, 0, st>>>(p);
    return hipGetLastError();
}

}  // namespace ozk
