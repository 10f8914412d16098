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

// the 8 weights of a word as 16 + q: element order 0, 4, 1, 5, 2, 6, 3, 7
OZK_DEV i32x4 unpack_w4(uint32_t w, _Float16) {   // q << 6 beside fp16's 16.0
    return i32x4{(int)(((w << 6) & 0x03C003C0u) | 0x4C004C00u),
                 (int)(((w << 2) & 0x03C003C0u) | 0x4C004C00u),
                 (int)(((w >> 2) & 0x03C003C0u) | 0x4C004C00u),
                 (int)(((w >> 6) & 0x03C003C0u) | 0x4C004C00u)};
}
OZK_DEV i32x4 unpack_w4(uint32_t w, __bf16) {     // q << 3 beside bf16's 16.0
    return i32x4{(int)(((w << 3) & 0x00780078u) | 0x41804180u),
                 (int)(((w >> 1) & 0x00780078u) | 0x41804180u),
                 (int)(((w >> 5) & 0x00780078u) | 0x41804180u),
                 (int)(((w >> 9) & 0x00780078u) | 0x41804180u)};
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

OZK_DEV float scale_at(const W4Params &p, int64_t i, int dtype16) {
    if (p.scales32) return ((const float *)p.scales)[i];
    const uint16_t u = ((const uint16_t *)p.scales)[i];
    return dtype16 == 2 ? (float)__builtin_bit_cast(_Float16, u) : bf16_bits_to_f32(u);
}

template <typename XT> OZK_DEV float x_value(const char *p) {
    if constexpr (sizeof(XT) == 4) {
        return *(const float *)p;
    } else {
        return from_bits16(*(const uint16_t *)p, XT{});
    }
}

// Waves: WN along n, WK along the chunks of K; a wave has RT blocks of 16 n
// and TT blocks of 16 rows of x; GPC groups per chunk of 128 k.
template <typename XT, int WN, int WK, int RT, int TT, int GPC>
__global__ __launch_bounds__(64 * WN * WK) void w4_kernel(W4Params p) {
    using MT = typename W4Type<XT>::M;
    constexpr int SL = W4Type<XT>::SL, NT = 64 * WN * WK, U = RT == 1 ? 4 : 2;
    constexpr int AC = SL > 1 ? 2 : 1;   // sums of the first slice and of the others, apart
    constexpr int D16 = std::is_same<XT, _Float16>::value ? 2 : 3;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wn = wave / WK, wk = wave % WK, g = lane >> 4, i16 = lane & 15;

    const int64_t nb = (int64_t)blockIdx.x * (16 * RT * WN) + wn * 16 * RT;
    const int64_t m0 = (int64_t)blockIdx.y * (16 * TT);
    const int rows = (int)(p.M - m0 < 16 * TT ? p.M - m0 : 16 * TT);
    const int64_t kbeg = (int64_t)blockIdx.z * p.range;
    const int64_t kend = kbeg + p.range < p.K ? kbeg + p.range : p.K;

    // x in the LDS: [slice][row][k], then the groups' sums [group][16 TT rows]
    const int pitch = p.held * 2 + 16;
    const int slice_bytes = rows * pitch;
    float *sums = (float *)(smem + SL * slice_bytes);
    const int sums_each = p.held / p.group * 16 * TT;   // [AC] of them

    int64_t nrow[RT];
    const uint8_t *wrow[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        const int64_t n = nb + 16 * r + i16;
        nrow[r] = n < p.N ? n : p.N - 1;
        wrow[r] = p.packed + nrow[r] * p.w_pitch;
    }

    f32x4 acc[RT][TT];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int t = 0; t < TT; ++t) acc[r][t] = f32x4{0.f, 0.f, 0.f, 0.f};

    struct Chunk {
        i32x4 w[RT];
        float s[RT][GPC], z[RT][GPC];
    };
    const int64_t pieces = (p.K + 31) / 32;          // 16-byte pieces of a row
    const int64_t groups = (p.K + p.group - 1) / p.group;
    auto load = [&](int64_t c, Chunk &ch) {          // chunk c: k from 128 c on
        const int64_t piece = c * 4 + g;
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            ch.w[r] = piece < pieces ? *(const i32x4 *)(wrow[r] + piece * 16) : i32x4{0, 0, 0, 0};
#pragma unroll
            for (int q = 0; q < GPC; ++q) {
                const int64_t gi = c * GPC + q < groups ? c * GPC + q : groups - 1;
                ch.s[r][q] = scale_at(p, nrow[r] * p.s_pitch + gi, D16);
                ch.z[r][q] = p.zeros ? 16.f + (float)p.zeros[nrow[r] * p.z_pitch + gi] : 24.f;
            }
        }
    };

    for (int64_t k0 = kbeg; k0 < kend; k0 += p.held) {
        const int64_t kstop = k0 + p.held < kend ? k0 + p.held : kend;
        const int64_t c0 = k0 / 128 + wk, c1 = (kstop + 127) / 128;
        Chunk cur[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (c0 + u * WK < c1) load(c0 + u * WK, cur[u]);

        if (k0 != kbeg) __syncthreads();             // the last part of x has been read
        // x: 8 elements a lane, in the order of the unpacked weights, zeros past K
        const int per_row = (int)((kstop - k0 + 127) / 128 * 16);
        const int all = rows * per_row;
        for (int i = threadIdx.x; i < (all + NT - 1) / NT * NT; i += NT) {
            const int row = i < all ? i / per_row : rows - 1, at = i - row * per_row;
            float v[8], sum[AC] = {};
            const char *from = p.x + ((m0 + row) * p.x_pitch + k0 + at * 8) * (int64_t)sizeof(XT);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                v[e] = i < all && k0 + at * 8 + e < p.K ? x_value<XT>(from + e * sizeof(XT)) : 0.f;
                if constexpr (SL > 1) {
                    const float h = from_bits16(to_bits16(v[e], MT{}), MT{});
                    sum[0] += h;
                    sum[1] += v[e] - h;
                } else {
                    sum[0] += v[e];
                }
            }
            if (i < all) {
#pragma unroll
                for (int s = 0; s < SL; ++s) {
                    uint16_t h[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        h[(e & 3) * 2 + (e >> 2)] = to_bits16(v[e], MT{});
                        if (SL > 1) v[e] -= from_bits16(h[(e & 3) * 2 + (e >> 2)], MT{});
                    }
                    i32x4 u;
                    __builtin_memcpy(&u, h, 16);
                    *(i32x4 *)(smem + s * slice_bytes + row * pitch + at * 16) = u;
                }
            }
#pragma unroll
            for (int a = 0; a < AC; ++a) {
#pragma unroll
                for (int d = 1; d < 16 / GPC; d <<= 1) sum[a] += __shfl_xor(sum[a], d);
                if (i < all && at % (16 / GPC) == 0)
                    sums[a * sums_each + at / (16 / GPC) * 16 * TT + row] = sum[a];
            }
        }
        __syncthreads();

        for (int64_t c = c0; c < c1; c += U * WK) {
            Chunk nxt[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (c + (U + u) * WK < c1) load(c + (U + u) * WK, nxt[u]);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t cu = c + u * WK;
                if (cu >= c1) break;
                const int kl = (int)(cu * 128 - k0);   // of the chunk, in the LDS
                uint32_t w[RT][4];
#pragma unroll
                for (int r = 0; r < RT; ++r) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) w[r][j] = (uint32_t)cur[u].w[r][j];
                    transpose_words(w[r]);
                }
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
#pragma unroll
                    for (int t = 0; t < TT; ++t) {
                        const float *xs = sums + (kl / 128 * GPC + q) * 16 * TT + 16 * t + 4 * g;
                        f32x4 x0 = *(const f32x4 *)xs, x1 = x0;
                        if constexpr (AC > 1) x1 = *(const f32x4 *)(xs + sums_each);
#pragma unroll
                        for (int r = 0; r < RT; ++r)
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const float z = cur[u].z[r][q];
                                float v = __builtin_fmaf(-z, x0[e], part[0][r][t][e]);
                                if constexpr (AC > 1)
                                    v += __builtin_fmaf(-z, x1[e], part[1][r][t][e]);
                                acc[r][t][e] = __builtin_fmaf(cur[u].s[r][q], v, acc[r][t][e]);
                            }
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) cur[u] = nxt[u];
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
                const float v = acc[r][t][e];
                if (p.splits > 1) {
                    p.part[((int64_t)blockIdx.z * p.M + m0 + row) * p.N + n] = v;
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
        const int64_t m = i / p.N, n = i - m * p.N;
        if constexpr (sizeof(XT) == 4) ((float *)p.y)[m * p.y_pitch + n] = v;
        else ((uint16_t *)p.y)[m * p.y_pitch + n] = to_bits16(v, XT{});
    }
}

// ---------------------------------------------------------------------------
// The format.  Symmetric: s = fl(max |w| fl(1 / 7)), z = 8; with zero points: s =
// fl((max(w, 0) - min(w, 0)) fl(1 / 15)), z = rint(-min(w, 0) / s).  q = rint(w / s)
// + z within 0 .. 15; a group of zeros has s = 0 and q = z.  NaN counts as 0.
// ---------------------------------------------------------------------------
template <typename T> OZK_DEV float load_value(const char *p, int64_t i) {
    if constexpr (sizeof(T) == 4) return ((const float *)p)[i];
    else return from_bits16(((const uint16_t *)p)[i], T{});
}
template <typename T> OZK_DEV void store_value(char *p, int64_t i, float v) {
    if constexpr (sizeof(T) == 4) ((float *)p)[i] = v;
    else ((uint16_t *)p)[i] = to_bits16(v, T{});
}
template <typename T> OZK_DEV float rounded(float v) {
    if constexpr (sizeof(T) == 4) return v;
    else return from_bits16(to_bits16(v, T{}), T{});
}

// 8 weights a lane: a group is 4, 8 or 16 lanes, a wave 512 weights of a row
template <typename T> __global__ __launch_bounds__(256) void quantize_w4_kernel(QuantParams p) {
    const int64_t per_row = (p.p_pitch * 2 + 511) / 512;
    const int64_t wave = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 6;
    const int lane = threadIdx.x & 63;
    const int64_t n = wave / per_row, k = (wave - n * per_row) * 512 + lane * 8;
    if (n >= p.N) return;
    float v[8], lo = 0.f, hi = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        v[e] = k + e < p.K ? load_value<T>(p.W, n * p.w_pitch + k + e) : 0.f;
        lo = fminf(lo, v[e]);     // (of a number and NaN the number)
        hi = fmaxf(hi, v[e]);
    }
    for (int d = 1; d < p.group / 8; d <<= 1) {
        lo = fminf(lo, __shfl_xor(lo, d));
        hi = fmaxf(hi, __shfl_xor(hi, d));
    }
    float s, z = 8.f;
    if (p.zeros) {
        s = rounded<T>((hi - lo) * (1.f / 15.f));
        z = s > 0.f ? fminf(fmaxf(rintf(-lo / s), 0.f), 15.f) : 0.f;
    } else {
        s = rounded<T>(fmaxf(hi, -lo) * (1.f / 7.f));
    }
    uint32_t word = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        float q = s > 0.f ? rintf(v[e] / s) : 0.f;
        if (q != q) q = 0.f;
        q = fminf(fmaxf(q + z, 0.f), 15.f);
        word |= (uint32_t)(int)q << (4 * e);
    }
    if (k < p.K && k % p.group == 0) {
        store_value<T>(p.scales, n * p.s_pitch + k / p.group, s);
        if (p.zeros) p.zeros[n * p.z_pitch + k / p.group] = (uint8_t)(int)z;
    }
    if (k / 2 < p.p_pitch) *(uint32_t *)(p.packed + n * p.p_pitch + k / 2) = word;
}

template <typename T, typename ST>
__global__ __launch_bounds__(256) void dequantize_w4_kernel(QuantParams p) {
    const int64_t per_row = (p.K + 7) / 8;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t n = i / per_row, k = (i - n * per_row) * 8;
    if (n >= p.N) return;
    const uint32_t word = *(const uint32_t *)(p.packed + n * p.p_pitch + k / 2);
    const float s = load_value<ST>(p.scales, n * p.s_pitch + k / p.group);
    const float z = p.zeros ? (float)p.zeros[n * p.z_pitch + k / p.group] : 8.f;
    const int64_t at = n * p.w_pitch + k;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = ((float)((word >> (4 * e)) & 15u) - z) * s;
    if (sizeof(T) == 2 && k + 8 <= p.K && ((uintptr_t)(p.out + at * 2) & 15) == 0) {
        uint16_t h[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) h[e] = sizeof(T) == 2 ? to_bits16(v[e], std::conditional_t<sizeof(T) == 2, T, __bf16>{}) : 0;
        i32x4 u;
        __builtin_memcpy(&u, h, 16);
        *(i32x4 *)(p.out + at * 2) = u;
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (k + e < p.K) store_value<T>(p.out, at + e, v[e]);
    }
}

namespace {

constexpr int kHeldBytes = 64 * 1024;   // of x in the LDS: two workgroups a CU

struct W4Shape { int wn, wk, rt, tt; };
W4Shape w4_shape(int64_t M) {
    if (M <= 4) return {1, 4, 1, 1};
    if (M <= 16) return {4, 1, 1, 1};
    if (M <= 32) return {4, 1, 2, 2};
    return {4, 1, 2, 4};
}
int lds_of(const W4Params &p, const W4Shape &s, int slices) {
    const int rows = (int)(p.M < 16 * s.tt ? p.M : 16 * s.tt);
    const int sums = p.held / p.group * 16 * s.tt * 4 * (slices > 1 ? 2 : 1);
    const int x = slices * rows * (p.held * 2 + 16) + sums;
    const int join = (s.wk - 1) * s.wn * s.rt * s.tt * 64 * 16;
    return x > join ? x : join;
}

template <typename XT, int WN, int WK, int RT, int TT, int GPC>
hipError_t w4_start(const W4Params &p, hipStream_t st) {
    const dim3 grid((uint32_t)((p.N + 16 * RT * WN - 1) / (16 * RT * WN)),
                    (uint32_t)((p.M + 16 * TT - 1) / (16 * TT)), (uint32_t)p.splits);
    const int lds = lds_of(p, {WN, WK, RT, TT}, W4Type<XT>::SL);
    if (hipError_t e = allow_lds<&w4_kernel<XT, WN, WK, RT, TT, GPC>>(lds); e != hipSuccess)
        return e;
    w4_kernel<XT, WN, WK, RT, TT, GPC><<<grid, 64 * WN * WK, lds, st>>>(p);
    return hipGetLastError();
}

template <typename XT, int WN, int WK, int RT, int TT>
hipError_t w4_go(const W4Params &p, hipStream_t st) {
    const hipError_t e = p.group == 32   ? w4_start<XT, WN, WK, RT, TT, 4>(p, st)
                         : p.group == 64 ? w4_start<XT, WN, WK, RT, TT, 2>(p, st)
                                         : w4_start<XT, WN, WK, RT, TT, 1>(p, st);
    if (e != hipSuccess || p.splits == 1) return e;
    const int64_t blocks = (p.M * p.N + 255) / 256;
    w4_join_kernel<XT><<<dim3((uint32_t)(blocks < 1024 ? blocks : 1024)), 256, 0, st>>>(p);
    return hipGetLastError();
}

template <typename XT> hipError_t w4_run(const W4Params &p, hipStream_t st) {
    if (p.M <= 4) return w4_go<XT, 1, 4, 1, 1>(p, st);
    if (p.M <= 16) return w4_go<XT, 4, 1, 1, 1>(p, st);
    if (p.M <= 32) return w4_go<XT, 4, 1, 2, 2>(p, st);
    return w4_go<XT, 4, 1, 2, 4>(p, st);
}

}  // namespace

void plan_w4(W4Params &p, int dtype) {
    const W4Shape s = w4_shape(p.M);
    const int slices = dtype == 1 ? 3 : 1;
    const int64_t rows = p.M < 16 * s.tt ? p.M : 16 * s.tt;
    const int64_t blocks = (p.N + 16 * s.rt * s.wn - 1) / (16 * s.rt * s.wn) *
                           ((p.M + 16 * s.tt - 1) / (16 * s.tt));
    const int64_t chunks = (p.K + 127) / 128;
    // enough workgroups for every CU, two chunks of work per wave at least
    int64_t splits = 1;
    while (splits < 32 && blocks * splits < 256 && chunks / (2 * splits) >= 2 * s.wk) splits *= 2;
    const int64_t per = (chunks + splits - 1) / splits;
    p.range = (int)(per * 128);
    p.splits = (int)((chunks + per - 1) / per);
    int64_t held = kHeldBytes / (slices * rows * 2 + 2 * s.tt) / (128 * s.wk) * (128 * s.wk);
    if (held < 128 * s.wk) held = 128 * s.wk;
    p.held = (int)(held < p.range ? held : p.range);
    p.part = nullptr;
}

hipError_t launch_w4(const W4Params &p, int dtype, hipStream_t st) {
    if (dtype == 1) return w4_run<float>(p, st);
    return dtype == 2 ? w4_run<_Float16>(p, st) : w4_run<__bf16>(p, st);
}

hipError_t launch_quantize_w4(const QuantParams &p, int dtype, hipStream_t st) {
    const int64_t waves = p.N * ((p.p_pitch * 2 + 511) / 512);
    const int64_t blocks = (waves + 3) / 4;
    if (blocks >= (int64_t)1 << 31) return hipErrorInvalidConfiguration;
    auto *k = dtype == 1   ? quantize_w4_kernel<float>
              : dtype == 2 ? quantize_w4_kernel<_Float16>
                           : quantize_w4_kernel<__bf16>;
    k<<<dim3((uint32_t)blocks), 256, 0, st>>>(p);
    return hipGetLastError();
}

hipError_t launch_dequantize_w4(const QuantParams &p, int dtype, int sd, hipStream_t st) {
    const int64_t blocks = (p.N * ((p.K + 7) / 8) + 255) / 256;
    if (blocks >= (int64_t)1 << 31) return hipErrorInvalidConfiguration;
    const dim3 grid((uint32_t)blocks);
    auto *k = dtype == 1   ? dequantize_w4_kernel<float, float>
              : dtype == 2 ? (sd == 1 ? dequantize_w4_kernel<_Float16, float>
                                      : dequantize_w4_kernel<_Float16, _Float16>)
                           : (sd == 1 ? dequantize_w4_kernel<__bf16, float>
                                      : dequantize_w4_kernel<__bf16, __bf16>);
    k<<<grid, 256, 0, st>>>(p);
    return hipGetLastError();
}

}  // namespace ozk
