// ozk_tile.h -- one C tile of a 16-bit matrix product on the matrix cores, for
// the grouped products (ozk_grouped.hip) and the orthogonalisation
// (ozk_orth.hip).
//
//   C[m, n] = sum_k A[m, k] B[n, k], accumulated in fp32
//
// An operand is read in one of two layouts: "rows", K-contiguous rows of A or
// of B^T, or "cols", whose rows run along K and hold consecutive m (n).  With
// S = 2 an element is the sum of two fp16 slices h + l of one scale, and the
// slice pairs hh, hl, lh are summed (ll is of the size of the slices' own
// rounding); 64 bytes of h and 64 bytes of l alternate in memory, so a
// 128-byte line holds both slices of 32 elements and the staging below is the
// same for both.
//
// A stage holds 128 bytes of K per row (S = 1: 64 elements, S = 2: 32 with
// both slices) of BM rows of A and BN rows of B, and is fetched by LDS-DMA in
// windows of 1 KB, one per wave instruction, into a ring of NST slots; where
// rows are not whole aligned 16-byte pieces the same windows go through
// registers (DMA = false).  "rows" are kept as 128-byte LDS rows, 16-byte
// chunks XORed with the row so that a 16-row fragment read (ds_read_b128)
// touches every bank once; "cols" as they come, read by ds_read_b64_tr_b16,
// which gives lane i of 16 the column i of 4 rows of 16 elements, 32-byte
// chunks XORed with the row to the same end.
//
// The MFMA is v_mfma_f32_16x16x32 with B's fragment first: a lane then holds 4
// consecutive n of one row m, stored with one instruction.
#pragma once

#include <type_traits>

#include "ozk_common.h"

namespace ozk {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));

OZK_DEV f32x4 mfma16(i32x4 a, i32x4 b, f32x4 c, _Float16) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
OZK_DEV f32x4 mfma16(i32x4 a, i32x4 b, f32x4 c, __bf16) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// fp32 -> 16 bits, to nearest even (NaN stays NaN)
OZK_DEV uint16_t to_bits16(float v, _Float16) { return __builtin_bit_cast(uint16_t, (_Float16)v); }
OZK_DEV uint16_t to_bits16(float v, __bf16) {
    return (uint16_t)(v != v ? 0x7FC0u : f32_to_bf16_bits(v));
}
OZK_DEV float from_bits16(uint16_t v, _Float16) { return (float)__builtin_bit_cast(_Float16, v); }
OZK_DEV float from_bits16(uint16_t v, __bf16) { return bf16_bits_to_f32(v); }

// An operand's part that a tile reads.
struct TileSrc {
    const char *base;   // its first row at k = 0 ("cols": the first column, at row k = 0)
    int64_t pitch;      // bytes between rows
    int rows;           // "rows": rows there are; "cols": bytes of a row there are
    int64_t klen;       // "rows": bytes of K; "cols": rows
};

constexpr uint32_t kTileOOB = 0x80000000u;   // past every buffer: the DMA writes zeros

template <int S_, bool ACOLS_, bool BCOLS_, int BM_, int BN_, int WM_, int WN_, int NST_>
struct TileShape {
    static constexpr int S = S_, BM = BM_, BN = BN_, WM = WM_, WN = WN_, NST = NST_;
    static constexpr bool ACOLS = ACOLS_, BCOLS = BCOLS_;
    static constexpr int WAVES = WM * WN, THREADS = 64 * WAVES;
    static constexpr int KS = 64 / S;                 // elements of K per stage
    static constexpr int MI = BM / WM / 16, NI = BN / WN / 16;
    static constexpr int A_BYTES = BM * 128, STAGE = (BM + BN) * 128;
    static constexpr int LP = STAGE / 1024 / WAVES;   // windows per wave and stage
    static constexpr int LDS_BYTES = NST * STAGE;
    static_assert(LP * WAVES * 1024 == STAGE, "windows split evenly over the waves");
    static_assert(BM % (16 * WM) == 0 && BN % (16 * WN) == 0, "whole 16 x 16 blocks");
    static_assert(LDS_BYTES <= 160 * 1024, "LDS");
};

// "cols" operands of BX columns: an LDS row (one k) is RB bytes
template <int S, int BX> struct ColsRow { static constexpr int RB = BX * 2 * S; };

// XOR of the 32-byte chunk of LDS row k: the 8 rows that 32 lanes of a
// transposing read touch (k = 0..3 and 8..11 and so on) fall into 8 different
// bank groups
template <int RB> OZK_DEV int cols_swz(int k) {
    if constexpr (RB >= 256) return (k & 3) | ((k >> 1) & 4);
    else if constexpr (RB == 128) return ((k >> 1) & 1) | ((k >> 2) & 2);
    else return (k >> 3) & 1;
}

// Where lane `lane` of 1 KB window w of an operand reads: byte offset from the
// stage's base, and its place along K (bytes of the 128 for "rows", the row
// for "cols") with which the last stage is cut.
struct WindowAt {
    uint32_t off;
    int k;
};
template <int S, bool COLS, int BX> OZK_DEV WindowAt window_at(const TileSrc &s, int w, int lane) {
    if constexpr (!COLS) {
        const int row = 8 * w + (lane >> 3);
        const int k = ((lane & 7) ^ ((row >> 1) & 7)) * 16;
        return {row < s.rows ? (uint32_t)(row * s.pitch) + k : kTileOOB, k};
    } else {
        constexpr int RB = ColsRow<S, BX>::RB;
        const int pos = w * 64 + lane;
        const int k = pos / (RB / 16), c16 = pos % (RB / 16);
        const int col = (((c16 >> 1) ^ cols_swz<RB>(k)) << 5) + (c16 & 1) * 16;
        return {col < s.rows ? (uint32_t)(k * s.pitch) + col : kTileOOB, k};
    }
}

// 16 bytes at an address of any alignment, of which the first `n` exist
OZK_DEV i32x4 load_piece(const char *p, int n) {
    i32x4 v = {0, 0, 0, 0};
    if (n >= 16) {
        __builtin_memcpy(&v, p, 16);
    } else {
        uint16_t e[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            e[i] = 0;
            if (2 * i < n) __builtin_memcpy(&e[i], p + 2 * i, 2);
        }
        __builtin_memcpy(&v, e, 16);
    }
    return v;
}

template <typename ST, typename Sh, bool DMA> struct TileLoop {
    static constexpr int S = Sh::S, LP = Sh::LP, MI = Sh::MI, NI = Sh::NI;
    f32x4 acc[MI][NI];

    OZK_DEV void run(const TileSrc &A, const TileSrc &B, char *smem) {
        const int lane = threadIdx.x & 63;
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const int wm = wave / Sh::WN, wn = wave % Sh::WN;
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < NI; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

        const int64_t ka = Sh::ACOLS ? Sh::KS : 128, kb_ = Sh::BCOLS ? Sh::KS : 128;
        const int nka = (int)((A.klen + ka - 1) / ka), nkb_b = (int)((B.klen + kb_ - 1) / kb_);
        const int nkb = nka < nkb_b ? nka : nkb_b;
        const int64_t stepA = Sh::ACOLS ? Sh::KS * A.pitch : 128;
        const int64_t stepB = Sh::BCOLS ? Sh::KS * B.pitch : 128;

        WindowAt win[LP];
#pragma unroll
        for (int q = 0; q < LP; ++q) {
            const int w = wave * LP + q;
            win[q] = w < Sh::BM / 8
                         ? window_at<S, Sh::ACOLS, Sh::BM>(A, w, lane)
                         : window_at<S, Sh::BCOLS, Sh::BN>(B, w - Sh::BM / 8, lane);
        }

        // what is left of K from stage kb on, as win[].k counts it
        auto left_a = [&](int kb) { return A.klen - kb * ka; };
        auto left_b = [&](int kb) { return B.klen - kb * kb_; };

        auto issue = [&](int kb) {
            char *dst = smem + (kb % Sh::NST) * Sh::STAGE + wave * LP * 1024;
            const __amdgpu_buffer_rsrc_t rA = __builtin_amdgcn_make_buffer_rsrc(
                (void *)(A.base + kb * stepA), (short)0, 0x7FFFFFFF, 0x00020000);
            const __amdgpu_buffer_rsrc_t rB = __builtin_amdgcn_make_buffer_rsrc(
                (void *)(B.base + kb * stepB), (short)0, 0x7FFFFFFF, 0x00020000);
            const int la = (int)(left_a(kb) < ka ? left_a(kb) : ka);
            const int lb = (int)(left_b(kb) < kb_ ? left_b(kb) : kb_);
#pragma unroll
            for (int q = 0; q < LP; ++q) {
                const bool isA = wave * LP + q < Sh::BM / 8;
                const uint32_t off = win[q].k < (isA ? la : lb) ? win[q].off : kTileOOB;
                auto *to = (__attribute__((address_space(3))) void *)(dst + q * 1024);
                __builtin_amdgcn_raw_ptr_buffer_load_lds(isA ? rA : rB, to, 16, off, 0, 0, 0);
            }
        };
        // the same through registers, for rows of any alignment
        i32x4 held[DMA ? 1 : LP];
        auto fetch = [&](int kb) {
#pragma unroll
            for (int q = 0; q < LP; ++q) {
                const bool isA = wave * LP + q < Sh::BM / 8;
                const char *base = isA ? A.base + kb * stepA : B.base + kb * stepB;
                const int64_t left = isA ? left_a(kb) : left_b(kb);
                const bool cols = isA ? Sh::ACOLS : Sh::BCOLS;
                int n = 0;
                if (win[q].off != kTileOOB && win[q].k < left) {
                    if (cols) {
                        // the column is what is left of the offset after its row
                        const int col = (int)(win[q].off - (uint32_t)(win[q].k *
                                                                      (isA ? A.pitch : B.pitch)));
                        n = (isA ? A.rows : B.rows) - col;
                    } else {
                        n = (int)(left - win[q].k < 16 ? left - win[q].k : 16);
                    }
                }
                held[q] = load_piece(base + (n > 0 ? win[q].off : 0u), n);
            }
        };
        auto put = [&](int kb) {
            char *dst = smem + (kb % Sh::NST) * Sh::STAGE + wave * LP * 1024 + lane * 16;
#pragma unroll
            for (int q = 0; q < LP; ++q) *(i32x4 *)(dst + q * 1024) = held[q];
        };

        const int g = lane >> 4, i16 = lane & 15;
        // Fragment (tile t of this wave, step ks) of an operand in LDS region
        // `buf`: S = 1: K step ks of the stage's two; S = 2: slice ks.
        auto frag = [&](const char *buf, auto cols_, auto bx_, int t0, int t, int ks) -> i32x4 {
            constexpr bool cols = decltype(cols_)::value;
            constexpr int BX = decltype(bx_)::value;
            if constexpr (!cols) {
                const int chunk = (4 * ks + g) ^ (i16 >> 1);
                return *(const i32x4 *)(buf + (t0 + t) * 2048 + i16 * 128 + chunk * 16);
            } else {
                constexpr int RB = ColsRow<S, BX>::RB;
                const int tt = t0 + t;
                const int c32 = S == 1 ? tt : (tt >> 1) * 4 + (tt & 1) + 2 * ks;
                const int k = (S == 1 ? 32 * ks : 0) + 8 * g + (i16 >> 2);
                const char *at = buf + k * RB + ((c32 ^ cols_swz<RB>(k)) << 5) + (i16 & 3) * 8;
                using L = __attribute__((address_space(3))) i16x4;
                const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((L *)at);
                const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((L *)(at + 4 * RB));
                const i32x2 a = __builtin_bit_cast(i32x2, lo), b = __builtin_bit_cast(i32x2, hi);
                return i32x4{a.x, a.y, b.x, b.y};
            }
        };
        auto compute = [&](int kb) {
            const char *bufA = smem + (kb % Sh::NST) * Sh::STAGE;
            const char *bufB = bufA + Sh::A_BYTES;
            i32x4 a[2][MI], b[2][NI];
            auto read = [&](int ks) {
#pragma unroll
                for (int j = 0; j < NI; ++j)
                    b[ks][j] = frag(bufB, std::integral_constant<bool, Sh::BCOLS>{},
                                    std::integral_constant<int, Sh::BN>{}, wn * NI, j, ks);
#pragma unroll
                for (int i = 0; i < MI; ++i)
                    a[ks][i] = frag(bufA, std::integral_constant<bool, Sh::ACOLS>{},
                                    std::integral_constant<int, Sh::BM>{}, wm * MI, i, ks);
            };
            auto mul = [&](int ka_, int kb2) {
#pragma unroll
                for (int i = 0; i < MI; ++i)
#pragma unroll
                    for (int j = 0; j < NI; ++j)
                        acc[i][j] = mfma16(b[kb2][j], a[ka_][i], acc[i][j], ST{});
            };
            read(0);
            if constexpr (S == 1) {
                mul(0, 0);
                read(1);
                mul(1, 1);
            } else {
                read(1);
                mul(0, 0);
                mul(0, 1);
                mul(1, 0);
            }
        };

        if constexpr (DMA) {
#pragma unroll
            for (int s = 0; s < Sh::NST - 1; ++s)
                if (s < nkb) issue(s);
            for (int kb = 0; kb < nkb; ++kb) {
                // the stages issued after kb may still be on their way
                const int after = nkb - 1 - kb < Sh::NST - 2 ? nkb - 1 - kb : Sh::NST - 2;
                if (after >= 3) wait_vmcnt<(Sh::NST > 4 ? 3 : 0) * LP>();
                else if (after == 2) wait_vmcnt<(Sh::NST > 3 ? 2 : 0) * LP>();
                else if (after == 1) wait_vmcnt<(Sh::NST > 2 ? 1 : 0) * LP>();
                else wait_vmcnt<0>();
                static_assert(Sh::NST <= 5 && 3 * LP < 64, "wait table");
                __builtin_amdgcn_s_waitcnt(0xC07F);   // this wave's reads of the slot refilled next
                exec_barrier();
                if (kb + Sh::NST - 1 < nkb) issue(kb + Sh::NST - 1);
                compute(kb);
            }
        } else {
            if (nkb > 0) {
                fetch(0);
                put(0);
            }
            for (int kb = 0; kb < nkb; ++kb) {
                __syncthreads();
                if (kb + 1 < nkb) fetch(kb + 1);
                compute(kb);
                // (the slot of kb + 1 was read last in step kb - 1, before the barrier)
                if (kb + 1 < nkb) put(kb + 1);
            }
        }
    }

    // f(m, n, v): the four values v of row m (of the tile), columns n .. n + 3
    template <typename F> OZK_DEV void each(F &&f) const {
        const int lane = threadIdx.x & 63;
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const int m0 = wave / Sh::WN * MI * 16 + (lane & 15);
        const int n0 = wave % Sh::WN * NI * 16 + (lane >> 4) * 4;
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < NI; ++j) f(m0 + 16 * i, n0 + 16 * j, acc[i][j]);
    }
};

// Tile `t` of `total` in the order in which XCD x (workgroups x, x + 8, ..)
// takes the x-th part of the tiles; -1: none
OZK_DEV int64_t xcd_tile(uint32_t block, uint32_t total) {
    const uint32_t per = (total + 7) / 8, i = block / 8;
    const uint32_t t = (block % 8) * per + i;
    return i < per && t < total ? (int64_t)t : -1;
}

}  // namespace ozk
