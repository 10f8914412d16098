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
OZK_DEV uint16_t to_bits16(float v, __bf16) { return __builtin_bit_cast(uint16_t, (__bf16)v); }
OZK_DEV float from_bits16(uint16_t v, _Float16) { return (float)__builtin_bit_cast(_Float16, v); }
OZK_DEV float from_bits16(uint16_t v, __bf16) { return bf16_bits_to_f32(v); }

// element i of fp32 or 16-bit values as fp32, and back
template <typename T> OZK_DEV float load_value(const char *p, int64_t i) {
    if constexpr (sizeof(T) == 4) return ((const float *)p)[i];
    else return from_bits16(((const uint16_t *)p)[i], T{});
}
template <typename T> OZK_DEV void store_value(char *p, int64_t i, float v) {
    if constexpr (sizeof(T) == 4) ((float *)p)[i] = v;
    else ((uint16_t *)p)[i] = to_bits16(v, T{});
}

// i / n for 0 <= i < 2^22, n a small part of it: (i + 1/2) / n is at least 1 / 2n
// away from a whole number, the two roundings of rcp * (i + 1/2) less
OZK_DEV int part_of(int i, int n, float rcp) { return (int)(((float)i + 0.5f) * rcp); }

// An operand's part that a tile reads.
struct TileSrc {
    const char *base;   // its first row at k = 0 ("cols": the first column, at row k = 0)
    int64_t pitch;      // bytes between rows
    int rows;           // "rows": rows there are; "cols": bytes of a row there are
    int64_t klen;       // "rows": bytes of K; "cols": rows
    const char *first;  // the whole operand's first byte
};

constexpr uint32_t kTileOOB = 0x80000000u;   // past every buffer: the DMA writes zeros

// KW > 1: so many groups of WM x WN waves, group w takes every KW-th stage from
// w on; the groups' sums are added in order at the end.
template <int S_, bool ACOLS_, bool BCOLS_, int BM_, int BN_, int WM_, int WN_, int NST_,
          int KW_ = 1>
struct TileShape {
    static constexpr int S = S_, BM = BM_, BN = BN_, WM = WM_, WN = WN_, NST = NST_, KW = KW_;
    static constexpr bool ACOLS = ACOLS_, BCOLS = BCOLS_;
    static constexpr int WAVES = WM * WN, THREADS = 64 * WAVES * KW;   // waves of a group
    static constexpr int KS = 64 / S;                 // elements of K per stage
    static constexpr int MI = BM / WM / 16, NI = BN / WN / 16;
    static constexpr int A_BYTES = BM * 128, STAGE = (BM + BN) * 128;
    static constexpr int LP = STAGE / 1024 / WAVES;   // windows per wave and stage
    // a wave's windows are all A's or all B's where that comes out even, else
    // LPA of A's and the others of B's
    static constexpr bool ONE = BM / 8 % LP == 0;
    static constexpr int LPA = ONE ? 0 : BM / 8 / WAVES;
    static_assert(ONE || (BM / 8 % WAVES == 0 && BN / 8 % WAVES == 0), "windows per operand");
    static constexpr int SLOT = KW * STAGE, JOIN = (KW - 1) * WAVES * MI * NI * 1024;
    static constexpr int LDS_BYTES = NST * SLOT > JOIN ? NST * SLOT : JOIN;
    // waves per SIMD that the registers have to leave room for
    static constexpr int PER_SIMD = 2;
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
    static_assert((RB & (RB - 1)) == 0, "the XOR leaves a chunk in its row");
    if constexpr (RB >= 256) return (k & 3) | ((k >> 1) & 4);
    else if constexpr (RB == 128) return ((k >> 1) & 1) | ((k >> 2) & 2);
    else return (k >> 3) & 1;
}

// a value that is the same in every lane, in scalar registers: the DMA's buffer
// descriptor and destination have to be there
OZK_DEV int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
OZK_DEV int64_t uniform(int64_t v) {
    const uint32_t lo = (uint32_t)uniform((int)(uint32_t)v);
    return (int64_t)(((uint64_t)(uint32_t)uniform((int)(v >> 32)) << 32) | lo);
}

// Where lane `lane` of 1 KB window w of an operand reads: byte offset from the
// stage's base, its place along K (bytes of the 128 for "rows", the row for
// "cols") with which the last stage is cut, and how many bytes there are
// ("rows": before that cut).
struct WindowAt {
    uint32_t off;
    int k, n;
};
template <int S, bool COLS, int BX> OZK_DEV WindowAt window_at(const TileSrc &s, int w, int lane) {
    if constexpr (!COLS) {
        const int row = 8 * w + (lane >> 3);
        const int k = ((lane & 7) ^ ((row >> 1) & 7)) * 16;
        const bool ok = row < s.rows;
        return {ok ? (uint32_t)(row * s.pitch) + k : kTileOOB, k, ok ? 16 : 0};
    } else {
        constexpr int RB = ColsRow<S, BX>::RB;
        const int pos = w * 64 + lane;
        const int k = pos / (RB / 16), c16 = pos % (RB / 16);
        const int col = (((c16 >> 1) ^ cols_swz<RB>(k)) << 5) + (c16 & 1) * 16;
        const int n = s.rows - col < 0 ? 0 : s.rows - col < 16 ? s.rows - col : 16;
        return {n > 0 ? (uint32_t)(k * s.pitch) + col : kTileOOB, k, n};
    }
}

// One LDS-DMA instruction: 16 bytes per lane from `base` + off to LDS byte `to`
// + PLUS + 16 * lane; zeros where off is past the 2 GiB behind base.  Written in
// assembly because behind the builtin the compiler waits for every DMA on its
// way before a ds_read_b64_tr_b16 (measured: 1028 us against 815 without the
// read-ahead below, 32768 x 2048 x 4096).  It has no register result; its LDS
// writes are waited for by wait_vmcnt and a barrier like the builtin's.  Nor
// does the compiler see that it reads the descriptor: a vector-memory
// instruction may do so from five wait states after a vector instruction wrote
// it on, and a v_readfirstlane can stand right before this block, so the five
// are in it: the addition, which m0 needs too, and the s_nop.
template <int PLUS> OZK_DEV void dma_piece(const char *base, uint32_t off, uint32_t to) {
    const uint64_t at = (uint64_t)(uintptr_t)base;
    const i32x4 desc = {uniform((int)(uint32_t)at), uniform((int)(uint32_t)(at >> 32)), 0x7FFFFFFF,
                        0x00020000};
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"   // m0 holds nothing else in these kernels
    asm volatile("s_add_u32 m0, %0, %3\n\ts_nop 3\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                 :
                 : "s"(uniform((int)to)), "v"(off), "s"(desc), "n"(PLUS)
                 : "memory", "m0", "scc");
#pragma clang diagnostic pop
}

// 16 bytes built element by element, the last first: a rolled loop, since code
// that is fetched and skipped costs short kernels more
OZK_DEV void push16(i32x4 &v, uint32_t e) {
    v.w = (int)__builtin_amdgcn_alignbit((uint32_t)v.w, (uint32_t)v.z, 16);
    v.z = (int)__builtin_amdgcn_alignbit((uint32_t)v.z, (uint32_t)v.y, 16);
    v.y = (int)__builtin_amdgcn_alignbit((uint32_t)v.y, (uint32_t)v.x, 16);
    v.x = (int)(((uint32_t)v.x << 16) | e);
}

// 16 bytes from an address of any alignment on, of which the first `n` (even)
// exist; `first`: the operand's first byte.  A piece with an end inside is read
// up to that end, from what lies before it, and shifted down: its elements one
// by one cost the edge tiles more than everything else (19944 x 220 x 103 in 5
// groups, dB: 264 us).
OZK_DEV i32x4 load_piece(const char *p, int n, const char *first) {
    i32x4 v = {0, 0, 0, 0};
    if (n >= 16) {
        __builtin_memcpy(&v, p, 16);
    } else if (n > 0) {
        const int s = 16 - n;
        if (p - first >= s) {
            __builtin_memcpy(&v, p - s, 16);
            if (s & 8) v = i32x4{v.z, v.w, 0, 0};
            if (s & 4) v = i32x4{v.y, v.z, v.w, 0};
            const uint32_t h = (uint32_t)(s & 2) * 8;
            v = i32x4{(int)__builtin_amdgcn_alignbit((uint32_t)v.y, (uint32_t)v.x, h),
                      (int)__builtin_amdgcn_alignbit((uint32_t)v.z, (uint32_t)v.y, h),
                      (int)__builtin_amdgcn_alignbit((uint32_t)v.w, (uint32_t)v.z, h),
                      (int)((uint32_t)v.w >> h)};
        } else {
#pragma unroll 1
            for (int i = n / 2 - 1; i >= 0; --i) push16(v, ((const uint16_t *)p)[i]);
        }
    }
    return v;
}

template <int N, typename F> OZK_DEV void static_for_tile(F &&f) {
    if constexpr (N > 0) {
        static_for_tile<N - 1>(f);
        f(std::integral_constant<int, N - 1>{});
    }
}

template <typename ST, typename Sh, bool DMA> struct TileLoop {
    static constexpr int S = Sh::S, LP = Sh::LP, MI = Sh::MI, NI = Sh::NI;
    f32x4 acc[MI][NI];

    // All waves; false in the waves whose sums another one has taken over.
    OZK_DEV bool run(const TileSrc &A, const TileSrc &B, char *smem) {
        const int lane = threadIdx.x & 63;
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) % Sh::WAVES;
        const int kw = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) / Sh::WAVES;
        const int wm = wave / Sh::WN, wn = wave % Sh::WN;
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < NI; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

        constexpr int ua = Sh::ACOLS ? Sh::KS : 128, ub = Sh::BCOLS ? Sh::KS : 128;
        const int nka = (int)((A.klen + ua - 1) / ua), nkb_b = (int)((B.klen + ub - 1) / ub);
        const int nkb = ((nka < nkb_b ? nka : nkb_b) + Sh::KW - 1) / Sh::KW;   // of each group

        // the operands as this wave stages them, `base` that of the stage it is at
        struct Feed {
            const char *base, *first;
            int64_t step;
            int whole, rest;   // whole stages, and what the one behind them has of K
            int slot;          // its first window's place in a stage
            // what the group's stage kb has of K, as WindowAt counts it
            OZK_DEV int left(int kb, int kw) const {
                const int at = kb * Sh::KW + kw;
                return at < whole ? 128 : at == whole ? rest : 0;
            }
        };
        constexpr int LPB = LP - Sh::LPA;
        Feed fa = {A.base, A.first, Sh::ACOLS ? Sh::KS * A.pitch : 128, (int)(A.klen / ua),
                   (int)(A.klen % ua), wave * (Sh::ONE ? LP : Sh::LPA) * 1024};
        Feed fb = {B.base, B.first, Sh::BCOLS ? Sh::KS * B.pitch : 128, (int)(B.klen / ub),
                   (int)(B.klen % ub), (Sh::ONE ? wave * LP : Sh::BM / 8 + wave * LPB) * 1024};
        if constexpr (Sh::KW > 1) {
            fa.base += kw * fa.step;
            fb.base += kw * fb.step;
            fa.step *= Sh::KW;
            fb.step *= Sh::KW;
        }
        // in scalar registers from here on, not moved there for every window
        for (Feed *f : {&fa, &fb}) {
            f->base = (const char *)uniform((int64_t)(uintptr_t)f->base);
            f->step = uniform(f->step);
        }
        const bool onlyA = Sh::ONE && wave * LP < Sh::BM / 8;
        Feed feed[Sh::ONE ? 1 : 2];
        if constexpr (Sh::ONE) {
            feed[0] = onlyA ? fa : fb;
        } else {
            feed[0] = fa;
            feed[1] = fb;
        }
        constexpr auto of = [](int q) { return Sh::ONE || q < Sh::LPA ? 0 : 1; };   // window q's feed
        // and its place among the feed's
        constexpr auto nth = [](int q) { return Sh::ONE || q < Sh::LPA ? q : q - Sh::LPA; };
        WindowAt win[LP];
#pragma unroll
        for (int q = 0; q < LP; ++q) {
            if constexpr (Sh::ONE) {
                const int w = wave * LP + q;
                win[q] = onlyA ? window_at<S, Sh::ACOLS, Sh::BM>(A, w, lane)
                               : window_at<S, Sh::BCOLS, Sh::BN>(B, w - Sh::BM / 8, lane);
            } else {
                win[q] = of(q) == 0 ? window_at<S, Sh::ACOLS, Sh::BM>(A, wave * Sh::LPA + nth(q), lane)
                                    : window_at<S, Sh::BCOLS, Sh::BN>(B, wave * LPB + nth(q), lane);
            }
        }
        auto advance = [&] {
#pragma unroll
            for (Feed &f : feed) f.base += f.step;
        };

        // Stage kb, which is the next one: the last whole one is followed by one
        // whose windows are cut, and then by empty ones (of a group of waves)
        auto begin = [&](int kb) {
            if (kb > 0) advance();
#pragma unroll
            for (int f = 0; f < (Sh::ONE ? 1 : 2); ++f) {
                const int left = feed[f].left(kb, kw);
                if (left < 128)
#pragma unroll
                    for (int q = 0; q < LP; ++q)
                        if (of(q) == f && win[q].k >= left) win[q].off = kTileOOB;
            }
        };
        // and windows Q0 .. Q1 of it
        const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)smem +
                             kw * Sh::STAGE;
        auto issue = [&](int kb, auto q0_, auto q1_) {
            constexpr int Q0 = decltype(q0_)::value, Q1 = decltype(q1_)::value;
            const uint32_t dst = lds + (uint32_t)kb % Sh::NST * Sh::SLOT;
            static_for_tile<Q1 - Q0>([&](auto q_) {
                constexpr int q = Q0 + decltype(q_)::value;
                const Feed &f = feed[of(q)];
                dma_piece<nth(q) * 1024>(f.base, win[q].off, dst + (uint32_t)f.slot);
            });
        };
        // the same through registers, for rows of any alignment
        i32x4 held[DMA ? 1 : LP];
        auto fetch = [&](int kb) {
            if (kb > 0) advance();
#pragma unroll
            for (int q = 0; q < LP; ++q) {
                const Feed &f = feed[of(q)];
                const bool cols = Sh::ONE ? (onlyA ? Sh::ACOLS : Sh::BCOLS)
                                          : (of(q) == 0 ? Sh::ACOLS : Sh::BCOLS);
                const int left = f.left(kb, kw) - win[q].k;
                int n = left > 0 ? win[q].n : 0;
                if (!cols && left < n) n = left;
                held[q] = load_piece(f.base + (n > 0 ? win[q].off : 0u), n, f.first);
            }
        };
        auto put = [&](int kb) {
            char *dst = smem + ((uint32_t)kb % Sh::NST) * Sh::SLOT + kw * Sh::STAGE + lane * 16;
#pragma unroll
            for (int q = 0; q < LP; ++q) *(i32x4 *)(dst + feed[of(q)].slot + nth(q) * 1024) = held[q];
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
        // A stage is 2 MI groups of MFMAs: group n multiplies A's fragment (step n
        // / MI, block n % MI) with B's.  S = 1: a step is one K step, B's fragments
        // of the step.  S = 2: step 0 is slice h of A with both slices of B, step 1
        // slice l of A with slice h of B.  A's fragments are read two groups ahead
        // into a ring of RA; behind the last read of a stage, two groups before its
        // end, comes the barrier that hands the slot back and the next stage over,
        // so the next stage's first reads run under the last MFMAs.
        constexpr int G = 2 * MI, BG = G - 2, RA = G % 4 == 0 ? 4 : 3;
        static_assert(G % RA == 0, "the ring goes on from stage to stage");
        i32x4 a[RA], b[2][NI], bn[NI];
        auto readA = [&](const char *buf, int n, auto n_) {
            constexpr int N_ = decltype(n_)::value;   // ring place
            a[N_] = frag(buf, std::integral_constant<bool, Sh::ACOLS>{},
                         std::integral_constant<int, Sh::BM>{}, wm * MI, n % MI, n / MI);
        };
        auto readB = [&](const char *buf, int j, int ks) -> i32x4 {
            return frag(buf + Sh::A_BYTES, std::integral_constant<bool, Sh::BCOLS>{},
                        std::integral_constant<int, Sh::BN>{}, wn * NI, j, ks);
        };
        auto first = [&](const char *buf) {   // what group 0 of a stage needs
#pragma unroll
            for (int j = 0; j < NI; ++j) b[0][j] = readB(buf, j, 0);
            if constexpr (S == 2)
#pragma unroll
                for (int j = 0; j < NI; ++j) b[1][j] = readB(buf, j, 1);
            readA(buf, 0, std::integral_constant<int, 0>{});
            readA(buf, 1, std::integral_constant<int, 1>{});
        };
        // ready(): stage kb + 1 has landed and every wave has read stage kb;
        // during(n): what else group n issues
        auto stage = [&](int kb, auto &&ready, auto &&during) {
            const char *buf = smem + ((uint32_t)kb % Sh::NST) * Sh::SLOT + kw * Sh::STAGE;
            const char *next = smem + ((uint32_t)(kb + 1) % Sh::NST) * Sh::SLOT + kw * Sh::STAGE;
            static_for_tile<G>([&](auto n_) {
                constexpr int n = decltype(n_)::value, i = n % MI;
                if constexpr (n == BG) ready();
                if constexpr (n + 2 < G) {
                    readA(buf, n + 2, std::integral_constant<int, (n + 2) % RA>{});
                    if constexpr (S == 1 && n < MI) {
                        constexpr int on = MI < BG ? MI : BG, per = (NI + on - 1) / on;
#pragma unroll
                        for (int j = n * per; j < (n + 1) * per && j < NI; ++j)
                            b[1][j] = readB(buf, j, 1);
                    }
                } else {
                    // the next stage's first fragments
                    readA(next, n + 2 - G, std::integral_constant<int, (n + 2) % RA>{});
#pragma unroll
                    for (int j = 0; j < NI; ++j)
                        if (j * 2 / NI == n - BG) {
                            (S == 1 ? b[0][j] : bn[j]) = readB(next, j, 0);
                            if (S == 2) b[1][j] = readB(next, j, 1);
                        }
                }
                during(n_);
                constexpr int r = n % RA;
#pragma unroll
                for (int j = 0; j < NI; ++j)
                    acc[i][j] = mfma16(b[S == 1 ? n / MI : 0][j], a[r], acc[i][j], ST{});
                if constexpr (S == 2 && n < MI)
#pragma unroll
                    for (int j = 0; j < NI; ++j)
                        acc[i][j] = mfma16(b[1][j], a[r], acc[i][j], ST{});
                __builtin_amdgcn_sched_barrier(0);
            });
            if constexpr (S == 2)
#pragma unroll
                for (int j = 0; j < NI; ++j) b[0][j] = bn[j];
        };

        if constexpr (DMA) {
            // NOW windows are issued right after the barrier, the others during the
            // next groups
            constexpr int NOW = LP < 2 ? LP : 2, NST = Sh::NST;
            static_assert((NST - 1) * LP < 64, "vmcnt");
            constexpr std::integral_constant<int, 0> Q0;
            constexpr std::integral_constant<int, NOW> QN;
            constexpr std::integral_constant<int, LP> QE;
#pragma unroll
            for (int s = 0; s < NST; ++s) {
                if (s >= nkb) continue;
                begin(s);
                if (s < NST - 1) issue(s, Q0, QE);
                else issue(s, Q0, QN);
            }
            if (nkb > 0) {
                // the first has landed; few stages: all have
                if (nkb >= NST) wait_vmcnt<(NST - 2) * LP + NOW>();
                else wait_vmcnt<0>();
                exec_barrier();
                first(smem + kw * Sh::STAGE);
            }
            // all: stages kb + NST - 1 and kb + NST exist
            auto one = [&](int kb, auto all_) {
                constexpr bool all = decltype(all_)::value;
                stage(
                    kb,
                    [&] {
                        // kb + 1 has landed; the last stages, on their way for a
                        // while, all have
                        if (all || kb + NST <= nkb) wait_vmcnt<(NST - 2) * LP>();
                        else wait_vmcnt<0>();
                        __builtin_amdgcn_s_waitcnt(0xC07F);   // this wave's reads of the slot
                        exec_barrier();
                        if (all || kb + NST < nkb) {
                            begin(kb + NST);
                            issue(kb + NST, Q0, QN);
                        }
                    },
                    [&](auto n_) {
                        // the rest of the stage begun behind the last barrier
                        constexpr int n = decltype(n_)::value;
                        constexpr int groups = BG > 1 ? BG : 1;
                        constexpr int per = (LP - NOW + groups - 1) / groups;
                        if constexpr (n < BG && NOW + n * per < LP) {
                            constexpr int to = NOW + (n + 1) * per < LP ? NOW + (n + 1) * per : LP;
                            if (all || kb + NST - 1 < nkb)
                                issue(kb + NST - 1, std::integral_constant<int, NOW + n * per>{},
                                      std::integral_constant<int, to>{});
                        }
                    });
            };
            int kb = 0;
            for (; kb < nkb - NST; ++kb) one(kb, std::true_type{});
            for (; kb < nkb; ++kb) one(kb, std::false_type{});
        } else {
            if (nkb > 0) {
                fetch(0);
                put(0);
                __syncthreads();
                if (nkb > 1) fetch(1);
                first(smem + kw * Sh::STAGE);
            }
            static_assert(DMA || Sh::NST == 2, "two slots");
            for (int kb = 0; kb < nkb; ++kb) {
                // stage kb + 1 goes into the slot of kb - 1, read before the last barrier
                stage(
                    kb,
                    [&] {
                        if (kb + 1 < nkb) put(kb + 1);
                        __syncthreads();
                        if (kb + 2 < nkb) fetch(kb + 2);
                    },
                    [](auto) {});
            }
        }

        if constexpr (Sh::KW > 1) {
            // the groups' sums, added in order through the LDS
            __syncthreads();
            f32x4 *part = (f32x4 *)smem;
            if (kw > 0)
#pragma unroll
                for (int i = 0; i < MI; ++i)
#pragma unroll
                    for (int j = 0; j < NI; ++j)
                        part[(((kw - 1) * Sh::WAVES + wave) * MI * NI + i * NI + j) * 64 + lane] =
                            acc[i][j];
            __syncthreads();
            if (kw > 0) return false;
#pragma unroll
            for (int w = 0; w < Sh::KW - 1; ++w)
#pragma unroll
                for (int i = 0; i < MI; ++i)
#pragma unroll
                    for (int j = 0; j < NI; ++j) {
                        const f32x4 v =
                            part[((w * Sh::WAVES + wave) * MI * NI + i * NI + j) * 64 + lane];
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[i][j][e] += v[e];
                    }
        }
        return true;
    }

    // f(m, n, lo, hi): the four values lo of row m (of the tile), columns n ..
    // n + 3, and those hi of columns n + 16 .. n + 19; n is the same multiple of 32
    // plus 4 (lane / 16) in every lane
    template <typename F> OZK_DEV void each_pair(F &&f) const {
        static_assert(NI % 2 == 0, "pairs of blocks");
        const int lane = threadIdx.x & 63;
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const int m0 = wave / Sh::WN * MI * 16 + (lane & 15);
        const int n0 = wave % Sh::WN * NI * 16 + (lane >> 4) * 4;
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < NI; j += 2) f(m0 + 16 * i, n0 + 16 * j, acc[i][j], acc[i][j + 1]);
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

// 8 bytes of block j (`lo`) and of block j + 1 (`hi`), 16 columns each, of which
// lane group g holds columns 4g .. 4g + 3: exchanged between neighbouring lane
// groups so that a lane has 8 consecutive columns, from pair_column(g) on.  A
// 16-byte store per lane then covers 64 bytes of a row, where 8-byte stores
// cover 32 (8192 x 8192 with K = 256: 75 -> 64 us).
OZK_DEV i32x4 join_pair(i32x2 lo, i32x2 hi) {
    const auto x = __builtin_amdgcn_permlane16_swap((uint32_t)lo.x, (uint32_t)hi.x, false, false);
    const auto y = __builtin_amdgcn_permlane16_swap((uint32_t)lo.y, (uint32_t)hi.y, false, false);
    return i32x4{(int)x[0], (int)y[0], (int)x[1], (int)y[1]};
}
// and back
OZK_DEV void split_pair(i32x4 v, i32x2 &lo, i32x2 &hi) {
    const auto x = __builtin_amdgcn_permlane16_swap((uint32_t)v.x, (uint32_t)v.z, false, false);
    const auto y = __builtin_amdgcn_permlane16_swap((uint32_t)v.y, (uint32_t)v.w, false, false);
    lo = i32x2{(int)x[0], (int)y[0]};
    hi = i32x2{(int)x[1], (int)y[1]};
}
OZK_DEV int pair_column(int g) { return 16 * (g & 1) + 8 * (g >> 1); }

// 4 x 4 transposition of 16-bit values over four neighbouring lanes: lane q
// holds value e of its own row at place e, afterwards value q of row e.
OZK_DEV i32x2 transpose_quad(i32x2 v) {
    const uint32_t q = threadIdx.x & 3;
    // pairs of lanes: low halves of both to the even lane, high halves to the odd
    uint32_t r[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t own = (uint32_t)(i ? v.y : v.x);
        const uint32_t other = (uint32_t)__builtin_amdgcn_mov_dpp((int)own, 0xB1, 0xF, 0xF, true);
        r[i] = q & 1 ? __builtin_amdgcn_perm(own, other, 0x07060302u)
                     : __builtin_amdgcn_perm(other, own, 0x05040100u);
    }
    // then the pairs: lanes 0, 1 keep their first word, lanes 2, 3 their second
    const uint32_t give = q & 2 ? r[0] : r[1];
    const uint32_t got = (uint32_t)__builtin_amdgcn_mov_dpp((int)give, 0x4E, 0xF, 0xF, true);
    return q & 2 ? i32x2{(int)got, (int)r[1]} : i32x2{(int)r[0], (int)got};
}

// Tile `t` of `total` in the order in which XCD x (workgroups x, x + 8, ..)
// takes the x-th part of the tiles; -1: none
OZK_DEV int64_t xcd_tile(uint32_t block, uint32_t total) {
    const uint32_t per = (total + 7) / 8, i = block / 8;
    const uint32_t t = (block % 8) * per + i;
    return i < per && t < total ? (int64_t)t : -1;
}

}  // namespace ozk
