// ozk_grouped.hip -- matrix products grouped by expert, with ragged groups.
//
// Rows offsets[g] .. offsets[g + 1] of A belong to group g, whose matrix they
// are multiplied with; the offsets stay on the device, so the grid is the most
// tiles that T rows in G groups can need and a workgroup finds its group from
// the offsets (one wave-wide prefix sum of the groups' tile counts).
// Workgroups past the last tile end at once.
#include "ozk_linear.h"
#include "ozk_tile.h"

namespace ozk {

// offsets[i] clamped to [0, T]: whatever the tensor holds, no row outside the
// operands is touched
OZK_DEV int64_t offset_at(const void *offsets, int wide, int64_t i, int64_t T) {
    const int64_t v = wide ? ((const int64_t *)offsets)[i] : (int64_t)((const int32_t *)offsets)[i];
    return v < 0 ? 0 : v > T ? T : v;
}

OZK_DEV int wave_sum_before(int v, int lane) {   // inclusive prefix sum over the wave
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int u = __shfl_up(v, d);
        if (lane >= d) v += u;
    }
    return v;
}

// The groups with the rows before the first (segment 0) and after the last
// (segment G + 1), which have no group: segment s spans lo .. hi.
struct Segment {
    int64_t s, lo, hi;
};
OZK_DEV Segment segment_at(const GroupedParams &p, int64_t s) {
    const int64_t lo = s == 0 ? 0 : offset_at(p.offsets, p.offsets64, s - 1, p.T);
    const int64_t hi = s == p.G + 1 ? p.T : offset_at(p.offsets, p.offsets64, s, p.T);
    return {s, lo, hi < lo ? lo : hi};
}

// The tile's values, rounded, to C [rows, cols]
template <typename ST, typename Loop>
OZK_DEV void store_tile(const Loop &t, char *C, int64_t pitch, int rows, int cols) {
    auto bits = [](f32x4 v) {
        uint16_t e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) e[i] = to_bits16(v[i], ST{});
        i32x2 u;
        __builtin_memcpy(&u, e, 8);
        return u;
    };
    auto put = [&](int m, int n, i32x2 u) {   // columns n .. n + 3
        uint16_t e[4];
        __builtin_memcpy(e, &u, 8);
        uint16_t *to = (uint16_t *)(C + m * pitch) + n;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (m < rows && n + i < cols) to[i] = e[i];
    };
    if constexpr (Loop::NI % 2 == 0) {
        const int g = (threadIdx.x >> 4) & 3;
        t.each_pair([&](int m, int n, f32x4 lo, f32x4 hi) {
            const i32x2 a = bits(lo), b = bits(hi);
            const int n32 = n - 4 * g;
            if (n32 + 32 <= cols) {
                const i32x4 v = join_pair(a, b);
                // (rows of any alignment)
                if (m < rows)
                    __builtin_memcpy(C + m * pitch + (n32 + pair_column(g)) * 2, &v, 16);
            } else {
                put(m, n, a);
                put(m, n + 16, b);
            }
        });
    } else {
        t.each([&](int m, int n, f32x4 v) {
            const i32x2 u = bits(v);
            if (n + 4 <= cols) {
                if (m < rows) __builtin_memcpy(C + m * pitch + n * 2, &u, 8);
            } else {
                put(m, n, u);
            }
        });
    }
}

template <typename ST, typename Sh, bool DMA>
__global__ __launch_bounds__(Sh::THREADS, Sh::PER_SIMD) void grouped_kernel(GroupedParams p) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int lane = threadIdx.x & 63;
    constexpr int BM = Sh::BM, BN = Sh::BN;
    const uint32_t tiles_n = (uint32_t)((p.N + BN - 1) / BN);

    // tile rows of all segments
    const int64_t segs = p.G + 2;
    uint32_t total = 0;
    for (int64_t s0 = 0; s0 < segs; s0 += 64) {
        int n = 0;
        if (s0 + lane < segs) {
            const Segment g = segment_at(p, s0 + lane);
            n = (int)((g.hi - g.lo + BM - 1) / BM);
        }
        total += (uint32_t)__builtin_amdgcn_readlane(wave_sum_before(n, lane), 63);
    }
    const int64_t tile = xcd_tile(blockIdx.x, total * tiles_n);
    if (tile < 0) return;

    // the segment that holds the tile, and in it the order: 8 tile rows at a
    // time, column by column, so that the workgroups of an XCD share a square
    // block of both operands in its L2
    int64_t seg = 0, lo = 0, hi = 0;
    uint32_t before = 0, tn = 0;
    for (int64_t s0 = 0; s0 < segs; s0 += 64) {
        Segment g = {0, 0, 0};
        int n = 0;
        if (s0 + lane < segs) {
            g = segment_at(p, s0 + lane);
            n = (int)((g.hi - g.lo + BM - 1) / BM);
        }
        const int upto = wave_sum_before(n, lane);
        const uint64_t past = __ballot((before + (uint32_t)upto) * tiles_n > (uint32_t)tile);
        if (past) {
            const int l = __ffsll((unsigned long long)past) - 1;
            seg = s0 + l;
            lo = __shfl(g.lo, l);
            hi = __shfl(g.hi, l);
            const uint32_t have = (uint32_t)__shfl(n, l);
            const uint32_t in = (uint32_t)tile - (before + (uint32_t)__shfl(upto, l) - have) * tiles_n;
            const uint32_t first = in / tiles_n / 8 * 8;
            const uint32_t high = have - first < 8 ? have - first : 8, at = in - first * tiles_n;
            tn = at / high;
            lo += (int64_t)(first + at - tn * high) * BM;
            break;
        }
        before += (uint32_t)__builtin_amdgcn_readlane(upto, 63);
    }
    seg = uniform(seg);
    lo = uniform(lo);
    hi = uniform(hi);
    tn = (uint32_t)uniform((int)tn);
    const int rows = (int)(hi - lo < BM ? hi - lo : BM);
    const int64_t n0 = (int64_t)tn * BN;
    const int cols = (int)(p.N - n0 < BN ? p.N - n0 : BN);

    TileLoop<ST, Sh, DMA> t;
    const bool none = seg == 0 || seg == p.G + 1;
    const int64_t ka = p.a_padded ? (p.K + 7) / 8 * 16 : p.K * 2;   // bytes of K
    const int64_t kb = p.b_padded ? (p.K + 7) / 8 * 16 : p.K * 2;
    TileSrc A = {p.A + lo * p.a_pitch, p.a_pitch, rows, none ? 0 : ka, p.A};
    const char *Bg = p.B + (none ? 0 : seg - 1) * p.b_group;
    const int row = p.b_padded ? (cols + 7) / 8 * 16 : cols * 2;   // bytes, B along N
    TileSrc B = Sh::BCOLS ? TileSrc{Bg + n0 * 2, p.b_pitch, row, none ? 0 : p.K, p.B}
                          : TileSrc{Bg + n0 * p.b_pitch, p.b_pitch, cols, none ? 0 : kb, p.B};
    if (!t.run(A, B, smem)) return;

    store_tile<ST>(t, p.C + lo * p.c_pitch + n0 * 2, p.c_pitch, rows, cols);
}

// Which of its `all` work items of which group a workgroup of the dB kernel
// takes.  Groups about as long as their mean: an XCD has groups of its own, whose
// rows its L2 then reads once.  A group of more than twice the mean: every group
// over all XCDs, the longest first, so that no XCD and no workgroup is left with
// them at the end (four classes of length are enough: the order in full took
// longer than it saved).  More than 64 groups: over all XCDs in their order.
// Measured (us, T x G x K x N; a group to an XCD / spread / spread and ordered):
//     16384 x 32 x 2048 x 1024, uneven   135 / 119 / 102
//     32768 x 16 x 2048 x 4096, uneven  1325 / 539 / 531
//     16384 x 32 x 2048 x 1024, even      88 /  95 / 100
struct GradItem {
    int64_t lo, hi;   // the group's rows
    int g, item;      // g < 0: none
};
OZK_DEV GradItem grad_item(const GroupedGradParams &p, uint32_t all) {
    const uint32_t slots = (all + 7) / 8;
    uint32_t r = blockIdx.x / 8 / slots;   // the place of its group in their order
    const uint32_t i = blockIdx.x / 8 - r * slots, x = (blockIdx.x + r) % 8;
    const uint32_t from = (uint32_t)((uint64_t)all * x / 8);
    const bool none = i >= (uint32_t)((uint64_t)all * (x + 1) / 8) - from;
    GradItem at = {0, 0, none ? -1 : (int)r, (int)(from + i)};
    if (p.G > 64) {
        if (none) return at;
        at.lo = uniform(offset_at(p.offsets, p.offsets64, r, p.T));
        at.hi = uniform(offset_at(p.offsets, p.offsets64, r + 1, p.T));
        return at;
    }
    const int lane = threadIdx.x & 63;
    int64_t lo = 0, hi = 0;
    if (lane < p.G) {
        lo = offset_at(p.offsets, p.offsets64, lane, p.T);
        hi = offset_at(p.offsets, p.offsets64, lane + 1, p.T);
    }
    const int64_t n = hi - lo;
    const uint64_t there = p.G == 64 ? ~0ull : ((uint64_t)1 << p.G) - 1;
    const uint64_t over2 = __ballot(n > 2 * p.share);
    if (over2) {
        if (none) return at;
        const uint64_t over4 = __ballot(n > 4 * p.share), over1 = __ballot(n > p.share);
        const uint64_t cls[4] = {over4, over2 & ~over4, over1 & ~over2, there & ~over1};
        uint32_t before = 0, rank = 0;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            if (cls[c] >> lane & 1)
                rank = before + (uint32_t)__popcll(cls[c] & (((uint64_t)1 << lane) - 1));
            before += (uint32_t)__popcll(cls[c]);
        }
        r = (uint32_t)__ffsll((unsigned long long)__ballot(lane < p.G && rank == r)) - 1;
    } else {
        const int64_t tile = xcd_tile(blockIdx.x, all * (uint32_t)p.G);
        if (tile < 0) return GradItem{0, 0, -1, 0};
        r = (uint32_t)tile / all;
        at.item = (int)((uint32_t)tile - r * all);
    }
    at.g = uniform((int)r);
    at.lo = uniform(__shfl(lo, at.g));
    at.hi = uniform(__shfl(hi, at.g));
    return at;
}

// dB: the rows of a group are the contraction, both operands "cols".  With
// splits > 1 workgroup s of a tile sums the s-th part of the group's rows into
// the workspace, and grouped_join_kernel adds the parts in order.
template <typename ST, typename Sh, bool DMA>
__global__ __launch_bounds__(Sh::THREADS, Sh::PER_SIMD) void grouped_grad_kernel(GroupedGradParams p) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    constexpr int BM = Sh::BM, BN = Sh::BN;
    const uint32_t tiles_k = (uint32_t)((p.K + BM - 1) / BM);
    const uint32_t tiles_n = (uint32_t)((p.N + BN - 1) / BN);
    const uint32_t each = tiles_k * tiles_n;
    const GradItem at = grad_item(p, each * (uint32_t)p.splits);
    if (at.g < 0) return;
    const int64_t g = at.g;
    const uint32_t s = (uint32_t)at.item / each, in = (uint32_t)at.item - s * each;
    // squares of tiles about as large as what an XCD has of a group
    const uint32_t h = p.block, first = in / tiles_n / h * h;
    const uint32_t high = tiles_k - first < h ? tiles_k - first : h, ahead = in - first * tiles_n;
    const uint32_t tn = ahead / high, tk = first + ahead - tn * high;
    int64_t lo = at.lo, hi = at.hi < at.lo ? at.lo : at.hi;
    if (p.splits > 1) {
        // whole stages each
        const int64_t stages = (hi - lo + Sh::KS - 1) / Sh::KS;
        const int64_t per = (stages + p.splits - 1) / p.splits * Sh::KS;
        lo += per * s;
        if (lo > hi) lo = hi;
        if (hi > lo + per) hi = lo + per;
    }
    const int64_t k0 = (int64_t)tk * BM, n0 = (int64_t)tn * BN;
    const int rows = (int)(p.K - k0 < BM ? p.K - k0 : BM);
    const int cols = (int)(p.N - n0 < BN ? p.N - n0 : BN);

    TileLoop<ST, Sh, DMA> t;
    const TileSrc A = {p.A + lo * p.a_pitch + k0 * 2, p.a_pitch,
                       p.a_padded ? (rows + 7) / 8 * 16 : rows * 2, hi - lo, p.A};
    const TileSrc B = {p.D + lo * p.d_pitch + n0 * 2, p.d_pitch,
                       p.d_padded ? (cols + 7) / 8 * 16 : cols * 2, hi - lo, p.D};
    if (!t.run(A, B, smem)) return;

    if (p.splits > 1) {
        float *P = p.part + ((int64_t)s * p.G + g) * p.K * p.N + k0 * p.N + n0;
        t.each([&](int m, int n, f32x4 v) {
            if (m >= rows) return;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (n + i < cols) P[(int64_t)m * p.N + n + i] = v[i];
        });
        return;
    }
    store_tile<ST>(t, p.dB + (int64_t)g * p.db_group + k0 * p.db_pitch + n0 * 2, p.db_pitch, rows,
                   cols);
}

template <typename ST>
__global__ __launch_bounds__(256) void grouped_join_kernel(GroupedGradParams p) {
    const int64_t each = p.K * p.N, all = p.G * each;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all;
         i += (int64_t)gridDim.x * 256) {
        float v = 0.f;
        for (int s = 0; s < p.splits; ++s) v += p.part[s * all + i];
        const int64_t g = i / each, r = (i - g * each) / p.N, c = i - g * each - r * p.N;
        ((uint16_t *)(p.dB + g * p.db_group + r * p.db_pitch))[c] = to_bits16(v, ST{});
    }
}

// Rows copied to whole 16-byte pieces, zeros behind their end: [groups] blocks of
// `rows` rows of `cols` 16-bit elements, one behind another in dst.
struct PackJob {
    const char *src;
    char *dst;
    int64_t group, pitch;    // bytes in src
    uint32_t rows, all;      // of a group, of all groups
    int cols, pieces;        // elements and 16-byte pieces of a row
    uint32_t blocks, per;    // workgroups, and rows of each
};
__global__ __launch_bounds__(256) void grouped_pack_kernel(PackJob a, PackJob b) {
    const bool second = blockIdx.x >= a.blocks;
    const PackJob &j = second ? b : a;
    const uint32_t r0 = (blockIdx.x - (second ? a.blocks : 0u)) * j.per;
    const uint32_t left = j.all - r0, rows = left < j.per ? left : j.per;
    const float rcp = 1.f / (float)j.pieces;
    for (int i = threadIdx.x; i < (int)rows * j.pieces; i += 256) {
        const int r = part_of(i, j.pieces, rcp), at = i - r * j.pieces;
        const uint32_t row = r0 + r, g = row / j.rows;
        const char *from = j.src + g * j.group + (int64_t)(row - g * j.rows) * j.pitch + at * 16;
        *(i32x4 *)(j.dst + (int64_t)row * j.pieces * 16 + at * 16) =
            load_piece(from, (j.cols - at * 8) * 2, j.src);
    }
}

namespace {

// rows that are whole aligned 16-byte pieces, which the LDS-DMA takes
bool whole_pieces(const void *p, int64_t pitch, int64_t group, int64_t cols, bool padded) {
    return (((uintptr_t)p | (uintptr_t)pitch | (uintptr_t)group) & 15) == 0 &&
           (padded || cols % 8 == 0);
}
bool a_pieces(const GroupedParams &p) { return whole_pieces(p.A, p.a_pitch, 0, p.K, p.a_padded); }
bool b_pieces(const GroupedParams &p) {
    return whole_pieces(p.B, p.b_pitch, p.b_group, p.b_cols ? p.N : p.K, p.b_padded);
}
int64_t pieces_of(int64_t cols) { return (cols + 7) / 8; }
size_t packed_bytes(int64_t rows, int64_t cols) { return (size_t)(rows * pieces_of(cols) * 16); }
PackJob pack_job(const char *src, char *dst, int64_t groups, int64_t group, int64_t rows,
                 int64_t pitch, int64_t cols) {
    PackJob j = {src, dst, group, pitch, (uint32_t)rows, (uint32_t)(rows * groups), (int)cols,
                 (int)pieces_of(cols), 0, 1};
    while (j.per < 4096 && (int64_t)j.per * j.pieces < 1024) j.per *= 2;
    j.blocks = (j.all + j.per - 1) / j.per;
    return j;
}
hipError_t pack(const PackJob &a, const PackJob &b, hipStream_t st) {
    grouped_pack_kernel<<<dim3(a.blocks + b.blocks), 256, 0, st>>>(a, b);
    return hipGetLastError();
}
// rows that the pack kernel counts in 32 bits, and copies of them no further apart
// than the tiles step (2^22 elements: overlapping rows can be longer than that)
bool packable(int64_t rows, int64_t cols) {
    return rows < (int64_t)1 << 30 && pieces_of(cols) < (int64_t)1 << 19;
}

template <typename ST, typename Sh, bool DMA>
hipError_t grouped_go(const GroupedParams &p, hipStream_t st) {
    // most tiles: every segment may end inside one
    const int64_t segs = p.G + 2 < p.T ? p.G + 2 : p.T;
    const int64_t tiles = (p.T / Sh::BM + segs) * ((p.N + Sh::BN - 1) / Sh::BN);
    if (tiles >= (int64_t)1 << 31) return hipErrorInvalidConfiguration;
    if (hipError_t e = allow_lds<&grouped_kernel<ST, Sh, DMA>>(Sh::LDS_BYTES); e != hipSuccess)
        return e;
    grouped_kernel<ST, Sh, DMA><<<dim3((uint32_t)((tiles + 7) / 8 * 8)), Sh::THREADS, Sh::LDS_BYTES, st>>>(p);
    return hipGetLastError();
}

template <typename ST, typename Sh, bool DMA>
hipError_t grad_go(const GroupedGradParams &p, hipStream_t st) {
    const int64_t each = ((p.K + Sh::BM - 1) / Sh::BM) * ((p.N + Sh::BN - 1) / Sh::BN);
    const int64_t slots = (each * p.splits + 7) / 8;
    if (slots >= (int64_t)1 << 28 || slots * p.G >= (int64_t)1 << 28)
        return hipErrorInvalidConfiguration;
    if (hipError_t e = allow_lds<&grouped_grad_kernel<ST, Sh, DMA>>(Sh::LDS_BYTES);
        e != hipSuccess)
        return e;
    GroupedGradParams q = p;
    q.share = p.T / p.G;
    for (q.block = 1; q.block < 8 && 4 * q.block * q.block <= slots;) q.block *= 2;
    grouped_grad_kernel<ST, Sh, DMA><<<dim3((uint32_t)(slots * 8 * p.G)), Sh::THREADS, Sh::LDS_BYTES, st>>>(q);
    return hipGetLastError();
}

// Tiles for T rows in G groups, the counts themselves being on the device: a
// group is taken to leave half a tile row unused.  Where the rows fill tiles of
// 64 x 128 at least once over, the tile is the one of the shortest time, rounds of
// workgroups (256 CUs, with 2 and 3 workgroups of the small tiles each) by a
// round's time, which is (us, K in 1024s)
//     256 x 256          3 + 27 K        192 x 256          5 + 21 K
//     128 x 128          1 + 18.5 K      64 x 128           5 + 13 K
// Measured (us, T x G x K x N, bf16, counts uneven; 256 x 256 / 192 x 256 /
// 128 x 128 / 64 x 128):
//     32768 x 16 x 2048 x 4096   533 / 609 / 672 / 732
//     16384 x 32 x 1024 x 2048    88 /  97 /  90 / 101
//     8192 x 8 x 1024 x 2048      58 /  53 /  53 /  55
//     4096 x 8 x 1024 x 4096      55 /  52 /  51 /  55
//     4096 x 4 x 2048 x 2048      50 /  44 /  57 /  55
//     2000 x 4 x 1024 x 4096      30 /  27 /  33 /  31
// Smaller groups take the tile that covers most groups whole (each tile row reads
// the group's matrix again); where a CU has one workgroup at most, two groups of
// waves share its stages.  Measured (us; 128 x 128 of 4 stages / 64 x 128 / 64 x 64
// in two groups / 32 x 64 in two groups of 4 stages):
//     1999 x 7 x 1000 x 520       14 /  13 /  11 /  19
//     512 x 8 x 1024 x 2048       15 /  17 /  14 /  20
//     300 x 8 x 4096 x 4096       46 /  67 /  71 /  71
//     200 x 32 x 1024 x 2048      30 /  23 /  26 /  35
//     2000 x 2 x 4096 x 256       38 /  48 /  25 /  16
//     4 x 4 x 4096 x 1024         40 /  39 /  20 /  15
//     16 x 16 x 1024 x 2048       13 /  12 / 8.4 / 7.7
template <typename ST, bool BCOLS> hipError_t grouped_plan(const GroupedParams &p, hipStream_t st) {
    const bool pieces = a_pieces(p) && b_pieces(p);
    const int64_t groups = p.G < 1 ? 1 : p.G < p.T ? p.G : p.T, rows = p.T / groups;
    auto tiles = [&](int64_t bm, int64_t bn) {
        return (p.T / bm + (groups + 1) / 2) * ((p.N + bn - 1) / bn);
    };
    if (!pieces) {
        if (rows >= 48) return grouped_go<ST, TileShape<1, false, BCOLS, 128, 128, 2, 2, 2>, false>(p, st);
        return grouped_go<ST, TileShape<1, false, BCOLS, 32, 64, 1, 4, 2>, false>(p, st);
    }
    if (rows > 24 && rows <= 128 && p.K * p.N >= (int64_t)1 << 22 && tiles(128, 128) >= 128)
        return grouped_go<ST, TileShape<1, false, BCOLS, 128, 128, 2, 4, 4>, true>(p, st);
    if (tiles(64, 128) >= 256) {
        const double k = (double)p.K / 1024;
        auto time = [&](int64_t bm, int64_t bn, int64_t at_once, double fixed, double slope) {
            return (double)((tiles(bm, bn) + at_once - 1) / at_once) * (fixed + slope * k);
        };
        const double t256 = time(256, 256, 256, 3, 27), t192 = time(192, 256, 256, 5, 21);
        const double t128 = time(128, 128, 512, 1, 18.5), t64 = time(64, 128, 768, 5, 13);
        if (t256 <= t192 && t256 <= t128 && t256 <= t64)
            return grouped_go<ST, TileShape<1, false, BCOLS, 256, 256, 2, 4, 2>, true>(p, st);
        if (t192 <= t128 && t192 <= t64)
            return grouped_go<ST, TileShape<1, false, BCOLS, 192, 256, 2, 4, 2>, true>(p, st);
        if (t128 <= t64)
            return grouped_go<ST, TileShape<1, false, BCOLS, 128, 128, 2, 4, 2>, true>(p, st);
        return grouped_go<ST, TileShape<1, false, BCOLS, 64, 128, 1, 4, 2>, true>(p, st);
    }
    if (tiles(32, 64) <= 256)
        return grouped_go<ST, TileShape<1, false, BCOLS, 32, 64, 1, 4, 4, 2>, true>(p, st);
    return grouped_go<ST, TileShape<1, false, BCOLS, 64, 64, 2, 2, 2, 2>, true>(p, st);
}

// The same for dB, whose row ranges (splits) are planned for 64 x 128.  Measured
// (us; 256 x 256 / 128 x 128 / 64 x 128):
//     16384 x 32 x 2048 x 1024    91 /  98 / 113
//     8192 x 64 x 1024 x 1024     53 /  55 /  59
//     3000 x 6 x 2048 x 1024      32 /  24 /  37
//     4096 x 4 x 1024 x 2048      43 /  33 /  46
//     1999 x 7 x 1000 x 520       25 /  13 /  12
template <typename ST> hipError_t grad_plan(const GroupedGradParams &p, hipStream_t st) {
    const bool pieces = whole_pieces(p.A, p.a_pitch, 0, p.K, p.a_padded) &&
                        whole_pieces(p.D, p.d_pitch, 0, p.N, p.d_padded);
    const int64_t large = ((p.K + 255) / 256) * ((p.N + 255) / 256) * p.G;
    const int64_t medium = ((p.K + 127) / 128) * ((p.N + 127) / 128) * p.G;
    hipError_t e;
    if (!pieces)
        e = grad_go<ST, TileShape<1, true, true, 128, 128, 2, 2, 2>, false>(p, st);
    else if (large >= 512)
        e = grad_go<ST, TileShape<1, true, true, 256, 256, 2, 4, 2>, true>(p, st);
    else if (medium >= 384)
        e = grad_go<ST, TileShape<1, true, true, 128, 128, 2, 4, 2>, true>(p, st);
    else
        e = grad_go<ST, TileShape<1, true, true, 64, 128, 1, 4, 2>, true>(p, st);
    if (e != hipSuccess || p.splits == 1) return e;
    const int64_t all = p.G * p.K * p.N;
    const int64_t blocks = (all + 255) / 256 < 2048 ? (all + 255) / 256 : 2048;
    grouped_join_kernel<ST><<<dim3((uint32_t)blocks), 256, 0, st>>>(p);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_grouped(const GroupedParams &p, int dtype, hipStream_t st) {
    if (dtype == 2) return p.b_cols ? grouped_plan<_Float16, true>(p, st) : grouped_plan<_Float16, false>(p, st);
    return p.b_cols ? grouped_plan<__bf16, true>(p, st) : grouped_plan<__bf16, false>(p, st);
}

// Rows that are no whole pieces go through registers, or are copied first
// where that pays: a copy costs 1e-12 s an element and 5e-6 s, the way through
// registers so much more a stage of a tile, 1.1e-6 s (2.5e-6 where B's rows run
// along N; a quarter of it in the small tiles of few rows; 3e-6 for dB), and again
// for every so many tiles.  Measured (us, T x G x K x N, B along N, with the copy /
// through registers):
//     8192 x 4 x 1001 x 1003       53 /  86     dB  70 /  224
//     32768 x 16 x 1023 x 2047    256 / 335     dB 440 / 1131
//     2000 x 2 x 4097 x 257        41 / 231     dB  46 /   49
//     948 x 13 x 1344 x 2259       52 /  92     dB  62 /   64
//     4030 x 28 x 1920 x 2121     190 / 168     dB 169 /  177
//     1000 x 64 x 1025 x 1025      76 /  35     dB 101 /   90
//     16 x 16 x 1025 x 2049        34 /  20     dB  56 /   46
PackedSizes plan_grouped_pack(const GroupedParams &p) {
    const bool a = !a_pieces(p), b = p.G > 0 && !b_pieces(p);
    const int64_t b_rows = p.b_cols ? p.K : p.N, b_len = p.b_cols ? p.N : p.K;
    if ((!a && !b) || p.T == 0 || p.K == 0 || p.N == 0 || !packable(p.T, p.K) ||
        !packable(p.G * b_rows, b_len))
        return {0, 0};
    const double cost = 1e-12 * ((a ? (double)p.T * p.K : 0) + (b ? (double)p.G * p.K * p.N : 0)) + 5e-6;
    const int64_t groups = p.G < 1 ? 1 : p.G < p.T ? p.G : p.T;
    const double tiles = ((double)p.T / 128 + groups / 2) * ((double)p.N / 128 + 1) / 1536;
    const double stage = (b && p.b_cols ? 2.5e-6 : 1.1e-6) * (p.T / groups >= 48 ? 1 : 0.25) *
                         (tiles > 1 ? tiles : 1);
    if (stage * ((p.K + 63) / 64) < cost) return {0, 0};
    return {a ? packed_bytes(p.T, p.K) : 0, b ? packed_bytes(p.G * b_rows, b_len) : 0};
}
PackedSizes plan_grad_pack(const GroupedGradParams &p) {
    const bool a = !whole_pieces(p.A, p.a_pitch, 0, p.K, p.a_padded);
    const bool d = !whole_pieces(p.D, p.d_pitch, 0, p.N, p.d_padded);
    if ((!a && !d) || p.T == 0 || p.K == 0 || p.N == 0 || p.G == 0 || !packable(p.T, p.K) ||
        !packable(p.T, p.N))
        return {0, 0};
    const double cost = 1e-12 * p.T * ((a ? (double)p.K : 0) + (d ? (double)p.N : 0)) + 5e-6;
    const double tiles = ((double)p.K / 128 + 1) * ((double)p.N / 128 + 1) * p.G / 1024;
    if (3e-6 * (tiles > 1 ? tiles : 1) * p.T / (64.0 * p.G * p.splits) < cost) return {0, 0};
    return {a ? packed_bytes(p.T, p.K) : 0, d ? packed_bytes(p.T, p.N) : 0};
}
hipError_t pack_grouped(GroupedParams &p, const PackedSizes &n, char *ws, hipStream_t st) {
    PackJob a = {}, b = {};
    const int64_t b_rows = p.b_cols ? p.K : p.N, b_len = p.b_cols ? p.N : p.K;
    if (n.a) {
        a = pack_job(p.A, ws, 1, 0, p.T, p.a_pitch, p.K);
        p.A = ws;
        p.a_pitch = pieces_of(p.K) * 16;
        p.a_padded = true;
    }
    if (n.b) {
        b = pack_job(p.B, ws + n.a, p.G, p.b_group, b_rows, p.b_pitch, b_len);
        p.B = ws + n.a;
        p.b_pitch = pieces_of(b_len) * 16;
        p.b_group = b_rows * p.b_pitch;
        p.b_padded = true;
    }
    return pack(a, b, st);
}
hipError_t pack_grad(GroupedGradParams &p, const PackedSizes &n, char *ws, hipStream_t st) {
    PackJob a = {}, b = {};
    if (n.a) {
        a = pack_job(p.A, ws, 1, 0, p.T, p.a_pitch, p.K);
        p.A = ws;
        p.a_pitch = pieces_of(p.K) * 16;
        p.a_padded = true;
    }
    if (n.b) {
        b = pack_job(p.D, ws + n.a, 1, 0, p.T, p.d_pitch, p.N);
        p.D = ws + n.a;
        p.d_pitch = pieces_of(p.N) * 16;
        p.d_padded = true;
    }
    return pack(a, b, st);
}

int grouped_grad_splits(int64_t T, int64_t K, int64_t N, int64_t G) {
    const int64_t tiles = ((K + 127) / 128) * ((N + 127) / 128) * G;
    const int64_t stages = (T / (G > 0 ? G : 1) + 63) / 64;
    int s = 1;
    while (s < 16 && tiles * s < 256 && stages / (2 * s) >= 8) s *= 2;
    return s;
}

hipError_t launch_grouped_grad(const GroupedGradParams &p, int dtype, hipStream_t st) {
    return dtype == 2 ? grad_plan<_Float16>(p, st) : grad_plan<__bf16>(p, st);
}

}  // namespace ozk
