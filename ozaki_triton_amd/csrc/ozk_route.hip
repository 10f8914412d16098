// ozk_route.hip -- the router of a layer of experts.
//
//   p = softmax(l) over the E experts; a token goes to the k experts of its
//   greatest logits, of equal ones to those of the lowest index; their weights
//   are their p, or with `normalize` their p over the sum of the k.
//   counts[e] = tokens that chose e; offsets: their running sum, the groups of the
//   grouped products; order: the slots t k + j sorted by expert, in their own
//   order within one; place: the slots' places there.
//   loss = E sum_e f_e P_e with f_e = counts[e] / (n k), P_e the mean of p[t, e],
//   over the n tokens that are not masked out.  Masked ones have expert E, weight 0
//   and the places behind the last group.
//
// Two launches: rows (softmax, choice, counts of each workgroup's tokens and the
// slots' places among them) and place (slots to their places: every workgroup adds
// up the counts of those before it; where that is much to read, a third launch,
// scan, does it once); few tokens need one workgroup and one launch.  The sums over
// tokens are those of fixed parts in a fixed order, no atomics but whole-number
// counts.
//
// A token takes GL lanes with V consecutive logits each, so that several share a
// wave; the k choices are k rounds of a maximum over keys (the logits' bits in
// the order of their values, NaN greatest) in lane exchanges.
//
// Bound by latency and, with many tokens, instructions, not by the bytes (22 MB of the
// first line are 4.5 us of a copy): the vector units of the rows kernel are busy 36% of the
// time with 32768 tokens, where waves wait for each other and for lane exchanges 55% of
// theirs, and 83% with 300000.  Measured (us, T x E, k; rows / place / gradient):
//     32768 x 64, 8, fp32   12.3 / 8.3 / 8.8      4099 x 40, 3, bf16   6.2 / 6.9 / 4.4
//     16 x 16, 2, bf16       6.9 (one launch)
#include "../../include/ozaki_amd.h"
#include "ozk_train.h"
#include "ozk_tile.h"

namespace ozk {

// lane exchanges over groups of GL lanes: f(own, other's) of pairs that cover the group
template <int GL, typename T, typename F> OZK_DEV T over_group(T v, F &&f) {
    static_assert(sizeof(T) == 4, "");
    auto dpp = [](T x, auto ctrl_) {
        constexpr int ctrl = decltype(ctrl_)::value;
        return __builtin_bit_cast(
            T, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), ctrl, 0xF, 0xF, true));
    };
    if constexpr (GL >= 2) v = f(v, dpp(v, std::integral_constant<int, 0xB1>{}));    // quad 1 0 3 2
    if constexpr (GL >= 4) v = f(v, dpp(v, std::integral_constant<int, 0x4E>{}));    // quad 2 3 0 1
    if constexpr (GL >= 8) v = f(v, dpp(v, std::integral_constant<int, 0x141>{}));   // mirror of 8
    if constexpr (GL >= 16) v = f(v, dpp(v, std::integral_constant<int, 0x140>{}));  // mirror of 16
    if constexpr (GL >= 32) {
        const auto x = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, v),
                                                        __builtin_bit_cast(uint32_t, v), false, false);
        v = f(__builtin_bit_cast(T, (uint32_t)x[0]), __builtin_bit_cast(T, (uint32_t)x[1]));
    }
    if constexpr (GL >= 64) {
        const auto x = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v),
                                                        __builtin_bit_cast(uint32_t, v), false, false);
        v = f(__builtin_bit_cast(T, (uint32_t)x[0]), __builtin_bit_cast(T, (uint32_t)x[1]));
    }
    return v;
}
template <int GL> OZK_DEV uint32_t group_max(uint32_t v) {
    return over_group<GL>(v, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
}
template <int GL> OZK_DEV float group_sum(float v) {
    return over_group<GL>(v, [](float a, float b) { return a + b; });
}

// Keys: whole numbers in the order of the values, -0 as 0, NaN above all, 0 below
// every logit's.  Of 16-bit logits a key has the index behind the value's bits,
// the lowest greatest, so that a maximum finds both.
template <typename T> OZK_DEV uint32_t key_of(float x, uint32_t index) {
    if constexpr (sizeof(T) == 4) {
        if (x != x) return 0xFFFFFFFFu;
        const uint32_t u = __float_as_uint(x + 0.f);
        return u & 0x80000000u ? ~u : u | 0x80000000u;
    } else {
        const uint32_t u = to_bits16(x + 0.f, T{});
        const uint32_t key = x != x ? 0xFFFFu : u & 0x8000u ? ~u & 0xFFFFu : u | 0x8000u;
        return key << 16 | (0xFFFFu - index);
    }
}
template <typename T> OZK_DEV float value_of(uint32_t key) {
    if constexpr (sizeof(T) == 4) {
        return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);
    } else {
        const uint32_t k = key >> 16;
        return from_bits16((uint16_t)(k & 0x8000u ? k & 0x7FFFu : ~k), T{});
    }
}

// A token's V logits of a lane, from expert e0 on; -inf behind the last expert
template <typename T, int V>
OZK_DEV void logits_at(const char *row, int e0, int E, bool there, float (&l)[V]) {
    if (there && e0 + V <= E) {
        T t[V];
        __builtin_memcpy(t, row + (int64_t)e0 * sizeof(T), V * sizeof(T));
#pragma unroll
        for (int v = 0; v < V; ++v) l[v] = (float)t[v];
    } else {
#pragma unroll
        for (int v = 0; v < V; ++v)
            l[v] = there && e0 + v < E ? load_value<T>(row, e0 + v) : -__builtin_inff();
    }
}

constexpr int kRouteWaves = 16;   // of a workgroup

// LDS of a workgroup: its slots' experts, those of each wave, sums
struct RouteLds {
    uint32_t *parts;       // [64], for prefix sums and the like
    uint32_t *last;        // where the groups end
    uint32_t *wave_hist;   // [waves][E + 1]
    float *psum;           // [waves][E]
    float *scale;          // [per]: what the weights are divided by
    float *value;          // [per k]: e to the chosen logits less the greatest
    uint16_t *expert;      // [per k]
    OZK_DEV RouteLds(char *at, int E, int64_t per, int k) {
        parts = (uint32_t *)at;
        last = parts + 4 * kRouteWaves;
        wave_hist = last + 4;
        psum = (float *)(wave_hist + kRouteWaves * (E + 1));
        scale = psum + kRouteWaves * E;
        value = scale + per;
        expert = (uint16_t *)(value + per * k);
    }
    static size_t bytes(int E, int64_t per, int k) {
        return 4 * (size_t)(4 * kRouteWaves + 4 + kRouteWaves * (2 * E + 1)) + 4 * (size_t)per + 6 * (size_t)(per * k);
    }
};

// Prefix sums over E values by the workgroup: v is that of index threadIdx.x (E
// is at most the 1024 lanes); the sum of those before.
OZK_DEV uint32_t before_in_block(uint32_t v, uint32_t *parts) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t s = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t u = __shfl_up(s, d);
        if (lane >= d) s += u;
    }
    __syncthreads();
    if (lane == 63) parts[wave] = s;
    __syncthreads();
    uint32_t before = s - v;
#pragma unroll
    for (int w = 0; w < kRouteWaves - 1; ++w) before += w < wave ? parts[w] : 0u;
    return before;
}

// offsets, counts and the loss, by one workgroup; total and P: of expert threadIdx.x
OZK_DEV void finish_counts(const RouteParams &p, uint32_t total, double P, uint32_t before,
                           uint32_t *parts) {
    const int e = threadIdx.x, lane = threadIdx.x & 63;
    if (e < p.E) {
        p.counts[e] = (int32_t)total;
        p.offsets[e] = (int32_t)before;
        if (e == p.E - 1) p.offsets[p.E] = (int32_t)(before + total);
    }
    // sum over e of counts P
    double s = e < p.E ? (double)total * P : 0.0;
    double n = e < p.E ? (double)total : 0.0;
#pragma unroll
    for (int d = 32; d; d >>= 1) {
        s += __shfl_xor(s, d);
        n += __shfl_xor(n, d);
    }
    double *sums = (double *)parts;   // [2][waves]
    __syncthreads();
    if (lane == 0) {
        sums[threadIdx.x >> 6] = s;
        sums[kRouteWaves + (threadIdx.x >> 6)] = n;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        s = n = 0.0;
#pragma unroll
        for (int w = 0; w < kRouteWaves; ++w) {
            s += sums[w];
            n += sums[kRouteWaves + w];
        }
        // n: slots, k to a token
        const double tokens = n / p.k;
        *p.loss = n > 0.0 ? (float)(p.E * s / (n * tokens)) : 0.f;
    }
}

template <typename T, int GL, int V, bool ONE>
__global__ __launch_bounds__(64 * kRouteWaves) void route_rows_kernel(RouteParams p) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    // (all of it dynamic: the limit that the launch raises counts that alone)
    const RouteLds lds(smem, p.E, p.per, p.k);
    constexpr int TPW = 64 / GL;   // tokens of a wave at a time
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int in = lane % GL, e0 = in * V;
    // a lane's keys greatest first, so that a round looks at one of them (with 4 of them, us,
    // unsorted / sorted: 300000 x 64, k = 8, fp32 145 / 129; 32768 x 64 20.4 / 19.4)
    constexpr bool SORTED = V == 4;
    const uint64_t below = (((uint64_t)1 << in) - 1) << (lane - in);   // the group's lanes before this
    const int64_t t0 = (int64_t)blockIdx.x * p.per;
    const int tokens = (int)(p.T - t0 < p.per ? p.T - t0 : p.per);
    for (int i = threadIdx.x; i < kRouteWaves * (p.E + 1); i += 64 * kRouteWaves) lds.wave_hist[i] = 0;

    float psum[V] = {};
    for (int r = wave * TPW; r < tokens; r += kRouteWaves * TPW) {
        const int t = r + lane / GL;
        const bool there = t < tokens;
        const bool valid = there && (!p.mask || p.mask[t0 + t]);
        float l[V];
        logits_at<T, V>(p.logits + (t0 + t) * p.pitch * (int64_t)sizeof(T), e0, p.E, valid, l);
        uint32_t key[V];
#pragma unroll
        for (int v = 0; v < V; ++v) key[v] = e0 + v < p.E ? key_of<T>(l[v], e0 + v) : 0u;
        uint32_t expert[V];
#pragma unroll
        for (int v = 0; v < V; ++v) expert[v] = e0 + v;
        if constexpr (SORTED) {   // exchanges of neighbours only, so that equal ones stay in order
            auto order = [&](int i) {
                const bool swap = key[i + 1] > key[i];
                const uint32_t k0 = key[i], k1 = key[i + 1], x0 = expert[i], x1 = expert[i + 1];
                key[i] = swap ? k1 : k0;
                key[i + 1] = swap ? k0 : k1;
                expert[i] = swap ? x1 : x0;
                expert[i + 1] = swap ? x0 : x1;
            };
#pragma unroll
            for (int n = 0; n < V; ++n)
#pragma unroll
                for (int i = n & 1; i + 1 < V; i += 2) order(i);
        }
        // k rounds; lane j of the group keeps the j-th choice, GL of them at a time
        float chosen = 0.f;
        uint32_t first = 0, kept = 0;
        for (int j0 = 0; j0 < p.k; j0 += GL) {
            const int here = p.k - j0 < GL ? p.k - j0 : GL;
            for (int j = 0; j < here; ++j) {
                uint32_t own = key[0];
                if constexpr (!SORTED)
#pragma unroll
                    for (int v = 1; v < V; ++v) own = key[v] > own ? key[v] : own;
                const uint32_t best = group_max<GL>(own);
                first = j0 + j == 0 ? best : first;
                kept = in == j ? best : kept;
                bool mine = own == best;
                if constexpr (sizeof(T) == 4) mine = mine && !(__ballot(mine) & below);
                if (mine) {
                    uint32_t at = expert[0];
                    if constexpr (SORTED) {
#pragma unroll
                        for (int v = 0; v + 1 < V; ++v) {
                            key[v] = key[v + 1];
                            expert[v] = expert[v + 1];
                        }
                        key[V - 1] = 0;
                    } else {   // the lowest that has it
                        bool found = false;
#pragma unroll
                        for (int v = 0; v < V; ++v) {
                            const bool hit = !found && key[v] == best;
                            found |= hit;
                            at = hit ? expert[v] : at;
                            key[v] = hit ? 0u : key[v];
                        }
                    }
                    if constexpr (sizeof(T) == 4)
                        if (there) lds.expert[t * p.k + j0 + j] = (uint16_t)(valid ? at : (uint32_t)p.E);
                }
            }
            if (in < here) {
                const float e = expf(value_of<T>(kept) - value_of<T>(first));
                chosen += e;
                if (there) {
                    lds.value[t * p.k + j0 + in] = e;
                    if constexpr (sizeof(T) == 2)
                        lds.expert[t * p.k + j0 + in] = (uint16_t)(valid ? 0xFFFFu - (kept & 0xFFFFu) : (uint32_t)p.E);
                }
            }
        }
        const float top = value_of<T>(first);
        chosen = group_sum<GL>(chosen);
        float q[V], sum = 0.f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            q[v] = e0 + v < p.E ? expf(l[v] - top) : 0.f;
            sum += q[v];
        }
        sum = group_sum<GL>(sum);
        if (in == 0 && there) lds.scale[t] = p.normalize ? chosen : sum;
        if (valid) {
            const float by = 1.f / sum;
#pragma unroll
            for (int v = 0; v < V; ++v) psum[v] += q[v] * by;
        }
    }
    // the wave's sums of p: the lanes that hold the same experts
#pragma unroll
    for (int v = 0; v < V; ++v) {
        float s = psum[v];
        for (int d = GL; d < 64; d <<= 1) s += __shfl_xor(s, d);
        if (lane < GL && e0 + v < p.E) lds.psum[wave * p.E + e0 + v] = s;
    }
    __syncthreads();

    // each wave a range of the slots, in order: weights, and how often each expert
    const int slots = tokens * p.k;
    const int range = (slots + kRouteWaves * 64 - 1) / (kRouteWaves * 64) * 64;
    const int lo = wave * range, hi = lo + range < slots ? lo + range : slots;
    uint32_t *hist = lds.wave_hist + wave * (p.E + 1);
    const int64_t s0 = t0 * p.k;
    for (int i = lo + lane; i < hi; i += 64) {
        const int t = (int)((uint32_t)i / (uint32_t)p.k), e = lds.expert[i];
        atomicAdd(&hist[e], 1u);
        p.experts[s0 + i] = e;
        p.weights[s0 + i] = e == p.E ? 0.f : lds.value[i] / lds.scale[t];
    }
    __syncthreads();
    // over the waves, in order; the workgroup's counts and sums
    uint32_t total = 0;
    double P = 0.0;
    if ((int)threadIdx.x <= p.E) {
        const int e = threadIdx.x;
#pragma unroll
        for (int w = 0; w < kRouteWaves; ++w) {
            uint32_t *h = &lds.wave_hist[w * (p.E + 1) + e];
            const uint32_t n = *h;
            *h = total;
            total += n;
        }
        if (e < p.E) {
#pragma unroll
            for (int w = 0; w < kRouteWaves; ++w) P += (double)lds.psum[w * p.E + e];
            if constexpr (!ONE) {
                p.hist[(int64_t)blockIdx.x * p.E + e] = total;
                p.psum[(int64_t)blockIdx.x * p.E + e] = (float)P;
            }
        }
    }
    if (p.E == 64 * kRouteWaves) {   // the masked ones' column has no lane of its own
        __syncthreads();
        if (threadIdx.x == 0) {
            uint32_t n = 0;
            for (int w = 0; w < kRouteWaves; ++w) {
                uint32_t *h = &lds.wave_hist[w * (p.E + 1) + p.E];
                const uint32_t m = *h;
                *h = n;
                n += m;
            }
        }
    }
    if constexpr (ONE) {
        const uint32_t before = before_in_block((int)threadIdx.x < p.E ? total : 0u, lds.parts);
        if ((int)threadIdx.x == p.E - 1) *lds.last = before + total;
        finish_counts(p, total, P, before, lds.parts);
        __syncthreads();
        if ((int)threadIdx.x < p.E)
#pragma unroll
            for (int w = 0; w < kRouteWaves; ++w) lds.wave_hist[w * (p.E + 1) + threadIdx.x] += before;
        if (threadIdx.x < kRouteWaves) lds.wave_hist[threadIdx.x * (p.E + 1) + p.E] += *lds.last;
    }
    __syncthreads();
    // the slots' places: those of the same expert before the range, then before it in it
    const int bits = 32 - __builtin_clz(p.E);
    for (int i0 = lo; i0 < hi; i0 += 64) {
        const int i = i0 + lane;
        const bool there = i < hi;
        const uint32_t e = there ? lds.expert[i] : 0xFFFFu;
        uint64_t same = __ballot(there);
        for (int b = 0; b < bits; ++b) {
            const uint64_t set = __ballot(e >> b & 1);
            same &= e >> b & 1 ? set : ~set;
        }
        if (there) {
            const uint32_t rank = (uint32_t)__popcll(same & (((uint64_t)1 << lane) - 1));
            const uint32_t at = hist[e] + rank;
            p.place[s0 + i] = (int32_t)at;
            if constexpr (ONE) p.order[at] = (int32_t)i;
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            if (rank == 0) hist[e] = at + (uint32_t)__popcll(same);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
}

// One workgroup to 16 experts: hist[b, e] becomes the slots of e in the workgroups
// before b; the totals go to counts, the sums of p to psum's first row.
__global__ __launch_bounds__(1024) void route_scan_kernel(RouteParams p) {
    __shared__ uint32_t sums[64][17];
    __shared__ double ps[64][17];
    const int e = blockIdx.x * 16 + threadIdx.x % 16, part = threadIdx.x / 16;
    const int each = (p.blocks + 63) / 64, lo = part * each;
    const int hi = lo + each < p.blocks ? lo + each : p.blocks;
    uint32_t n = 0;
    double P = 0.0;
    if (e < p.E)
        for (int b = lo; b < hi; ++b) {
            n += p.hist[(int64_t)b * p.E + e];
            P += (double)p.psum[(int64_t)b * p.E + e];
        }
    sums[part][threadIdx.x % 16] = n;
    ps[part][threadIdx.x % 16] = P;
    __syncthreads();
    uint32_t before = 0;
    for (int q = 0; q < part; ++q) before += sums[q][threadIdx.x % 16];
    if (e < p.E) {
        for (int b = lo; b < hi; ++b) {
            uint32_t *h = &p.hist[(int64_t)b * p.E + e];
            const uint32_t m = *h;
            *h = before;
            before += m;
        }
        if (part == 63) {
            p.counts[e] = (int32_t)before;
            P = 0.0;
            for (int q = 0; q < 64; ++q) P += ps[q][threadIdx.x % 16];
            p.psum[e] = (float)P;
        }
    }
}

// (one workgroup more than there are, the first: it writes the counts, the offsets
// and the loss)
template <bool SCANNED> __global__ __launch_bounds__(1024) void route_place_kernel(RouteParams p) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    __shared__ __attribute__((aligned(16))) uint32_t parts[4 * kRouteWaves];
    uint32_t *start = (uint32_t *)smem;   // [E + 1]
    const int e = threadIdx.x;
    const int block = (int)blockIdx.x - 1;
    const bool rest = block < 0;   // counts, offsets, loss
    const int64_t t0 = (int64_t)block * p.per, s0 = t0 * p.k;
    const int tokens = (int)(p.T - t0 < p.per ? p.T - t0 : p.per), slots = rest ? 0 : tokens * p.k;
    // on their way while the counts are added up
    const int first = e < slots ? p.experts[s0 + e] : 0, first_at = e < slots ? p.place[s0 + e] : 0;
    uint32_t total = 0, earlier = 0;      // of expert e: slots of all workgroups, of those before
    double P = 0.0;
    if constexpr (SCANNED) {
        if (e < p.E) {
            total = (uint32_t)p.counts[e];
            if (rest) P = (double)p.psum[e];
            else earlier = p.hist[(int64_t)block * p.E + e];
        }
    } else {
        // `ways` lanes to an expert, each every ways-th workgroup's counts; 32 of them at
        // most, as theirs are added up one after the other (rows and place of 4096 x 2, us:
        // 512 ways 37, 32 ways 11; 4096 x 16: 64 ways 13.5, 32 ways 11.7)
        uint32_t *sums = start + (p.E + 2) / 2 * 2;   // [2][1024]
        double *ps = (double *)(sums + 2048);         // [1024]
        const int ways = p.E > 32 ? 1024 / p.E : 32, of = e % p.E, way = e / p.E;
        if (way < ways) {
#pragma unroll 8
            for (int b = way; b < p.blocks; b += ways) {
                const uint32_t n = p.hist[(int64_t)b * p.E + of];
                total += n;
                earlier += b < block ? n : 0u;
            }
            if (rest)
#pragma unroll 8
                for (int b = way; b < p.blocks; b += ways) P += (double)p.psum[(int64_t)b * p.E + of];
            sums[e] = total;
            sums[1024 + e] = earlier;
            ps[e] = P;
        }
        __syncthreads();
        total = earlier = 0;
        P = 0.0;
        if (e < p.E)
#pragma unroll 4
            for (int w = 0; w < ways; ++w) {
                total += sums[w * p.E + e];
                earlier += sums[1024 + w * p.E + e];
                if (rest) P += ps[w * p.E + e];
            }
    }
    const uint32_t before = before_in_block(total, parts);
    if (rest) {
        finish_counts(p, total, P, before, parts);
        return;
    }
    if (e < p.E) {
        start[e] = before + earlier;
        if (e == p.E - 1) start[p.E] = before + total;   // behind the last group
    }
    __syncthreads();
    if (p.mask) {
        // and the masked slots of the workgroups before: all of theirs less the experts'
        const uint32_t upto = before_in_block(earlier, parts) + earlier;
        __syncthreads();
        if (e == 64 * kRouteWaves - 1) start[p.E] += (uint32_t)s0 - upto;
        __syncthreads();
    }
    for (int i = threadIdx.x; i < slots; i += 1024) {
        const uint32_t at = i == e ? start[first] + (uint32_t)first_at
                                   : start[p.experts[s0 + i]] + (uint32_t)p.place[s0 + i];
        p.place[s0 + i] = (int32_t)at;
        p.order[at] = (int32_t)(s0 + i);
    }
}

// LDS writes of a wave's other lanes before reads, and back
OZK_DEV void settle_wave() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// The logits' gradient.  With q = softmax(l), c_e the counts and n the tokens:
//   dl = q (g - sum q g), g_e = dloss E c_e / (n k n), and
//   normalised weights (a softmax over the chosen): dl at them += w (dw - sum w dw)
//   others (q at the chosen): g at them += dw
template <typename T, int GL, int V>
__global__ __launch_bounds__(256) void route_grad_kernel(RouteGradParams p) {
    constexpr int TPW = 64 / GL;
    __shared__ __attribute__((aligned(16))) float spread[4][TPW][GL * V];
    const int lane = threadIdx.x & 63, in = lane % GL, e0 = in * V;
    float *at_experts = spread[threadIdx.x >> 6][lane / GL];
    float g0[V] = {};
    if (p.dloss) {
        uint32_t c[V], sum = 0;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            c[v] = e0 + v < p.E ? (uint32_t)p.counts[e0 + v] : 0u;
            sum += c[v];
        }
        sum = over_group<GL>(sum, [](uint32_t a, uint32_t b) { return a + b; });
        const double n = (double)sum / p.k;
        // less their mean, which changes nothing in g - sum q g: balanced counts would
        // cancel there in 32 bits
        const double by = sum ? (double)*p.dloss * p.E / ((double)sum * n) : 0.0;
#pragma unroll
        for (int v = 0; v < V; ++v) g0[v] = (float)(by * ((double)c[v] - (double)sum / p.E));
    }
    const int64_t step = (int64_t)gridDim.x * 4 * TPW;
    for (int64_t r = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * TPW; r < p.T; r += step) {
        const int64_t t = r + lane / GL;
        const bool there = t < p.T, valid = there && (!p.mask || p.mask[t]);
        float l[V], g[V], d[V] = {};
        logits_at<T, V>(p.logits + t * p.pitch * (int64_t)sizeof(T), e0, p.E, valid, l);
        float top = l[0];
        bool nan = l[0] != l[0];
#pragma unroll
        for (int v = 1; v < V; ++v) {
            top = l[v] > top ? l[v] : top;
            nan |= l[v] != l[v];
        }
        // (max as whole numbers orders by value, too; NaN is carried by the sums)
        top = over_group<GL>(nan ? __builtin_inff() : top, [](float a, float b) { return a > b ? a : b; });
        float sum = 0.f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            l[v] = e0 + v < p.E ? expf(l[v] - top) : 0.f;
            sum += l[v];
            g[v] = g0[v];
        }
        sum = group_sum<GL>(sum);
        const float by = 1.f / sum;
        if (p.dw) {
            // lane j has the token's j-th choice; through the LDS to its expert's lane
            const int64_t s = t * p.k;
            float mean = 0.f;
            if (p.normalize) {
                for (int j = in; j < p.k; j += GL)
                    if (valid) mean = fmaf(p.weights[s + j], p.dw[s + j], mean);
                mean = group_sum<GL>(mean);
            }
#pragma unroll
            for (int v = 0; v < V; ++v) at_experts[e0 + v] = 0.f;
            settle_wave();
            for (int j = in; j < p.k; j += GL) {
                const uint32_t e = valid ? (uint32_t)p.experts[s + j] : 0xFFFFFFFFu;
                if (e < (uint32_t)p.E)   // whatever the tensor holds
                    at_experts[e] = p.normalize ? p.weights[s + j] * (p.dw[s + j] - mean) : p.dw[s + j];
            }
            settle_wave();
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float add = at_experts[e0 + v];
                if (p.normalize) d[v] = add;
                else g[v] += add;
            }
            settle_wave();
        }
        float dot = 0.f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            l[v] *= by;
            dot = fmaf(l[v], e0 + v < p.E ? g[v] : 0.f, dot);
        }
        dot = group_sum<GL>(dot);
        if (!there) continue;
#pragma unroll
        for (int v = 0; v < V; ++v) d[v] = valid ? fmaf(l[v], g[v] - dot, d[v]) : 0.f;
        char *out = p.dlogits + t * p.E * (int64_t)sizeof(T);
        if (e0 + V <= p.E) {
            T o[V];
#pragma unroll
            for (int v = 0; v < V; ++v) o[v] = (T)d[v];
            __builtin_memcpy(out + (int64_t)e0 * sizeof(T), o, V * sizeof(T));
        } else {
#pragma unroll
            for (int v = 0; v < V; ++v)
                if (e0 + v < p.E) store_value<T>(out, e0 + v, d[v]);
        }
    }
}

namespace {

// Lanes of a token and values of a lane, by E.  4 values: with 8 a wave takes twice
// the tokens at once, which pays only where there are many (rows alone, us, with 4 /
// with 8, unsorted: 32768 x 64, k = 8, fp32 13.4 / 12.5, 12.3 with 4 sorted; 4099 x 40,
// k = 3, bf16 6.3 / 8.1; 16 x 16, k = 2 6.8 / 7.8).
template <typename F> hipError_t with_shape(int E, F &&f) {
    using std::integral_constant;
#define OZK_ROUTE(GL, V) return f(integral_constant<int, GL>{}, integral_constant<int, V>{})
    if (E <= 8) OZK_ROUTE(2, 4);
    if (E <= 16) OZK_ROUTE(4, 4);
    if (E <= 32) OZK_ROUTE(8, 4);
    if (E <= 64) OZK_ROUTE(16, 4);
    if (E <= 128) OZK_ROUTE(32, 4);
    if (E <= 256) OZK_ROUTE(64, 4);
    if (E <= 512) OZK_ROUTE(64, 8);
    OZK_ROUTE(64, 16);
#undef OZK_ROUTE
}
int lanes_of(int E) {
    int lanes = 2;
    while (lanes < 64 && E > 4 * lanes) lanes *= 2;
    return lanes;
}

template <typename T> hipError_t route_go(const RouteParams &p, hipStream_t st) {
    return with_shape(p.E, [&](auto gl, auto v) {
        constexpr int GL = decltype(gl)::value, V = decltype(v)::value;
        const size_t lds = RouteLds::bytes(p.E, p.per, p.k);
        if (p.blocks == 1) {
            if (hipError_t e = allow_lds<&route_rows_kernel<T, GL, V, true>>((int)lds); e != hipSuccess)
                return e;
            route_rows_kernel<T, GL, V, true><<<1, 64 * kRouteWaves, lds, st>>>(p);
        } else {
            if (hipError_t e = allow_lds<&route_rows_kernel<T, GL, V, false>>((int)lds); e != hipSuccess)
                return e;
            route_rows_kernel<T, GL, V, false><<<(uint32_t)p.blocks, 64 * kRouteWaves, lds, st>>>(p);
        }
        return hipGetLastError();
    });
}
template <typename T> hipError_t route_grad_go(const RouteGradParams &p, hipStream_t st) {
    return with_shape(p.E, [&](auto gl, auto v) {
        constexpr int GL = decltype(gl)::value, V = decltype(v)::value;
        const int64_t blocks = (p.T + 4 * (64 / GL) - 1) / (4 * (64 / GL));
        route_grad_kernel<T, GL, V><<<(uint32_t)(blocks < 4096 ? blocks : 4096), 256, 0, st>>>(p);
        return hipGetLastError();
    });
}

}  // namespace

void plan_route(RouteParams &p) {
    // a workgroup's tokens: whole steps of its waves, a workgroup to a CU, or two where
    // that leaves 6 steps each, as many as the LDS of two or of one holds (rows and place,
    // us, 256 / 512 workgroups: 32768 x 64, k = 8, fp32 19.3 / 22.3; 300000 x 64 84 / 76;
    // 65536 x 256, k = 8, bf16 64 / 61)
    const int64_t step = (int64_t)kRouteWaves * 64 / lanes_of(p.E);
    const int64_t fixed = (int64_t)RouteLds::bytes(p.E, 0, 0), each = 4 + 6 * p.k;
    const int64_t room = fixed + step * each <= 78 * 1024 ? 78 * 1024 : 150 * 1024;
    const int64_t most = (room - fixed) / each;
    const int64_t blocks = p.T > 256 * 12 * step ? 512 : 256;
    int64_t per = ((p.T + blocks - 1) / blocks + step - 1) / step * step;
    if (per > most) per = most < step ? most : most / step * step;
    if (per == 0) per = step;
    p.per = per;
    p.blocks = p.T > per ? (int)((p.T + per - 1) / per) : 1;
}

hipError_t launch_route(const RouteParams &p, int dtype, hipStream_t st) {
    hipError_t e = dtype == OZK_F32   ? route_go<float>(p, st)
                   : dtype == OZK_F16 ? route_go<_Float16>(p, st)
                                      : route_go<__bf16>(p, st);
    if (e != hipSuccess || p.blocks == 1) return e;
    // up to 32 counts to a lane are read again by every workgroup
    if ((int64_t)p.blocks * p.E <= 32 * 1024) {
        const size_t lds = 4 * ((p.E + 2) / 2 * 2) + 8 * 1024 + 8 * 1024;
        route_place_kernel<false><<<(uint32_t)p.blocks + 1, 1024, lds, st>>>(p);
        return hipGetLastError();
    }
    route_scan_kernel<<<(uint32_t)((p.E + 15) / 16), 1024, 0, st>>>(p);
    if (e = hipGetLastError(); e != hipSuccess) return e;
    route_place_kernel<true><<<(uint32_t)p.blocks + 1, 1024, 4 * (p.E + 1), st>>>(p);
    return hipGetLastError();
}
hipError_t launch_route_grad(const RouteGradParams &p, int dtype, hipStream_t st) {
    return dtype == OZK_F32   ? route_grad_go<float>(p, st)
           : dtype == OZK_F16 ? route_grad_go<_Float16>(p, st)
                              : route_grad_go<__bf16>(p, st);
}

}  // namespace ozk
