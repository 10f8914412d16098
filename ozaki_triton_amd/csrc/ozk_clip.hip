// ozk_clip.hip -- the norm of many tensors taken as one vector, and their scaling
// to a norm of at most max_norm.
//
// norm = sqrt(sum of squares), in 64 bits from each element on: the square of an
// fp32 or bf16 value can be past fp32's range in both directions, and sums of 1e9
// elements would lose their last ones in 32 bits.  The sum is that of fixed parts
// in a fixed order (no atomics): the same bits every time.
//
// Tensors are cut into pieces of one size, which the workgroups take in turn; a
// launch carries its tensors' addresses in its arguments (so a captured graph
// keeps them), kClipTensors at most.  Bound by memory: every element read once
// for the norm, read and written once more for the scaling (268M bf16 elements: 83 us,
// 6.5 TB/s, and 192 us, 5.6 TB/s).
#include "../../include/ozaki_amd.h"
#include "ozk_train.h"
#include "ozk_tile.h"

namespace ozk {

// The tensor that holds piece i (the last whose first piece is not past it):
// every lane compares two of them
OZK_DEV int tensor_of(const ClipParams &p, uint32_t i) {
    const int lane = threadIdx.x & 63;
    const bool a = lane < p.count && p.t[lane].first <= i;
    const bool b = lane + 64 < p.count && p.t[lane + 64 < kClipTensors ? lane + 64 : 0].first <= i;
    return __popcll(__ballot(a)) + __popcll(__ballot(b)) - 1;
}
struct Piece {
    const char *in;
    char *out;
    int n, dtype;   // elements
};
OZK_DEV Piece piece_of(const ClipParams &p, uint32_t i) {
    const ClipTensor &t = p.t[uniform(tensor_of(p, i))];
    const int64_t at = (int64_t)(i - t.first) * p.size, left = t.n - at;
    const int64_t byte = at * (t.dtype == OZK_F32 ? 4 : 2);
    return {t.in + byte, t.out + byte, (int)(left < p.size ? left : p.size), t.dtype};
}

template <typename T> OZK_DEV void values(i32x4 v, float (&f)[16 / sizeof(T)]) {
    if constexpr (sizeof(T) == 4) {
        __builtin_memcpy(f, &v, 16);
    } else {
        uint16_t e[8];
        __builtin_memcpy(e, &v, 16);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = from_bits16(e[i], T{});
    }
}

// 16 bytes of any alignment.  NT: past the caches, for tensors of more than these
// hold: reads then need not wait for the dirty lines that they would push out of the
// memory-side cache (512 MiB in 60 tensors, a call, norm / norm and scaling in place: 94 /
// 321 us without, 85 / 274 with).
typedef int i32x4_any __attribute__((ext_vector_type(4), aligned(2)));
template <bool NT> OZK_DEV i32x4 load16(const char *p) {
    if constexpr (NT) return __builtin_nontemporal_load((const i32x4_any *)p);
    else return *(const i32x4_any *)p;
}
template <bool NT> OZK_DEV void store16(char *p, i32x4 v) {
    if constexpr (NT) __builtin_nontemporal_store((i32x4_any)v, (i32x4_any *)p);
    else *(i32x4_any *)p = v;
}

// A piece by the 256 lanes of a workgroup: whole 16-byte parts, four at a time, then
// the elements behind the last.
constexpr int kAtOnce = 4;

template <typename T, bool NT> OZK_DEV double piece_squares(const Piece &c) {
    constexpr int V = 16 / sizeof(T);
    const int parts = c.n / V;
    double s[4] = {};
    auto add = [&](i32x4 v) {
        float f[V];
        values<T>(v, f);
#pragma unroll
        for (int i = 0; i < V; ++i) s[i & 3] = fma((double)f[i], (double)f[i], s[i & 3]);
    };
    int i = threadIdx.x;
    for (; i + (kAtOnce - 1) * 256 < parts; i += kAtOnce * 256) {
        i32x4 v[kAtOnce];
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) v[u] = load16<NT>(c.in + (int64_t)(i + u * 256) * 16);
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) add(v[u]);
    }
    for (; i < parts; i += 256) add(load16<NT>(c.in + (int64_t)i * 16));
    if ((int)threadIdx.x < c.n - parts * V) {
        const double x = (double)load_value<T>(c.in, parts * V + threadIdx.x);
        s[0] = fma(x, x, s[0]);
    }
    return (s[0] + s[1]) + (s[2] + s[3]);
}

// the 256 lanes' values, in a fixed order, in every lane
OZK_DEV double sum256(double v) {
    __shared__ double part[4];
#pragma unroll
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    return (part[0] + part[1]) + (part[2] + part[3]);
}

template <bool NT> __global__ __launch_bounds__(256) void square_sums_kernel(ClipParams p) {
    double s = 0.0;
    for (uint32_t i = blockIdx.x; i < p.pieces; i += gridDim.x) {
        const Piece c = piece_of(p, i);
        s += c.dtype == OZK_F32   ? piece_squares<float, NT>(c)
             : c.dtype == OZK_F16 ? piece_squares<_Float16, NT>(c)
                                  : piece_squares<__bf16, NT>(c);
    }
    s = sum256(s);
    if (threadIdx.x == 0) p.part[p.part0 + blockIdx.x] = s;
}

// the norm of all partial sums, in every lane of a workgroup
OZK_DEV double norm_of(const ClipParams &p) {
    double s = 0.0;
#pragma unroll 4
    for (uint32_t i = threadIdx.x; i < p.parts; i += 256) s += p.part[i];
    return sqrt(sum256(s));
}

__global__ __launch_bounds__(256) void norm_kernel(ClipParams p) {
    const double norm = norm_of(p);
    if (threadIdx.x == 0) *p.norm = (float)norm;
}

// fp32: the product in 64 bits, rounded once.  16 bits: in 32 bits, whose rounding is
// 2^-13 of theirs, by's exponent apart, as by itself may be below 32 bits' range (a bf16
// value of 3e38 times 1e-45 is an ordinary number).
template <typename T, bool NT> OZK_DEV void piece_scale(const Piece &c, double by) {
    constexpr int V = 16 / sizeof(T);
    const int parts = c.n / V;
    int exponent;
    const float mantissa = (float)frexp(by, &exponent);
    auto one = [&](float f) {   // the same for every element, wherever it lies
        if constexpr (sizeof(T) == 4) return (float)((double)f * by);
        else return __builtin_ldexpf(f * mantissa, exponent);
    };
    auto scaled = [&](i32x4 v) {
        float f[V];
        values<T>(v, f);
        i32x4 r;
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < V; ++i) f[i] = one(f[i]);
            __builtin_memcpy(&r, f, 16);
        } else {
            uint16_t e[V];
#pragma unroll
            for (int i = 0; i < V; ++i) e[i] = to_bits16(one(f[i]), T{});
            __builtin_memcpy(&r, e, 16);
        }
        return r;
    };
    int i = threadIdx.x;
    for (; i + (kAtOnce - 1) * 256 < parts; i += kAtOnce * 256) {
        i32x4 v[kAtOnce];
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) v[u] = load16<NT>(c.in + (int64_t)(i + u * 256) * 16);
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u)
            store16<NT>(c.out + (int64_t)(i + u * 256) * 16, scaled(v[u]));
    }
    for (; i < parts; i += 256)
        store16<NT>(c.out + (int64_t)i * 16, scaled(load16<NT>(c.in + (int64_t)i * 16)));
    if ((int)threadIdx.x < c.n - parts * V) {
        const int64_t at = parts * V + threadIdx.x;
        store_value<T>(c.out, at, one(load_value<T>(c.in, at)));
    }
}

template <bool NT> __global__ __launch_bounds__(256) void scale_kernel(ClipParams p) {
    const double norm = norm_of(p);
    if (p.norm && blockIdx.x == 0 && threadIdx.x == 0) *p.norm = (float)norm;
    // NaN makes everything NaN
    const double by = norm <= p.max_norm ? 1.0 : p.max_norm / norm;
    // the last pieces first: the memory-side cache holds what the norm's pass read last
    for (uint32_t j = blockIdx.x; j < p.pieces; j += gridDim.x) {
        const Piece c = piece_of(p, p.pieces - 1 - j);
        if (by == 1.0 && c.in == c.out) continue;
        if (c.dtype == OZK_F32) piece_scale<float, NT>(c, by);
        else if (c.dtype == OZK_F16) piece_scale<_Float16, NT>(c, by);
        else piece_scale<__bf16, NT>(c, by);
    }
}

hipError_t launch_square_sums(const ClipParams &p, uint32_t grid, hipStream_t st) {
    if (p.past_caches) square_sums_kernel<true><<<dim3(grid), 256, 0, st>>>(p);
    else square_sums_kernel<false><<<dim3(grid), 256, 0, st>>>(p);
    return hipGetLastError();
}
hipError_t launch_norm(const ClipParams &p, hipStream_t st) {
    norm_kernel<<<dim3(1), 256, 0, st>>>(p);
    return hipGetLastError();
}
hipError_t launch_scale(const ClipParams &p, uint32_t grid, hipStream_t st) {
    if (p.past_caches) scale_kernel<true><<<dim3(grid), 256, 0, st>>>(p);
    else scale_kernel<false><<<dim3(grid), 256, 0, st>>>(p);
    return hipGetLastError();
}

}  // namespace ozk
