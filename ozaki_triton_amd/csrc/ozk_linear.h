// ozk_linear.h -- parameter blocks and launchers of the operators for linear
// layers, shared between their C entry points (ozk_linear_api.cpp) and their
// kernels.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <atomic>

namespace ozk {

// Raises kernel K's dynamic-LDS limit where `bytes` needs it, once per device.
template <auto K> hipError_t allow_lds(int bytes) {
    static std::atomic<uint64_t> done{0};
    if (bytes <= 64 * 1024) return hipSuccess;
    int dev = 0;
    if (hipError_t e = hipGetDevice(&dev); e != hipSuccess) return e;
    const uint64_t bit = dev < 64 ? (uint64_t)1 << dev : 0;
    if (done.load(std::memory_order_relaxed) & bit) return hipSuccess;
    const hipError_t e = hipFuncSetAttribute(
        (const void *)K, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
    if (e == hipSuccess) done.fetch_or(bit, std::memory_order_relaxed);
    return e;
}

// C[t, n] = sum_k A[t, k] B[g(t), k, n] with rows offsets[g] .. offsets[g + 1]
// of group g; rows of no group get zeros.
struct GroupedParams {
    const char *A;          // [T, K], rows of a_pitch bytes
    const char *B;          // [G] matrices, b_group bytes apart; rows of b_pitch bytes:
    char *C;                // K rows of N (b_cols) or N rows of K
    const void *offsets;    // [G + 1], int32 or int64
    int64_t T, K, N, G;
    int64_t a_pitch, b_group, b_pitch, c_pitch;
    int b_cols, offsets64;
    bool a_padded, b_padded;   // rows go on with zeros up to a whole 16-byte piece
};
// dB[g, k, n] = sum over the rows t of group g of A[t, k] D[t, n]
struct GroupedGradParams {
    const char *A;          // [T, K]
    const char *D;          // [T, N]
    char *dB;               // [G, K, N], matrices db_group bytes apart
    const void *offsets;
    int64_t T, K, N, G;
    int64_t a_pitch, d_pitch, db_group, db_pitch;
    int offsets64;
    bool a_padded, d_padded;
    float *part;            // workspace: partial sums of the row ranges (splits > 1)
    int splits;
    // set by the launch
    int64_t share;      // rows of a group on average
    uint32_t block;     // tiles on a side of the squares they are taken in
};
// Operands that are copied to whole 16-byte pieces first (packed): the bytes of
// the copies, 0 for none.  plan_* say which; pack_* point the parameters at the
// copies in `ws` and enqueue them.
struct PackedSizes {
    size_t a, b;
    size_t total() const { return a + b; }
};
PackedSizes plan_grouped_pack(const GroupedParams &p);
PackedSizes plan_grad_pack(const GroupedGradParams &p);
hipError_t pack_grouped(GroupedParams &p, const PackedSizes &n, char *ws, hipStream_t st);
hipError_t pack_grad(GroupedGradParams &p, const PackedSizes &n, char *ws, hipStream_t st);
// dtype: 2 fp16, 3 bf16
hipError_t launch_grouped(const GroupedParams &p, int dtype, hipStream_t st);
hipError_t launch_grouped_grad(const GroupedGradParams &p, int dtype, hipStream_t st);
int grouped_grad_splits(int64_t T, int64_t K, int64_t N, int64_t G);


// y[m, n] = sum_k x[m, k] (q[n, k] - z[n, k / group]) s[n, k / group]
struct W4Params {
    const char *x;            // [M, K], rows of x_pitch elements
    const uint8_t *packed;    // [N], rows of w_pitch bytes, k even in the low half of byte k / 2
    const void *scales;       // [N, groups], rows of s_pitch elements
    const uint8_t *zeros;     // [N, groups], rows of z_pitch; null: every zero point is 8
    char *y;                  // [M, N], rows of y_pitch elements
    int64_t M, N, K;
    int64_t x_pitch, w_pitch, s_pitch, z_pitch, y_pitch;
    int scales32;             // scales are fp32 (else x's type)
    int group;                // 32, 64 or 128
    float *part;              // workspace [splits, M, N] where splits > 1
    int splits, range;        // K ranges and elements of one (whole chunks of 128)
    int held;                 // elements of K of x in the LDS at a time
};
// dtype: 1 fp32, 2 fp16, 3 bf16
void plan_w4(W4Params &p, int dtype);
hipError_t launch_w4(const W4Params &p, int dtype, hipStream_t st);

struct QuantParams {
    const char *W;            // [N, K], rows of w_pitch elements (null: dequantise into out)
    char *out;
    uint8_t *packed;
    char *scales;             // W's type
    uint8_t *zeros;           // null: symmetric, zero point 8
    int64_t N, K, w_pitch, p_pitch, s_pitch, z_pitch;
    int group;
};
hipError_t launch_quantize_w4(const QuantParams &p, int dtype, hipStream_t st);
hipError_t launch_dequantize_w4(const QuantParams &p, int dtype, int scale_dtype, hipStream_t st);

// Newton-Schulz orthogonalisation of batch matrices G [M, N]; inside, X is
// [m, n] with m <= n (G transposed where M > N).  A plan is a list of products
//   D = f_acc L R + f_y Y + f_i I
// of matrices that are kept as slices, the last one into the result.
enum OrthKind {
    kOrthXX = 0,     // D [m, m] = X X^T
    kOrthSym = 1,    // D [m, m] symmetric, L and R symmetric and commuting
    kOrthX = 2,      // D [m, n], R and Y of X's size
    kOrthLast = 3,   // the same into the result
    // where the scales are measured (OrthPlan): through fp32 values, their norm and
    // slices of them over it
    kOrthNewB = 4,   // D [m, m], of A
    kOrthNewX = 5    // D [m, n], of B and X
};
constexpr int kOrthSquares = 5;   // [m, m] buffers
struct OrthOp {
    int kind;
    int L, R, Y, D;          // buffers: 0 .. 4 square, -1 and -2 X's two, -9 none
    float f_acc, f_y, f_i;   // scales of the slices included (not the measured ones)
};
constexpr int kOrthMaxOps = 4 * 64;
struct OrthPlan {
    OrthOp op[kOrthMaxOps];
    int ops;
    int squares, xs;         // buffers used
    float start_scale;       // of X's slices at the start, a power of two
    bool measured;           // slices of X / |X|, of A / |X|^2 and of B / |B|, norms on the GPU
};
struct OrthParams {
    const char *G;
    char *out;
    int64_t batch, M, N;
    int64_t g_batch, g_row, o_batch, o_row;    // elements
    double eps;
    float start_scale;
    // workspace
    double *sums;                              // [batch, blocks] partial sums of squares
    int blocks;
    double *norms;                             // [2, batch], |X| and |B| where measured, else null
    char *X[2], *S[kOrthSquares];              // slices
};
int orth_blocks(int64_t batch, int64_t M, int64_t N);
hipError_t launch_orth(const OrthParams &p, const OrthPlan &plan, int dtype, hipStream_t st);

}  // namespace ozk
