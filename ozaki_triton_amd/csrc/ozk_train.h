// ozk_train.h -- parameter blocks and launchers of what stands around a model's
// linear layers in training and serving: the dense product with its epilogue
// (ozk_dense.h), the router (ozk_route.hip), gradient norms and clipping
// (ozk_clip.hip); shared between their C entry points (ozk_train_api.cpp) and
// their kernels.
#pragma once

#include "ozk_linear.h"

namespace ozk {

// C[m, n] = act(sum_k A[m, k] B[n, k] + bias[n]) + res[m, n]
struct DenseParams {
    const char *A;           // [M, K], rows of a_pitch bytes (wgrad: K rows of M)
    const char *B;           // N rows of K, b_pitch bytes apart, or K rows of N (b_cols)
    char *C;                 // [M, N]
    const char *bias;        // [N] or null
    const char *res;         // [M, N] or null
    char *Z;                 // null, or [M, N], rows of N: what act is applied to, rounded
    int64_t M, N, K;
    int64_t a_pitch, b_pitch, c_pitch, r_pitch;   // bytes
    int act;                 // OZK_ACT_*
    bool a_cols, b_cols;
    bool a_padded, b_padded;   // rows go on with zeros up to a whole 16-byte piece
    float *part;             // workspace [splits, M, N]: partial sums of the K ranges (splits > 1)
    int splits;
    // where given, workgroups behind the tiles' add up db (DenseGradParams)
    const float *sums;
    char *db;
    int64_t db_n, db_blocks;
};
// a product of a few rows, which is not cut into tiles
bool dense_few(const DenseParams &p);
// K ranges that the product is cut into
int dense_splits(const DenseParams &p);
hipError_t launch_dense(const DenseParams &p, int dtype, hipStream_t st);

// dz = dy act'(z), and partial column sums of dz
struct DenseGradParams {
    const char *dy;          // [M, N]
    const char *z;           // [M, N], rows of N; null: act is the identity
    char *dz;                // [M, N], rows of dz_pitch bytes, zeros behind N (null: not wanted)
    float *sums;             // [blocks, N] (null: not wanted)
    char *db;                // [N]
    int64_t M, N, dy_pitch, dz_pitch;
    int act;
    int64_t rows;            // of a workgroup
    int lanes;               // set by the launch
};
int64_t dense_grad_rows(int64_t M, int64_t N);   // rows of a workgroup
hipError_t launch_dense_grad(const DenseGradParams &p, int dtype, hipStream_t st);
hipError_t launch_dense_bias(const DenseGradParams &p, int dtype, hipStream_t st);

// The router: see ozk_route.hip
struct RouteParams {
    const char *logits;      // [T, E], rows of pitch elements
    const uint8_t *mask;     // [T], 0: the token is left out; null: none is
    int64_t T, pitch;
    int E, k, normalize;
    int32_t *experts;        // [T, k]
    float *weights;          // [T, k]
    int32_t *order, *place;  // [T k], [T, k]
    int32_t *offsets;        // [E + 1]
    int32_t *counts;         // [E]
    float *loss;
    // workspace
    uint32_t *hist;          // [blocks, E]: slots of each expert, later those before the block
    float *psum;             // [blocks, E]: sums of the probabilities
    int64_t per;             // tokens of a workgroup
    int blocks;
};
void plan_route(RouteParams &p);
hipError_t launch_route(const RouteParams &p, int dtype, hipStream_t st);
struct RouteGradParams {
    const char *logits;
    const uint8_t *mask;
    int64_t T, pitch;
    int E, k, normalize;
    const int32_t *experts, *counts;
    const float *weights;
    const float *dw;         // [T, k] or null
    const float *dloss;      // one value, or null
    char *dlogits;           // [T, E], rows of E
};
hipError_t launch_route_grad(const RouteGradParams &p, int dtype, hipStream_t st);

// Norm of many tensors and their scaling: see ozk_clip.hip
struct ClipTensor {
    const char *in;
    char *out;
    int64_t n;
    uint32_t first;          // its first piece
    int dtype;
};
constexpr int kClipTensors = 112;   // of one launch (a launch takes 4 KB of arguments)
struct ClipParams {
    ClipTensor t[kClipTensors];
    int count;
    uint32_t pieces;         // of all tensors of the launch
    uint32_t size;           // elements of a piece
    uint32_t part0, parts;   // first partial sum of this launch, and how many all have
    double *part;
    double max_norm;
    bool past_caches;        // the tensors are more than the memory-side cache holds
    float *norm;             // written by the launch that has it, else null
};
hipError_t launch_square_sums(const ClipParams &p, uint32_t grid, hipStream_t st);
hipError_t launch_norm(const ClipParams &p, hipStream_t st);
hipError_t launch_scale(const ClipParams &p, uint32_t grid, hipStream_t st);

}  // namespace ozk
