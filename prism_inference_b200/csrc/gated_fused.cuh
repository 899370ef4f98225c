// gated_fused.cuh - the gated feed-forward kernels for dim <= 256 (gated_fused.cu), as gated_ffn.cu calls
// them.
#pragma once
#include "gated_tc.cuh"

namespace prism {

constexpr int kFusedMaxDim = 256;

// Tensor maps: x and dy [rows][dim] with boxes {64, 128}; w_gate, w_up [hidden][dim] with boxes {64, 128}
// forward, {64, 64} backward; the others by direction.
struct FusedMaps {
    CUtensorMap x, wg, wu, out;  // out: y or dx, box {32, 32}
    CUtensorMap residual;        // forward, where there is one: box {32, 32}
    CUtensorMap wd;              // forward: [dim][hidden], box {64, bn / 2}; backward: box {32, 128}, 64-byte swizzle
    CUtensorMap dy, wg_mn, wu_mn, p;  // backward: boxes {64, 64} of the weights; p [3][rows][hidden] (dg, du, h), box {64, 32}
};
struct FusedArgs {
    int rows, dim, hidden;
    int tiles;   // of 256 rows
    int bn;      // N of the products over dim: 128 or 256
    int act;
    const void *b_gate, *b_up, *b_down;
    int residual;  // forward: there is one
    int first;              // backward: the first chunk of rows, the column sums start here
    float *sums, *sums_dy;  // backward: [CTAs][4][2 hidden] of dg and du, [CTAs][dim] of dy
    uint32_t* err;
};

// CTA pairs of a launch over `tiles` row tiles
inline int fused_pairs(int tiles, int sm_count) { return tiles < sm_count / 2 ? tiles : sm_count / 2; }
cudaError_t launch_gated_fused(bool bf16, bool backward, const FusedArgs& a, const FusedMaps& m, const prism_ctx* ctx, cudaStream_t s);

}  // namespace prism
