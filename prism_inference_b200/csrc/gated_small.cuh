// gated_small.cuh - the gated feed-forward block for a few rows (gated_small.cu), as gated_ffn.cu calls it.
#pragma once
#include "gated_tc.cuh"

namespace prism {

// Up to 8 rows, while the multiplications (on the CUDA cores) stay small beside the weights' bytes.
// Measured against the tensor-core path: 1 row of 256 x 1024 3.9 us against 25, 8 rows 11.8 against 25; 1
// row of 1024 x 4096 8.2 against 33, 4 rows 25 against 33, but 8 rows 45 against 33.
constexpr int kSmallRows = 8;
inline bool is_small(int64_t rows, int64_t dim, int64_t hidden) {
    return rows <= kSmallRows && (rows - 1) * dim * hidden <= 1 << 24;
}

struct SmallArgs {
    int rows, dim, hidden, act;
    const void *x, *w_gate, *b_gate, *w_up, *b_up, *w_down, *b_down, *residual;
    int64_t xs, rs, ys;
    float* h;  // workspace [rows][hidden]
    void* y;
};
cudaError_t launch_gated_small(bool bf16, const SmallArgs& a, cudaStream_t s);

}  // namespace prism
