// gated_small.cu - the gated feed-forward block for a few rows (a token or a handful): no tensor tile is
// worth filling, the weights' bytes and the latency count.
//
// Two launches.  The first gives each warp hidden columns: its lanes read a gate row and an up row in
// 16-byte pieces, multiply them with all the rows of x and leave h in fp32 in the workspace.  The second
// gives each warp an output column the same way.  All warps of the GPU stream weights at once; the second
// launch starts while the first runs and has its first weights in registers when h is there.
#include "gated_small.cuh"

namespace prism {
namespace {

constexpr int kThreads = 128, kWarps = kThreads / 32;

template <typename T>
PRISM_DEV void unpack8(const uint4& v, float (&f)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) unpack2<T>(w[j], f[2 * j], f[2 * j + 1]);
}
PRISM_DEV float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// h[r][j] for hidden column j = a warp
template <typename T, int R>
__global__ void __launch_bounds__(kThreads) small_up_kernel(const SmallArgs a) {
    grid_dep_wait();
    grid_dep_launch();  // the next launch may start: what came before this one is done
    const int lane = threadIdx.x & 31, j = blockIdx.x * kWarps + threadIdx.x / 32;
    if (j >= a.hidden) return;
    const T *wg = static_cast<const T*>(a.w_gate) + (int64_t)j * a.dim, *wu = static_cast<const T*>(a.w_up) + (int64_t)j * a.dim;
    const T* x = static_cast<const T*>(a.x);
    float g[R], u[R];
#pragma unroll
    for (int r = 0; r < R; ++r) g[r] = u[r] = 0.0f;
#pragma unroll 2
    for (int k = lane * 8; k < a.dim; k += 256) {
        float fg[8], fu[8];
        unpack8<T>(*reinterpret_cast<const uint4*>(wg + k), fg);
        unpack8<T>(*reinterpret_cast<const uint4*>(wu + k), fu);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float fx[8];
            unpack8<T>(r < a.rows ? *reinterpret_cast<const uint4*>(x + r * a.xs + k) : make_uint4(0, 0, 0, 0), fx);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                g[r] = fmaf(fg[e], fx[e], g[r]);
                u[r] = fmaf(fu[e], fx[e], u[r]);
            }
        }
    }
    float gv = 0.0f, uv = 0.0f;  // lane r keeps row r
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const float sg = warp_sum(g[r]), su = warp_sum(u[r]);
        if (lane == r) gv = sg, uv = su;
    }
    if (lane < R && lane < a.rows) {
        if (a.b_gate) gv += to_f32(static_cast<const T*>(a.b_gate)[j]);
        if (a.b_up) uv += to_f32(static_cast<const T*>(a.b_up)[j]);
        const float h = a.act == kActSilu ? gate<kActSilu>(gv) : a.act == kActGelu ? gate<kActGelu>(gv) : gate<kActRelu>(gv);
        a.h[(int64_t)lane * a.hidden + j] = h * uv;
    }
}

// y[r][d] for output column d = a warp
template <typename T, int R>
__global__ void __launch_bounds__(kThreads) small_down_kernel(const SmallArgs a) {
    const int lane = threadIdx.x & 31, d = blockIdx.x * kWarps + threadIdx.x / 32;
    // 16-byte pieces of the weights read before h is there: the launch before has seen everything earlier done
    // before it let this one start
    constexpr int kAhead = 4;
    uint4 w[kAhead];
    const T* wd = static_cast<const T*>(a.w_down) + (int64_t)min(d, a.dim - 1) * a.hidden;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
        const int k = lane * 8 + 256 * i;
        w[i] = k < a.hidden ? *reinterpret_cast<const uint4*>(wd + k) : make_uint4(0, 0, 0, 0);
    }
    grid_dep_wait();
    if (d >= a.dim) return;
    float y[R];
#pragma unroll
    for (int r = 0; r < R; ++r) y[r] = 0.0f;
    auto add = [&](const uint4& v, int k) {
        float f[8];
        unpack8<T>(v, f);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (r >= a.rows) break;
            const float4* h = reinterpret_cast<const float4*>(a.h + (int64_t)r * a.hidden + k);
            const float4 p = h[0], q = h[1];
            const float fh[8] = {p.x, p.y, p.z, p.w, q.x, q.y, q.z, q.w};
#pragma unroll
            for (int e = 0; e < 8; ++e) y[r] = fmaf(f[e], fh[e], y[r]);
        }
    };
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
        if (lane * 8 + 256 * i < a.hidden) add(w[i], lane * 8 + 256 * i);
#pragma unroll 2
    for (int k = lane * 8 + 256 * kAhead; k < a.hidden; k += 256) add(*reinterpret_cast<const uint4*>(wd + k), k);
    float v = 0.0f;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const float s = warp_sum(y[r]);
        if (lane == r) v = s;
    }
    if (lane < R && lane < a.rows) {
        if (a.b_down) v += to_f32(static_cast<const T*>(a.b_down)[d]);
        if (a.residual) v += to_f32(static_cast<const T*>(a.residual)[lane * a.rs + d]);
        static_cast<T*>(a.y)[lane * a.ys + d] = from_f32<T>(v);
    }
}

template <typename T, int R>
cudaError_t launch(const SmallArgs& a, cudaStream_t s) {
    cudaError_t e = launch_pdl(small_up_kernel<T, R>, dim3((a.hidden + kWarps - 1) / kWarps), dim3(kThreads), 0, s, a);
    if (e != cudaSuccess) return e;
    return launch_pdl(small_down_kernel<T, R>, dim3((a.dim + kWarps - 1) / kWarps), dim3(kThreads), 0, s, a);
}
template <typename T>
cudaError_t launch(const SmallArgs& a, cudaStream_t s) {
    if (a.rows == 1) return launch<T, 1>(a, s);
    if (a.rows == 2) return launch<T, 2>(a, s);
    if (a.rows <= 4) return launch<T, 4>(a, s);
    return launch<T, 8>(a, s);
}

}  // namespace

cudaError_t launch_gated_small(bool bf16, const SmallArgs& a, cudaStream_t s) {
    return bf16 ? launch<__nv_bfloat16>(a, s) : launch<__half>(a, s);
}

}  // namespace prism
