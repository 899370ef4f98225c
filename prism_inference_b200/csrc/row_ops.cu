// row_ops.cu - layer norm (forward, backward) and dropout with the residual add: the row-wise
// operators of the trainable sub-block  y = x + dropout(ffn(norm(x))).
#include <algorithm>
#include <type_traits>

#include "train_util.cuh"

namespace prism {
namespace {

// ---- rows in registers ---------------------------------------------------------------------
// A team of TEAM threads holds one row: thread t owns the NV groups of VEC consecutive columns that
// start at (j * TEAM + t) * VEC, VEC values = 16 bytes.  16 values a thread: with a whole warp on a
// 256-wide row the butterflies and the loop cost more instructions than the row's arithmetic (199
// against 94 us for 522,240 rows of fp16).
template <typename T>
struct Pack {
    static constexpr int N = 16 / sizeof(T);
    union {
        uint4 q;
        T v[N];
    };
    PRISM_DEV Pack() {}
};
template <typename T>
struct RowTensor {
    T* p;
    int64_t stride;
};

// first column of group j of thread t
template <typename T, int TEAM>
PRISM_DEV int col_of(int t, int j) { return (j * TEAM + t) * Pack<T>::N; }

// FAST kernels know that every row of every tensor starts on a 16-byte boundary and that dim is a
// multiple of a group.  The others take rows at any multiple of the type's size, m bytes past a
// 16-byte boundary: memory is still read and written in aligned 16-byte chunks, and a thread's group is
// cut out of its own chunk and the next thread's (a shuffle).  (Single-value accesses instead: 310
// against 137 us for 65,536 x 1001 fp16 forward.)
PRISM_DEV uint4 shift_down(const uint4& a, const uint4& b, uint32_t m) {  // bytes m .. m + 15 of a, b
    uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    if (m & 8) {
#pragma unroll
        for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
    }
    if (m & 4) {
#pragma unroll
        for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
    }
    const uint32_t bits = (m & 3) * 8;
    return make_uint4(__funnelshift_r(w[0], w[1], bits), __funnelshift_r(w[1], w[2], bits), __funnelshift_r(w[2], w[3], bits),
                      __funnelshift_r(w[3], w[4], bits));
}
// the chunk at `at`, of which only [lo, hi) is the tensor's memory
template <typename T>
PRISM_DEV uint4 load_chunk(const char* at, const char* lo, const char* hi) {
    Pack<T> p;
    if (at >= lo && at + 16 <= hi) {
        p.q = *reinterpret_cast<const uint4*>(at);
    } else {
#pragma unroll
        for (int e = 0; e < Pack<T>::N; ++e) {
            const char* v = at + e * sizeof(T);
            p.v[e] = v >= lo && v < hi ? *reinterpret_cast<const T*>(v) : from_f32<T>(0.0f);
        }
    }
    return p.q;
}
PRISM_DEV uint4 shfl_next(const uint4& v, int delta) {  // from the lane `delta` further
    return make_uint4(__shfl_sync(0xffffffffu, v.x, (threadIdx.x + delta) & 31), __shfl_sync(0xffffffffu, v.y, (threadIdx.x + delta) & 31),
                      __shfl_sync(0xffffffffu, v.z, (threadIdx.x + delta) & 31), __shfl_sync(0xffffffffu, v.w, (threadIdx.x + delta) & 31));
}

// Group j of this thread's row as loaded (`settle` turns it into values, so that loads can be in flight
// while the row before is worked on).
template <bool FAST>
struct Raw {
    uint4 own, next;
};
template <>
struct Raw<true> {
    uint4 own;
};
template <bool FAST, typename T, int TEAM>
PRISM_DEV Raw<FAST> load_group(const RowTensor<const T>& x, int64_t row, int64_t rows, int dim, int t, int j) {
    constexpr int VEC = Pack<T>::N, kSeg = TEAM < 32 ? TEAM : 32;  // threads whose chunks follow one another in a warp
    const int c = col_of<T, TEAM>(t, j);
    Raw<FAST> p;
    p.own = make_uint4(0, 0, 0, 0);
    const bool in = row < rows;
    const T* src = x.p + (in ? row : 0) * x.stride + c;
    if constexpr (FAST) {
        if (in && c < dim) p.own = *reinterpret_cast<const uint4*>(src);
    } else {
        const char *lo = reinterpret_cast<const char*>(x.p), *hi = reinterpret_cast<const char*>(x.p + (rows - 1) * x.stride + dim);
        const uint32_t m = (uint32_t)(uintptr_t)src & 15u;
        const char* at = reinterpret_cast<const char*>(src) - m;
        // this chunk holds columns from c - m / size on: wanted by this thread and the one before
        if (in && c < dim + VEC) p.own = load_chunk<T>(at, lo, hi);
        p.next = make_uint4(0, 0, 0, 0);
        if (t % kSeg == kSeg - 1 && in && m && c < dim) p.next = load_chunk<T>(at + 16, lo, hi);
    }
    return p;
}
// its values, zeros outside [0, rows) x [0, dim).  Whole warps (the shuffles).
template <bool FAST, typename T, int TEAM>
PRISM_DEV Pack<T> settle(const Raw<FAST>& raw, const RowTensor<const T>& x, int64_t row, int64_t rows, int dim, int t, int j) {
    constexpr int VEC = Pack<T>::N, kSeg = TEAM < 32 ? TEAM : 32;
    Pack<T> p;
    p.q = raw.own;
    if constexpr (!FAST) {
        const int c = col_of<T, TEAM>(t, j);
        const bool in = row < rows;
        const uint32_t m = (uint32_t)(uintptr_t)(x.p + (in ? row : 0) * x.stride + c) & 15u;
        uint4 next = shfl_next(p.q, 1);
        if (t % kSeg == kSeg - 1) next = raw.next;
        p.q = shift_down(p.q, next, m);
#pragma unroll
        for (int e = 0; e < VEC; ++e)
            if (!in || c + e >= dim) p.v[e] = from_f32<T>(0.0f);
    }
    return p;
}
template <bool FAST, typename T, int TEAM>
PRISM_DEV void store_group(const RowTensor<T>& y, int64_t row, int64_t rows, int dim, int t, int j, const Pack<T>& p) {
    constexpr int VEC = Pack<T>::N, kSeg = TEAM < 32 ? TEAM : 32;
    const int c = col_of<T, TEAM>(t, j);
    const bool in = row < rows;
    T* dst = y.p + (in ? row : 0) * y.stride + c;
    if (FAST) {
        if (in && c < dim) *reinterpret_cast<uint4*>(dst) = p.q;
        return;
    }
    // The aligned chunk at dst - m: the last m bytes of the group before and the first 16 - m of this
    // one.  Chunks that are not wholly of this row, or whose other group another warp has, go value by
    // value.
    const uint32_t m = (uint32_t)(uintptr_t)dst & 15u;
    const int n0 = (int)((16 - m) / sizeof(T)), s = t % kSeg;
    const uint4 before = shfl_next(p.q, -1);
    const bool mine = (m == 0 || s > 0) && c + n0 <= dim, later = s < kSeg - 1 && c + VEC + n0 <= dim;
    if (!in) return;
    if (mine) *reinterpret_cast<uint4*>(reinterpret_cast<char*>(dst) - m) = m ? shift_down(before, p.q, 16 - m) : p.q;
#pragma unroll
    for (int e = 0; e < VEC; ++e)
        if (c + e < dim && !(e < n0 ? mine : later)) dst[e] = p.v[e];
}
// a parameter vector's value: fp32, or the rows' type T
template <typename T>
PRISM_DEV float param_at(const void* w, int f32, int c) {
    return f32 ? static_cast<const float*>(w)[c] : to_f32(static_cast<const T*>(w)[c]);
}

// columns c .. c + VEC - 1 of a parameter vector, `none` where there is none
template <typename T>
PRISM_DEV void load_params(const void* w, int f32, int c, int dim, float none, float* out) {
    constexpr int VEC = Pack<T>::N;
    if (w && c + VEC <= dim && (uintptr_t)w % 16 == 0) {
        if (f32) {
#pragma unroll
            for (int e = 0; e < VEC; e += 4) {
                const float4 v = *reinterpret_cast<const float4*>(static_cast<const float*>(w) + c + e);
                out[e] = v.x, out[e + 1] = v.y, out[e + 2] = v.z, out[e + 3] = v.w;
            }
        } else {
            Pack<T> p;
            p.q = *reinterpret_cast<const uint4*>(static_cast<const T*>(w) + c);
#pragma unroll
            for (int e = 0; e < VEC; ++e) out[e] = to_f32(p.v[e]);
        }
    } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) out[e] = w && c + e < dim ? param_at<T>(w, f32, c + e) : none;
    }
}

// Sums over a team.  Teams of up to a warp: butterfly, every lane gets the same bits.  Larger teams:
// butterfly, then the warps' sums in order from shared memory, between barriers of the team's own.
template <int TEAM, int N>
PRISM_DEV void team_sum(float (&a)[N], float2* red) {
    constexpr int kW = TEAM < 32 ? TEAM : 32;
#pragma unroll
    for (int o = kW / 2; o > 0; o >>= 1) {
#pragma unroll
        for (int i = 0; i < N; ++i) a[i] += __shfl_xor_sync(0xffffffffu, a[i], o);
    }
    if (TEAM > 32) {
        const int first = (threadIdx.x / TEAM) * (TEAM / 32), bar = 1 + threadIdx.x / TEAM;
        named_bar_sync(bar, TEAM);  // the sums of the call before have been read
        if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = make_float2(a[0], a[N - 1]);
        named_bar_sync(bar, TEAM);
        a[0] = a[N - 1] = 0.0f;
#pragma unroll
        for (int w = 0; w < TEAM / 32; ++w) {
            const float2 v = red[first + w];
            a[0] += v.x;
            if (N > 1) a[N - 1] += v.y;
        }
    }
}

struct NormArgs {
    const void *x, *weight, *bias;
    void* y;
    float *mean, *rstd;
    int64_t rows, xs, ys;
    int dim, param_f32;
    float eps;
};
struct NormBackArgs {
    const void *x, *weight, *dy, *add;
    const float *mean, *rstd;
    void* dx;
    float* part;  // [gridDim.x][2][dim] partial dweight, dbias (NULL: neither is wanted)
    int64_t rows, xs, dys, adds, dxs;
    int dim, param_f32;
};

constexpr int kThreads = 256, kWarps = kThreads / 32;

// the first row of this warp, and this lane's row
template <int TEAM>
PRISM_DEV int64_t warp_row() {
    constexpr int kTeams = kThreads / TEAM;
    return (int64_t)blockIdx.x * kTeams + (TEAM < 32 ? (threadIdx.x / 32) * (32 / TEAM) : threadIdx.x / TEAM);
}

// y = (x - mean) rstd w + b.  One pass over memory: the row stays in registers between the mean,
// the centred second moment and the output.  Memory-bound: 2 R D s bytes.  The next row's loads
// are issued before this row's sums, so each team keeps two rows in flight.
template <bool FAST, typename T, int TEAM, int NV>
__global__ void __launch_bounds__(kThreads, FAST && NV * Pack<T>::N <= 16 ? 3 : 1) norm_kernel(const NormArgs a) {
    constexpr int VEC = Pack<T>::N, kN = VEC * NV, kTeams = kThreads / TEAM;
    constexpr bool kHold = kN <= 16;  // weight and bias stay in registers across rows
    __shared__ float2 red[kWarps];
    const int t = threadIdx.x % TEAM;
    const int64_t step = (int64_t)gridDim.x * kTeams;
    const RowTensor<const T> x{static_cast<const T*>(a.x), a.xs};
    const RowTensor<T> y{static_cast<T*>(a.y), a.ys};
    const float inv = 1.0f / (float)a.dim;
    Raw<FAST> nxt[NV];
    // every lane of a warp walks the same number of rows (the shuffles need the whole warp); teams
    // past the last row work on zeros and store nothing
    int64_t row0 = warp_row<TEAM>();
    const int team = TEAM < 32 ? (threadIdx.x & 31) / TEAM : 0;
#pragma unroll
    for (int j = 0; j < NV; ++j) nxt[j] = load_group<FAST, T, TEAM>(x, row0 + team, a.rows, a.dim, t, j);
    float w[kHold ? kN : VEC], b[kHold ? kN : VEC];
    if (kHold) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            load_params<T>(a.weight, a.param_f32, col_of<T, TEAM>(t, j), a.dim, 1.0f, w + j * VEC);
            load_params<T>(a.bias, a.param_f32, col_of<T, TEAM>(t, j), a.dim, 0.0f, b + j * VEC);
        }
    }
    for (; row0 < a.rows; row0 += step) {
        Pack<T> cur[NV];
#pragma unroll
        for (int j = 0; j < NV; ++j) cur[j] = settle<FAST, T, TEAM>(nxt[j], x, row0 + team, a.rows, a.dim, t, j);
        if (row0 + step < a.rows) {
#pragma unroll
            for (int j = 0; j < NV; ++j) nxt[j] = load_group<FAST, T, TEAM>(x, row0 + step + team, a.rows, a.dim, t, j);
        }
        float v[kN], s[1] = {0.0f};
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            v[i] = to_f32(cur[i / VEC].v[i % VEC]);
            s[0] += v[i];
        }
        team_sum<TEAM>(s, red);
        const float mean = s[0] * inv;
        s[0] = 0.0f;
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            v[i] -= mean;
            const int c = (i / VEC * TEAM + t) * VEC + (FAST ? 0 : i % VEC);
            if (c < a.dim) s[0] = fmaf(v[i], v[i], s[0]);
        }
        team_sum<TEAM>(s, red);
        const float rstd = rsqrtf(fmaf(s[0], inv, a.eps));
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            if (!kHold) {
                load_params<T>(a.weight, a.param_f32, col_of<T, TEAM>(t, j), a.dim, 1.0f, w);
                load_params<T>(a.bias, a.param_f32, col_of<T, TEAM>(t, j), a.dim, 0.0f, b);
            }
            Pack<T> o;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const int i = j * VEC + e, k = kHold ? i : e;
                o.v[e] = from_f32<T>(fmaf(v[i] * rstd, w[k], b[k]));
            }
            store_group<FAST, T, TEAM>(y, row0 + team, a.rows, a.dim, t, j, o);
        }
        if (t == 0 && row0 + team < a.rows) {
            if (a.mean) a.mean[row0 + team] = mean;
            if (a.rstd) a.rstd[row0 + team] = rstd;
        }
    }
}

// With xh = (x - mean) rstd and g = dy w:
//   dx = rstd (g - mean_c(g) - xh mean_c(g xh)) [+ add],  dweight = sum_r dy xh,  dbias = sum_r dy.
// One pass over x and dy: each thread keeps its columns' dweight and dbias sums over all the rows
// its team walks, the CTA's warps are added in order, and norm_fold_kernel adds the CTAs' partial
// sums in order (no atomics: the same inputs give the same bits).
// the registers that two CTAs an SM leave each thread hold 16 16-bit values' sums and loads, no more
template <bool FAST, typename T, int NV>
__host__ __device__ constexpr int back_ctas_per_sm() {
    return FAST && sizeof(T) == 2 && NV * Pack<T>::N <= 16 ? 2 : 1;
}
template <bool FAST, typename T, int TEAM, int NV>
__global__ void __launch_bounds__(kThreads, back_ctas_per_sm<FAST, T, NV>()) norm_back_kernel(const NormBackArgs a) {
    constexpr int VEC = Pack<T>::N, kN = VEC * NV, kTeams = kThreads / TEAM;
    constexpr bool kHold = kN <= 16;
    constexpr int kParts = TEAM < 32 ? kWarps : kTeams;  // sums of whole columns in a CTA: warps or teams
    extern __shared__ float fold[];  // [kParts][2][dim], teams smaller than the CTA
    __shared__ float2 red[kWarps];
    const int t = threadIdx.x % TEAM, team = TEAM < 32 ? (threadIdx.x & 31) / TEAM : 0;
    const int64_t step = (int64_t)gridDim.x * kTeams;
    const RowTensor<const T> x{static_cast<const T*>(a.x), a.xs}, dy{static_cast<const T*>(a.dy), a.dys},
        add{static_cast<const T*>(a.add), a.adds};
    const RowTensor<T> dx{static_cast<T*>(a.dx), a.dxs};
    const float inv = 1.0f / (float)a.dim;
    float dw[kN], db[kN];
#pragma unroll
    for (int i = 0; i < kN; ++i) dw[i] = db[i] = 0.0f;
    int64_t row0 = warp_row<TEAM>();
    // the next row's loads are in flight during this row's sums and its store
    Raw<FAST> nx[NV], ng[NV], na[NV];
    float mean = 0.0f, rstd = 0.0f;
    auto load = [&](int64_t r0) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            nx[j] = load_group<FAST, T, TEAM>(x, r0 + team, a.rows, a.dim, t, j);
            ng[j] = load_group<FAST, T, TEAM>(dy, r0 + team, a.rows, a.dim, t, j);
            if (add.p) na[j] = load_group<FAST, T, TEAM>(add, r0 + team, a.rows, a.dim, t, j);
        }
        const bool in = r0 + team < a.rows;
        mean = in ? a.mean[r0 + team] : 0.0f;
        rstd = in ? a.rstd[r0 + team] : 0.0f;
    };
    load(row0);
    float w[kHold ? kN : VEC];
    if (kHold) {
#pragma unroll
        for (int j = 0; j < NV; ++j) load_params<T>(a.weight, a.param_f32, col_of<T, TEAM>(t, j), a.dim, 1.0f, w + j * VEC);
    }
    for (; row0 < a.rows; row0 += step) {
        const float m = mean, r = rstd;
        float s[2] = {0.0f, 0.0f};
        // columns past the row hold zeros, whose xh is not zero: they take no part (as rows past the last)
        const int lim = row0 + team < a.rows ? a.dim : 0;
        Pack<T> px[NV], pg[NV], pa[NV];
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            px[j] = settle<FAST, T, TEAM>(nx[j], x, row0 + team, a.rows, a.dim, t, j);
            pg[j] = settle<FAST, T, TEAM>(ng[j], dy, row0 + team, a.rows, a.dim, t, j);
            if (add.p) pa[j] = settle<FAST, T, TEAM>(na[j], add, row0 + team, a.rows, a.dim, t, j);
        }
        if (row0 + step < a.rows) load(row0 + step);
        // dy and x stay as loaded: g and xh are worked out again after the sums, which costs less than
        // the registers to keep them
        auto value = [&](int i, float& d, float& g, float& xh) {
            const int c = (i / VEC * TEAM + t) * VEC + (FAST ? 0 : i % VEC);
            d = to_f32(pg[i / VEC].v[i % VEC]);
            xh = c < lim ? (to_f32(px[i / VEC].v[i % VEC]) - m) * r : 0.0f;
            g = d * w[kHold ? i : i % VEC];
        };
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            if (!kHold && i % VEC == 0) load_params<T>(a.weight, a.param_f32, col_of<T, TEAM>(t, i / VEC), a.dim, 1.0f, w);
            float d, g, xh;
            value(i, d, g, xh);
            dw[i] = fmaf(d, xh, dw[i]);
            db[i] += d;
            s[0] += g;
            s[1] = fmaf(g, xh, s[1]);
        }
        team_sum<TEAM>(s, red);
        const float m0 = s[0] * inv, m1 = s[1] * inv;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            if (!kHold) load_params<T>(a.weight, a.param_f32, col_of<T, TEAM>(t, j), a.dim, 1.0f, w);
            Pack<T> o;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                float d, g, xh;
                value(j * VEC + e, d, g, xh);
                d = r * (g - m0 - xh * m1);
                if (add.p) d += to_f32(pa[j].v[e]);
                o.v[e] = from_f32<T>(d);
            }
            store_group<FAST, T, TEAM>(dx, row0 + team, a.rows, a.dim, t, j, o);
        }
    }
    if (!a.part) return;
    float* out = a.part + (int64_t)blockIdx.x * 2 * a.dim;
    if (TEAM < kThreads) {
        if (TEAM < 32) {  // a warp's teams by butterfly
#pragma unroll
            for (int i = 0; i < kN; ++i) {
#pragma unroll
                for (int o = TEAM; o < 32; o <<= 1) {
                    dw[i] += __shfl_xor_sync(0xffffffffu, dw[i], o);
                    db[i] += __shfl_xor_sync(0xffffffffu, db[i], o);
                }
            }
        }
        float* mine = fold + (threadIdx.x / (TEAM < 32 ? 32 : TEAM)) * 2 * a.dim;
        if (TEAM >= 32 || (threadIdx.x & 31) < TEAM) {
#pragma unroll
            for (int i = 0; i < kN; ++i) {
                const int c = (i / VEC * TEAM + t) * VEC + i % VEC;
                if (c < a.dim) {
                    mine[c] = dw[i];
                    mine[a.dim + c] = db[i];
                }
            }
        }
        __syncthreads();
        for (int c = threadIdx.x; c < 2 * a.dim; c += kThreads) {
            float s = 0.0f;
#pragma unroll
            for (int k = 0; k < kParts; ++k) s += fold[k * 2 * a.dim + c];
            out[c] = s;
        }
    } else {
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            const int c = (i / VEC * TEAM + t) * VEC + i % VEC;
            if (c < a.dim) {
                out[c] = dw[i];
                out[a.dim + c] = db[i];
            }
        }
    }
}

// Adds the CTAs' partial sums: 32 columns a CTA, 32 threads a column over every 32nd partial, then the
// 32 in order.  In 64 bits: in 32 these last additions, of nearly whole sums, made up more than half of the
// squared error (4,099 x 1,001 fp32, root mean square over the columns: 1.4e-7 against 7.2e-8), and the kernel
// waits for its loads anyway.
template <typename T>
__global__ void __launch_bounds__(1024)
    norm_fold_kernel(const float* part, int n_part, int dim, void* dweight, void* dbias, int param_f32) {
    __shared__ double red[32][33];
    grid_dep_wait();
    const int lane = threadIdx.x & 31, k = threadIdx.x >> 5;
    const int c = blockIdx.x * 32 + lane;  // over [dweight | dbias]
    double s = 0.0;
    if (c < 2 * dim)
        for (int p = k; p < n_part; p += 32) s += part[(int64_t)p * 2 * dim + c];
    red[k][lane] = s;
    __syncthreads();
    if (k == 0 && c < 2 * dim) {
        s = 0.0;
#pragma unroll
        for (int i = 0; i < 32; ++i) s += red[i][lane];
        void* dst = c < dim ? dweight : dbias;
        const int i = c < dim ? c : c - dim;
        if (dst) {
            if (param_f32)
                static_cast<float*>(dst)[i] = (float)s;
            else
                static_cast<T*>(dst)[i] = from_f32<T>((float)s);
        }
    }
}

// ---- dropout ---------------------------------------------------------------------------------
// Philox4x32-10 (Salmon, Moraes, Dror, Shaw: Parallel random numbers, as easy as 1, 2, 3; 2011).
// The key of every round, worked out once a thread: a third of the generator's instructions otherwise.
struct PhiloxKeys {
    uint32_t x[10], y[10];
    PRISM_DEV explicit PhiloxKeys(uint64_t seed) {
#pragma unroll
        for (int r = 0; r < 10; ++r) {
            x[r] = (uint32_t)seed + r * 0x9E3779B9u;
            y[r] = (uint32_t)(seed >> 32) + r * 0xBB67AE85u;
        }
    }
};
PRISM_DEV uint4 philox(uint64_t block, uint64_t offset, const PhiloxKeys& k) {
    uint4 c = make_uint4((uint32_t)block, (uint32_t)(block >> 32), (uint32_t)offset, (uint32_t)(offset >> 32));
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t p0 = (uint64_t)0xD2511F53u * c.x, p1 = (uint64_t)0xCD9E8D57u * c.z;
        c = make_uint4((uint32_t)(p1 >> 32) ^ c.y ^ k.x[r], (uint32_t)p1, (uint32_t)(p0 >> 32) ^ c.w ^ k.y[r], (uint32_t)p0);
    }
    return c;
}
// element i of a block: kept iff its 16 bits are >= t / 65536.  What it holds when dropped does not matter
// (an infinity or NaN goes too), so a choice, not a product with 0.
PRISM_DEV float drop(uint32_t word, int i, uint32_t t16, float x, float scale, float res) {
    const bool keep = (i & 1 ? word : word << 16) >= t16;  // t16: threshold << 16
    return keep ? fmaf(x, scale, res) : res;
}

struct DropArgs {
    const void *x, *residual;
    void* y;
    const uint64_t* rng;  // {seed, offset}
    int64_t rows, xs, rs, ys;
    int dim;
    uint32_t threshold;  // of 65536: an element is kept iff its 16 bits are >= threshold
    float scale;
};

// y = residual + (kept ? x scale : 0).  Element i = row * dim + column takes bits 16 (i % 8) .. of
// the Philox block with counter (i / 8, offset) and key seed, so the mask depends on neither
// strides nor launch shape, and the gradient's call draws it again instead of reading it.
// 16 bits an element: with 32 the ten rounds (some 80 instructions a block) would cost as much
// time as the memory traffic.  One thread does UNR blocks of 8 elements, loads first.
// Contiguous tensors are one long row (dim = total); VEC needs 16-byte aligned groups of 8.
template <typename T, bool VEC8, bool FLAT>
__global__ void __launch_bounds__(kThreads) dropout_kernel(const DropArgs a) {
    const uint64_t seed = a.rng[0], offset = a.rng[1];
    const PhiloxKeys keys(seed);
    const uint32_t t16 = a.threshold << 16;
    const int64_t n = a.rows * a.dim, blocks = (n + 7) / 8, stride = (int64_t)gridDim.x * kThreads;
    const T *x = static_cast<const T*>(a.x), *res = static_cast<const T*>(a.residual);
    T* y = static_cast<T*>(a.y);
    constexpr int UNR = 2, E = 16 / sizeof(T);
    for (int64_t b0 = (int64_t)blockIdx.x * kThreads + threadIdx.x; b0 < blocks; b0 += UNR * stride) {
        if (VEC8) {
            Pack<T> px[UNR][8 / E], pr[UNR][8 / E];
            int64_t yo[UNR];
            bool full[UNR];
#pragma unroll
            for (int u = 0; u < UNR; ++u) {
                const int64_t b = b0 + u * stride;
                full[u] = b * 8 + 8 <= n;
                if (!full[u]) continue;
                int64_t r = 0, c = b * 8;
                if (!FLAT) {
                    const uint32_t per = (uint32_t)a.dim / 8;
                    r = (blocks >> 32) ? b / per : (int64_t)((uint32_t)b / per);
                    c = (b - r * per) * 8;
                }
                yo[u] = r * a.ys + c;
#pragma unroll
                for (int q = 0; q < 8 / E; ++q) {
                    px[u][q].q = *reinterpret_cast<const uint4*>(x + r * a.xs + c + q * E);
                    if (res) pr[u][q].q = *reinterpret_cast<const uint4*>(res + r * a.rs + c + q * E);
                }
            }
#pragma unroll
            for (int u = 0; u < UNR; ++u) {
                const int64_t b = b0 + u * stride;
                if (b >= blocks) continue;
                const uint4 w = philox(b, offset, keys);
                const uint32_t bits[4] = {w.x, w.y, w.z, w.w};
                if (full[u]) {
#pragma unroll
                    for (int q = 0; q < 8 / E; ++q) {
                        Pack<T> o;
#pragma unroll
                        for (int e = 0; e < E; ++e) {
                            const int i = q * E + e;
                            o.v[e] = from_f32<T>(drop(bits[i >> 1], i, t16, to_f32(px[u][q].v[e]), a.scale, res ? to_f32(pr[u][q].v[e]) : 0.0f));
                        }
                        *reinterpret_cast<uint4*>(y + yo[u] + q * E) = o.q;
                    }
                } else {  // the last block of a flat tensor (rows of a strided one are multiples of 8)
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int64_t at = b * 8 + i;
                        if (at < n) y[at] = from_f32<T>(drop(bits[i >> 1], i, t16, to_f32(x[at]), a.scale, res ? to_f32(res[at]) : 0.0f));
                    }
                }
            }
        } else {
#pragma unroll 1
            for (int u = 0; u < UNR; ++u) {
                const int64_t b = b0 + u * stride;
                if (b >= blocks) break;
                const uint4 w = philox(b, offset, keys);
                const uint32_t bits[4] = {w.x, w.y, w.z, w.w};
                int64_t r = (b * 8) / a.dim;
                int c = (int)(b * 8 - r * a.dim);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    if (r < a.rows)
                        y[r * a.ys + c] = from_f32<T>(drop(bits[i >> 1], i, t16, to_f32(x[r * a.xs + c]), a.scale, res ? to_f32(res[r * a.rs + c]) : 0.0f));
                    if (++c == a.dim) {
                        c = 0;
                        ++r;
                    }
                }
            }
        }
    }
}

// ---- host --------------------------------------------------------------------------------------

#define fail prism::set_error

constexpr int kNormMaxDim = 16384;
constexpr int kBackCtasPerSm = 2;  // at most: sizes the workspace

// What a row's threads hold, by type and width: f(FAST, TEAM, NV) as constants.  16 values a thread up to
// the width of a CTA's 256 threads (with a warp and 32 values on 1000-wide rows, backward: 208 against
// 108 us for 65,536 rows of fp16, for want of warps), then more.
template <typename T, typename F>
int with_shape(bool fast, int dim, F&& f) {
    constexpr int V = Pack<T>::N, NV = 16 / V;
    using std::integral_constant;
#define SHAPE(TEAM, GROUPS)                                                                        \
    return fast ? f(std::true_type{}, integral_constant<int, TEAM>{}, integral_constant<int, GROUPS>{}) \
                : f(std::false_type{}, integral_constant<int, TEAM>{}, integral_constant<int, GROUPS>{})
    if (dim <= 64) SHAPE(4, NV);
    if (dim <= 128) SHAPE(8, NV);
    if (dim <= 256) SHAPE(16, NV);
    if (dim <= 512) SHAPE(32, NV);
    if (dim <= 1024) SHAPE(64, NV);
    if (dim <= 2048) SHAPE(128, NV);
    if (dim <= 4096) SHAPE(256, NV);
    if (dim <= 8192) SHAPE(256, 2 * NV);
    SHAPE(256, 4 * NV);
#undef SHAPE
}

template <typename F>
int with_type(int dtype, F&& f) {
    if (dtype == PRISM_DTYPE_F16) return f(__half{});
    if (dtype == PRISM_DTYPE_BF16) return f(__nv_bfloat16{});
    return f(float{});
}

// base and row pitch multiples of 16 bytes
bool vec_ok(const void* p, int64_t stride, int64_t es) {
    return !p || (((uintptr_t)p & 15) == 0 && (stride * es) % 16 == 0);
}

int check_norm(const char* who, const prism_norm_params* p) {
    if (!dtype_known(p->dtype) || (p->param_dtype != p->dtype && p->param_dtype != PRISM_DTYPE_F32))
        return fail(PRISM_E_ARG, "%s: dtype %d / param_dtype %d (the parameters are the rows' type or fp32)", who, p->dtype,
                    p->param_dtype);
    if (p->rows < 0 || p->dim <= 0) return fail(PRISM_E_ARG, "%s: rows %lld, dim %d", who, (long long)p->rows, p->dim);
    if (p->dim > kNormMaxDim) return fail(PRISM_E_UNSUPPORTED, "%s: dim %d above %d", who, p->dim, kNormMaxDim);
    return PRISM_OK;
}
int check_param(const char* who, const char* name, const void* t, int dtype) {
    return t && (uintptr_t)t % dtype_bytes(dtype) ? fail(PRISM_E_ALIGN, "%s: %s is not aligned to its type", who, name) : PRISM_OK;
}
int check_stride(const char* who, const char* name, const void* t, int64_t stride, int64_t rows, int dim, int es) {
    if (!t) return PRISM_OK;
    if ((uintptr_t)t % es) return fail(PRISM_E_ALIGN, "%s: %s is not aligned to its type", who, name);
    if (rows > 1 && stride < dim)
        return fail(PRISM_E_ARG, "%s: %s_stride %lld below dim %d", who, name, (long long)stride, dim);
    if (rows > (int64_t)1 << 40) return fail(PRISM_E_RANGE, "%s: rows %lld", who, (long long)rows);
    if (rows > 1 && (stride > (int64_t)1 << 40 || !extent_ok(rows, stride)))
        return fail(PRISM_E_RANGE, "%s: %s_stride %lld", who, name, (long long)stride);
    return PRISM_OK;
}
// outputs may be an input itself (same address and stride), never share bytes with it otherwise
bool bad_alias(const void* out, int64_t so, const void* in, int64_t si, int64_t rows, int64_t dim, int64_t es) {
    if (rows <= 1) so = si = dim;
    if (out == in && so == si) return false;
    return rows_overlap(out, so, in, si, rows, dim, es);
}

// CTAs of the backward kernel: one partial sum each
int back_ctas(const prism_ctx* ctx, int64_t rows, int teams, int per_sm) {
    return (int)std::min<int64_t>((rows + teams - 1) / teams, (int64_t)ctx->sm_count * per_sm);
}

}  // namespace
}  // namespace prism

using namespace prism;

extern "C" int prism_layer_norm(prism_ctx* ctx, const prism_norm_params* p, const void* x, const void* weight,
                                const void* bias, void* y, float* mean, float* rstd, void* stream) {
    if (!ctx || !p) return fail(PRISM_E_ARG, "prism_layer_norm: NULL argument");
    int rc = check_norm("prism_layer_norm", p);
    if (rc) return rc;
    if (p->rows == 0) return PRISM_OK;
    if (!x || !y) return fail(PRISM_E_ARG, "prism_layer_norm: NULL argument");
    const int es = dtype_bytes(p->dtype);
    if ((rc = check_stride("prism_layer_norm", "x", x, p->x_stride, p->rows, p->dim, es)) ||
        (rc = check_stride("prism_layer_norm", "y", y, p->y_stride, p->rows, p->dim, es)) ||
        (rc = check_param("prism_layer_norm", "weight", weight, p->param_dtype)) ||
        (rc = check_param("prism_layer_norm", "bias", bias, p->param_dtype)) ||
        (rc = check_param("prism_layer_norm", "mean", mean, PRISM_DTYPE_F32)) ||
        (rc = check_param("prism_layer_norm", "rstd", rstd, PRISM_DTYPE_F32)))
        return rc;
    if (bad_alias(y, p->y_stride, x, p->x_stride, p->rows, p->dim, es))
        return fail(PRISM_E_ARG, "prism_layer_norm: y overlaps x");
    if (bytes_overlap(mean, (size_t)p->rows * 4, rstd, (size_t)p->rows * 4))
        return fail(PRISM_E_ARG, "prism_layer_norm: mean and rstd overlap");
    DeviceGuard g(ctx->device);
    const int64_t xs = p->rows > 1 ? p->x_stride : p->dim, ys = p->rows > 1 ? p->y_stride : p->dim;
    NormArgs a{x, weight, bias, y, mean, rstd, p->rows, xs, ys, p->dim,
               p->param_dtype == PRISM_DTYPE_F32, p->eps};
    return with_type(p->dtype, [&](auto tag) {
        using T = decltype(tag);
        const bool fast = p->dim % Pack<T>::N == 0 && vec_ok(x, xs, es) && vec_ok(y, ys, es);
        return with_shape<T>(fast, p->dim, [&](auto quick, auto team, auto nv) {
            constexpr int kTeams = kThreads / decltype(team)::value;
            const int64_t want = (p->rows + kTeams - 1) / kTeams;
            const int grid = (int)std::min<int64_t>(want, (int64_t)ctx->sm_count * 3);
            norm_kernel<decltype(quick)::value, T, decltype(team)::value, decltype(nv)::value>
                <<<grid, kThreads, 0, as_stream(stream)>>>(a);
            return cuda_rc(cudaGetLastError(), "prism_layer_norm");
        });
    });
}

extern "C" int prism_layer_norm_backward_workspace(prism_ctx* ctx, const prism_norm_params* p, size_t* bytes) {
    if (!ctx || !p || !bytes) return fail(PRISM_E_ARG, "prism_layer_norm_backward_workspace: NULL argument");
    int rc = check_norm("prism_layer_norm_backward_workspace", p);
    if (rc) return rc;
    // one partial [2][dim] in fp32 a CTA, for any team size
    *bytes = (size_t)std::min<int64_t>(p->rows, (int64_t)ctx->sm_count * kBackCtasPerSm) * 2 * p->dim * 4;
    return PRISM_OK;
}

extern "C" int prism_layer_norm_backward(prism_ctx* ctx, const prism_norm_params* p, const void* x, const void* weight,
                                         const float* mean, const float* rstd, const void* dy, const void* add, void* dx,
                                         void* dweight, void* dbias, void* workspace, size_t workspace_bytes,
                                         void* stream) {
    const char* who = "prism_layer_norm_backward";
    if (!ctx || !p) return fail(PRISM_E_ARG, "%s: NULL argument", who);
    int rc = check_norm(who, p);
    if (rc) return rc;
    if ((rc = check_param(who, "weight", weight, p->param_dtype)) || (rc = check_param(who, "dweight", dweight, p->param_dtype)) ||
        (rc = check_param(who, "dbias", dbias, p->param_dtype)) || (rc = check_param(who, "mean", mean, PRISM_DTYPE_F32)) ||
        (rc = check_param(who, "rstd", rstd, PRISM_DTYPE_F32)))
        return rc;
    const size_t n = (size_t)p->dim * dtype_bytes(p->param_dtype);
    if (bytes_overlap(dweight, n, dbias, n)) return fail(PRISM_E_ARG, "%s: dweight and dbias overlap", who);
    DeviceGuard g(ctx->device);
    if (p->rows == 0) {  // no rows: the sums are zero
        if (dweight && (rc = cuda_rc(cudaMemsetAsync(dweight, 0, n, as_stream(stream)), who))) return rc;
        if (dbias && (rc = cuda_rc(cudaMemsetAsync(dbias, 0, n, as_stream(stream)), who))) return rc;
        return PRISM_OK;
    }
    if (!x || !mean || !rstd || !dy || !dx) return fail(PRISM_E_ARG, "%s: NULL argument", who);
    const int es = dtype_bytes(p->dtype);
    if ((rc = check_stride(who, "x", x, p->x_stride, p->rows, p->dim, es)) ||
        (rc = check_stride(who, "dy", dy, p->dy_stride, p->rows, p->dim, es)) ||
        (rc = check_stride(who, "add", add, p->add_stride, p->rows, p->dim, es)) ||
        (rc = check_stride(who, "dx", dx, p->dx_stride, p->rows, p->dim, es)))
        return rc;
    if (bad_alias(dx, p->dx_stride, x, p->x_stride, p->rows, p->dim, es) ||
        bad_alias(dx, p->dx_stride, dy, p->dy_stride, p->rows, p->dim, es) ||
        bad_alias(dx, p->dx_stride, add, p->add_stride, p->rows, p->dim, es))
        return fail(PRISM_E_ARG, "%s: dx overlaps an input", who);
    const bool sums = dweight || dbias;
    size_t need = 0;
    prism_layer_norm_backward_workspace(ctx, p, &need);
    if (sums && (!workspace || workspace_bytes < need))
        return fail(PRISM_E_ARG, "%s: workspace of %zu bytes, %zu needed", who, workspace ? workspace_bytes : (size_t)0, need);
    if (sums && ((uintptr_t)workspace & 15)) return fail(PRISM_E_ALIGN, "%s: workspace is not 16-byte aligned", who);
    const auto of = [&](int64_t stride) { return p->rows > 1 ? stride : (int64_t)p->dim; };
    NormBackArgs a{x,  weight, dy, add, mean, rstd, dx, sums ? static_cast<float*>(workspace) : nullptr,
                   p->rows, of(p->x_stride), of(p->dy_stride), of(p->add_stride), of(p->dx_stride), p->dim,
                   p->param_dtype == PRISM_DTYPE_F32};
    return with_type(p->dtype, [&](auto tag) {
        using T = decltype(tag);
        int grid = 0;
        const bool fast = p->dim % Pack<T>::N == 0 && vec_ok(x, a.xs, es) && vec_ok(dy, a.dys, es) && vec_ok(add, a.adds, es) && vec_ok(dx, a.dxs, es);
        int rc = with_shape<T>(fast, p->dim, [&](auto quick, auto team, auto nv) {
            constexpr int kTeam = decltype(team)::value;
            auto kernel = norm_back_kernel<decltype(quick)::value, T, kTeam, decltype(nv)::value>;
            grid = back_ctas(ctx, p->rows, kThreads / kTeam, back_ctas_per_sm<decltype(quick)::value, T, decltype(nv)::value>());
            // at most 32 KB: a team's width grows with dim
            const size_t smem = sums && kTeam < kThreads ? (size_t)(kTeam < 32 ? kWarps : kThreads / kTeam) * p->dim * 8 : 0;
            kernel<<<grid, kThreads, smem, as_stream(stream)>>>(a);
            return cuda_rc(cudaGetLastError(), who);
        });
        if (rc || !sums) return rc;
        return cuda_rc(launch_pdl(norm_fold_kernel<T>, dim3((2 * p->dim + 31) / 32), dim3(1024), 0, as_stream(stream),
                                  (const float*)workspace, grid, p->dim, dweight, dbias,
                                  (int)(p->param_dtype == PRISM_DTYPE_F32)),
                       who);
    });
}

extern "C" int prism_dropout_add(prism_ctx* ctx, const prism_dropout_params* p, const void* x, const void* residual,
                                 const uint64_t* rng, void* y, void* stream) {
    const char* who = "prism_dropout_add";
    if (!ctx || !p) return fail(PRISM_E_ARG, "%s: NULL argument", who);
    if (!dtype_known(p->dtype)) return fail(PRISM_E_ARG, "%s: dtype %d", who, p->dtype);
    if (p->rows < 0 || p->dim <= 0) return fail(PRISM_E_ARG, "%s: rows %lld, dim %d", who, (long long)p->rows, p->dim);
    if (p->threshold < 0 || p->threshold > 65535)
        return fail(PRISM_E_ARG, "%s: threshold %d (of 65536; 65536 would drop everything)", who, p->threshold);
    if (p->rows == 0) return PRISM_OK;
    if (!x || !rng || !y) return fail(PRISM_E_ARG, "%s: NULL argument", who);
    if ((uintptr_t)rng % 8) return fail(PRISM_E_ALIGN, "%s: rng is not 8-byte aligned", who);
    const int es = dtype_bytes(p->dtype);
    int rc;
    if ((rc = check_stride(who, "x", x, p->x_stride, p->rows, p->dim, es)) ||
        (rc = check_stride(who, "residual", residual, p->residual_stride, p->rows, p->dim, es)) ||
        (rc = check_stride(who, "y", y, p->y_stride, p->rows, p->dim, es)))
        return rc;
    if (p->rows > ((int64_t)1 << 62) / p->dim) return fail(PRISM_E_RANGE, "%s: rows %lld x dim %d", who, (long long)p->rows, p->dim);
    if (bad_alias(y, p->y_stride, x, p->x_stride, p->rows, p->dim, es) ||
        bad_alias(y, p->y_stride, residual, p->residual_stride, p->rows, p->dim, es))
        return fail(PRISM_E_ARG, "%s: y overlaps an input", who);
    DeviceGuard g(ctx->device);
    DropArgs a{x, residual, y, rng, p->rows, p->x_stride, p->residual_stride, p->y_stride, p->dim, (uint32_t)p->threshold,
               65536.0f / (float)(65536 - p->threshold)};
    const bool flat = p->rows == 1 || (p->x_stride == p->dim && p->y_stride == p->dim && (!residual || p->residual_stride == p->dim));
    const bool vec = flat ? vec_ok(x, 0, es) && vec_ok(y, 0, es) && vec_ok(residual, 0, es)
                          : p->dim % 8 == 0 && vec_ok(x, p->x_stride, es) && vec_ok(y, p->y_stride, es) &&
                                vec_ok(residual, p->residual_stride, es);
    const int64_t blocks = (p->rows * p->dim + 7) / 8;
    const int grid = (int)std::min<int64_t>((blocks + kThreads - 1) / kThreads, (int64_t)ctx->sm_count * 8);
    return with_type(p->dtype, [&](auto tag) {
        using T = decltype(tag);
        if (vec && flat)
            dropout_kernel<T, true, true><<<grid, kThreads, 0, as_stream(stream)>>>(a);
        else if (vec)
            dropout_kernel<T, true, false><<<grid, kThreads, 0, as_stream(stream)>>>(a);
        else
            dropout_kernel<T, false, false><<<grid, kThreads, 0, as_stream(stream)>>>(a);
        return cuda_rc(cudaGetLastError(), who);
    });
}
