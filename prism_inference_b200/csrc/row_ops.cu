// row_ops.cu - layer norm (forward, backward) and dropout with the residual add: the row-wise
// operators of the trainable sub-block  y = x + dropout(ffn(norm(x))).
#include <algorithm>
#include <type_traits>

#include "train_util.cuh"

namespace prism {
namespace {

// ---- rows in registers ---------------------------------------------------------------------
// A team of TEAM threads holds one row: thread t owns the NV groups of VEC consecutive columns
// that start at (j * TEAM + t) * VEC.  VEC values are one 16-byte access where base and stride
// allow it (VEC > 1), single values otherwise.  A row's last, partial group goes by single values.
template <typename T, int VEC, int TEAM, int NV>
struct Row {
    static constexpr int kN = VEC * NV;
    PRISM_DEV static int col(int t, int j) { return (j * TEAM + t) * VEC; }
};

template <typename T, int VEC>
struct alignas(VEC * sizeof(T)) Pack {
    T v[VEC];
};

template <typename T, int VEC>
PRISM_DEV Pack<T, VEC> load_pack(const T* row, int c, int dim) {
    Pack<T, VEC> p;
    if (c + VEC <= dim) {
        p = *reinterpret_cast<const Pack<T, VEC>*>(row + c);
    } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) p.v[e] = c + e < dim ? row[c + e] : from_f32<T>(0.0f);
    }
    return p;
}
template <typename T, int VEC>
PRISM_DEV void store_pack(T* row, int c, int dim, const Pack<T, VEC>& p) {
    if (c + VEC <= dim) {
        *reinterpret_cast<Pack<T, VEC>*>(row + c) = p;
    } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e)
            if (c + e < dim) row[c + e] = p.v[e];
    }
}
// a parameter vector's value: fp32, or the rows' type T
template <typename T>
PRISM_DEV float param_at(const void* w, int f32, int c) {
    return f32 ? static_cast<const float*>(w)[c] : to_f32(static_cast<const T*>(w)[c]);
}

// Sums of two values over a team.  Teams of up to a warp: butterfly, every lane gets the same bits.
// Teams of a whole CTA: butterfly, then the warps' sums in order from shared memory.
template <int TEAM>
PRISM_DEV void team_sum2(float& a, float& b, float2* red) {
    constexpr int kW = TEAM < 32 ? TEAM : 32;
#pragma unroll
    for (int o = kW / 2; o > 0; o >>= 1) {
        a += __shfl_xor_sync(0xffffffffu, a, o);
        b += __shfl_xor_sync(0xffffffffu, b, o);
    }
    if (TEAM > 32) {
        __syncthreads();  // the sums of the call before have been read
        if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = make_float2(a, b);
        __syncthreads();
        a = b = 0.0f;
#pragma unroll
        for (int w = 0; w < TEAM / 32; ++w) {
            a += red[w].x;
            b += red[w].y;
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

constexpr int kThreads = 256;

// y = (x - mean) rstd w + b.  One pass over memory: the row stays in registers between the mean,
// the centred second moment and the output.  Memory-bound: 2 R D s bytes.  The next row's loads
// are issued before this row's sums, so each team keeps two rows in flight.
template <typename T, int VEC, int TEAM, int NV>
__global__ void __launch_bounds__(kThreads) norm_kernel(const NormArgs a) {
    using R = Row<T, VEC, TEAM, NV>;
    __shared__ float2 red[kThreads / 32];
    constexpr int kTeams = kThreads / TEAM;
    constexpr bool kHold = R::kN <= 16;  // weight and bias stay in registers across rows
    const int t = threadIdx.x % TEAM;
    const int64_t step = (int64_t)gridDim.x * kTeams;
    int64_t row = (int64_t)blockIdx.x * kTeams + threadIdx.x / TEAM;
    const T* x = static_cast<const T*>(a.x);
    T* y = static_cast<T*>(a.y);
    const float inv = 1.0f / (float)a.dim;
    float w[kHold ? R::kN : 1], b[kHold ? R::kN : 1];
    if (kHold) {
#pragma unroll
        for (int i = 0; i < R::kN; ++i) {
            const int c = R::col(t, i / VEC) + i % VEC;
            w[i] = a.weight && c < a.dim ? param_at<T>(a.weight, a.param_f32, c) : 1.0f;
            b[i] = a.bias && c < a.dim ? param_at<T>(a.bias, a.param_f32, c) : 0.0f;
        }
    }
    Pack<T, VEC> cur[NV], nxt[NV];
    // every thread of a warp runs the same number of rows (the shuffles need the whole warp);
    // teams past the last row work on zeros and store nothing
    auto load = [&](Pack<T, VEC>(&p)[NV], int64_t r) {
        const T* src = x + (r < a.rows ? r : 0) * a.xs;
        const int lim = r < a.rows ? a.dim : 0;
#pragma unroll
        for (int j = 0; j < NV; ++j) p[j] = load_pack<T, VEC>(src, R::col(t, j), lim);
    };
    const int64_t first = (int64_t)blockIdx.x * kTeams + (TEAM < 32 ? (threadIdx.x / 32) * (32 / TEAM) : threadIdx.x / TEAM);
    load(cur, row);
    for (int64_t lead = first; lead < a.rows; lead += step, row += step) {
        if (lead + step < a.rows) load(nxt, row + step);
        float v[R::kN], s0 = 0.0f, s1 = 0.0f;
#pragma unroll
        for (int i = 0; i < R::kN; ++i) {
            v[i] = to_f32(cur[i / VEC].v[i % VEC]);
            s0 += v[i];
        }
        team_sum2<TEAM>(s0, s1, red);
        const float mean = s0 * inv;
        float q = 0.0f;
#pragma unroll
        for (int i = 0; i < R::kN; ++i) {
            v[i] -= mean;
            if (R::col(t, i / VEC) + i % VEC < a.dim) q = fmaf(v[i], v[i], q);
        }
        s1 = 0.0f;
        team_sum2<TEAM>(q, s1, red);
        const float rstd = rsqrtf(fmaf(q, inv, a.eps));
        if (row < a.rows) {
            T* dst = y + row * a.ys;
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int c = R::col(t, j);
                Pack<T, VEC> o;
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const int i = j * VEC + e;
                    float wi, bi;
                    if (kHold) {
                        wi = w[kHold ? i : 0];
                        bi = b[kHold ? i : 0];
                    } else {
                        wi = a.weight && c + e < a.dim ? param_at<T>(a.weight, a.param_f32, c + e) : 1.0f;
                        bi = a.bias && c + e < a.dim ? param_at<T>(a.bias, a.param_f32, c + e) : 0.0f;
                    }
                    o.v[e] = from_f32<T>(fmaf(v[i] * rstd, wi, bi));
                }
                store_pack<T, VEC>(dst, c, a.dim, o);
            }
            if (t == 0) {
                if (a.mean) a.mean[row] = mean;
                if (a.rstd) a.rstd[row] = rstd;
            }
        }
#pragma unroll
        for (int j = 0; j < NV; ++j) cur[j] = nxt[j];
    }
}

// With xh = (x - mean) rstd and g = dy w:
//   dx = rstd (g - mean_c(g) - xh mean_c(g xh)) [+ add],  dweight = sum_r dy xh,  dbias = sum_r dy.
// One pass over x and dy: each thread keeps its columns' dweight and dbias sums over all the rows
// its team walks, the CTA's teams are added in order, and norm_fold_kernel adds the CTAs' partial
// sums in order (no atomics: the same inputs give the same bits).
template <typename T, int VEC, int TEAM, int NV>
__global__ void __launch_bounds__(kThreads) norm_back_kernel(const NormBackArgs a) {
    using R = Row<T, VEC, TEAM, NV>;
    extern __shared__ float fold[];  // [2][dim], teams smaller than the CTA
    __shared__ float2 red[kThreads / 32];
    constexpr int kTeams = kThreads / TEAM;
    constexpr bool kHold = R::kN <= 16;
    const int t = threadIdx.x % TEAM;
    const int64_t step = (int64_t)gridDim.x * kTeams;
    int64_t row = (int64_t)blockIdx.x * kTeams + threadIdx.x / TEAM;
    const T *x = static_cast<const T*>(a.x), *dy = static_cast<const T*>(a.dy), *add = static_cast<const T*>(a.add);
    T* dx = static_cast<T*>(a.dx);
    const float inv = 1.0f / (float)a.dim;
    float w[kHold ? R::kN : 1];
    if (kHold) {
#pragma unroll
        for (int i = 0; i < R::kN; ++i) {
            const int c = R::col(t, i / VEC) + i % VEC;
            w[i] = a.weight && c < a.dim ? param_at<T>(a.weight, a.param_f32, c) : 1.0f;
        }
    }
    float dw[R::kN], db[R::kN];
#pragma unroll
    for (int i = 0; i < R::kN; ++i) dw[i] = db[i] = 0.0f;
    const int64_t first = (int64_t)blockIdx.x * kTeams + (TEAM < 32 ? (threadIdx.x / 32) * (32 / TEAM) : threadIdx.x / TEAM);
    for (int64_t lead = first; lead < a.rows; lead += step, row += step) {
        const bool in = row < a.rows;
        const int64_t r = in ? row : 0;
        const int lim = in ? a.dim : 0;
        const float mean = in ? a.mean[r] : 0.0f, rstd = in ? a.rstd[r] : 0.0f;
        Pack<T, VEC> px[NV], pg[NV];
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            px[j] = load_pack<T, VEC>(x + r * a.xs, R::col(t, j), lim);
            pg[j] = load_pack<T, VEC>(dy + r * a.dys, R::col(t, j), lim);
        }
        float g[R::kN], xh[R::kN], s0 = 0.0f, s1 = 0.0f;
#pragma unroll
        for (int i = 0; i < R::kN; ++i) {
            const int c = R::col(t, i / VEC) + i % VEC;
            const float d = to_f32(pg[i / VEC].v[i % VEC]);
            // columns past the row hold zeros, whose xh is not zero: they take no part
            xh[i] = c < lim ? (to_f32(px[i / VEC].v[i % VEC]) - mean) * rstd : 0.0f;
            float wi;
            if (kHold)
                wi = w[kHold ? i : 0];
            else
                wi = a.weight && c < a.dim ? param_at<T>(a.weight, a.param_f32, c) : 1.0f;
            g[i] = d * wi;
            dw[i] = fmaf(d, xh[i], dw[i]);
            db[i] += d;
            s0 += g[i];
            s1 = fmaf(g[i], xh[i], s1);
        }
        team_sum2<TEAM>(s0, s1, red);
        const float m0 = s0 * inv, m1 = s1 * inv;
        if (in) {
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int c = R::col(t, j);
                Pack<T, VEC> o, pa;
                if (add) pa = load_pack<T, VEC>(add + r * a.adds, c, a.dim);
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const int i = j * VEC + e;
                    float d = rstd * (g[i] - m0 - xh[i] * m1);
                    if (add) d += to_f32(pa.v[e]);
                    o.v[e] = from_f32<T>(d);
                }
                store_pack<T, VEC>(dx + r * a.dxs, c, a.dim, o);
            }
        }
    }
    if (!a.part) return;
    float* out = a.part + (int64_t)blockIdx.x * 2 * a.dim;
    if (TEAM < kThreads) {
        // a warp's teams by butterfly, then the warps one after the other
        constexpr int kWarps = kThreads / 32;
        if (TEAM < 32) {
#pragma unroll
            for (int i = 0; i < R::kN; ++i) {
#pragma unroll
                for (int o = TEAM; o < 32; o <<= 1) {
                    dw[i] += __shfl_xor_sync(0xffffffffu, dw[i], o);
                    db[i] += __shfl_xor_sync(0xffffffffu, db[i], o);
                }
            }
        }
        for (int wp = 0; wp < kWarps; ++wp) {
            if ((int)(threadIdx.x >> 5) == wp && (threadIdx.x & 31) < TEAM) {
#pragma unroll
                for (int i = 0; i < R::kN; ++i) {
                    const int c = R::col(t, i / VEC) + i % VEC;
                    if (c < a.dim) {
                        fold[c] = wp ? fold[c] + dw[i] : dw[i];
                        fold[a.dim + c] = wp ? fold[a.dim + c] + db[i] : db[i];
                    }
                }
            }
            __syncthreads();
        }
        for (int c = threadIdx.x; c < 2 * a.dim; c += kThreads) out[c] = fold[c];
    } else {
#pragma unroll
        for (int i = 0; i < R::kN; ++i) {
            const int c = R::col(t, i / VEC) + i % VEC;
            if (c < a.dim) {
                out[c] = dw[i];
                out[a.dim + c] = db[i];
            }
        }
    }
}

// Adds the CTAs' partial sums: 32 columns a CTA, 8 threads a column over every 8th partial, then the 8
// in order.
template <typename T>
__global__ void __launch_bounds__(kThreads)
    norm_fold_kernel(const float* part, int n_part, int dim, void* dweight, void* dbias, int param_f32) {
    __shared__ float red[8][33];
    grid_dep_wait();
    const int lane = threadIdx.x & 31, k = threadIdx.x >> 5;
    const int c = blockIdx.x * 32 + lane;  // over [dweight | dbias]
    float s = 0.0f;
    if (c < 2 * dim)
        for (int p = k; p < n_part; p += 8) s += part[(int64_t)p * 2 * dim + c];
    red[k][lane] = s;
    __syncthreads();
    if (k == 0 && c < 2 * dim) {
        s = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) s += red[i][lane];
        void* dst = c < dim ? dweight : dbias;
        const int i = c < dim ? c : c - dim;
        if (dst) {
            if (param_f32)
                static_cast<float*>(dst)[i] = s;
            else
                static_cast<T*>(dst)[i] = from_f32<T>(s);
        }
    }
}

// ---- dropout ---------------------------------------------------------------------------------
// Philox4x32-10 (Salmon, Moraes, Dror, Shaw: Parallel random numbers, as easy as 1, 2, 3; 2011).
PRISM_DEV uint4 philox(uint4 c, uint2 k) {
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t p0 = (uint64_t)0xD2511F53u * c.x, p1 = (uint64_t)0xCD9E8D57u * c.z;
        c = make_uint4((uint32_t)(p1 >> 32) ^ c.y ^ k.x, (uint32_t)p1, (uint32_t)(p0 >> 32) ^ c.w ^ k.y, (uint32_t)p0);
        k.x += 0x9E3779B9u;
        k.y += 0xBB67AE85u;
    }
    return c;
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
    const uint2 key = make_uint2((uint32_t)seed, (uint32_t)(seed >> 32));
    const int64_t n = a.rows * a.dim, blocks = (n + 7) / 8, stride = (int64_t)gridDim.x * kThreads;
    const T *x = static_cast<const T*>(a.x), *res = static_cast<const T*>(a.residual);
    T* y = static_cast<T*>(a.y);
    constexpr int UNR = 2, E = 16 / sizeof(T);
    for (int64_t b0 = (int64_t)blockIdx.x * kThreads + threadIdx.x; b0 < blocks; b0 += UNR * stride) {
        if (VEC8) {
            Pack<T, E> px[UNR][8 / E], pr[UNR][8 / E];
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
                    px[u][q] = *reinterpret_cast<const Pack<T, E>*>(x + r * a.xs + c + q * E);
                    if (res) pr[u][q] = *reinterpret_cast<const Pack<T, E>*>(res + r * a.rs + c + q * E);
                }
            }
#pragma unroll
            for (int u = 0; u < UNR; ++u) {
                const int64_t b = b0 + u * stride;
                if (b >= blocks) continue;
                const uint4 w = philox(make_uint4((uint32_t)b, (uint32_t)(b >> 32), (uint32_t)offset, (uint32_t)(offset >> 32)), key);
                const uint32_t bits[4] = {w.x, w.y, w.z, w.w};
                if (full[u]) {
#pragma unroll
                    for (int q = 0; q < 8 / E; ++q) {
                        Pack<T, E> o;
#pragma unroll
                        for (int e = 0; e < E; ++e) {
                            const int i = q * E + e;
                            const uint32_t h = (i & 1) ? bits[i >> 1] >> 16 : bits[i >> 1] & 0xffffu;
                            const float v = h >= a.threshold ? to_f32(px[u][q].v[e]) * a.scale : 0.0f;
                            o.v[e] = from_f32<T>(res ? v + to_f32(pr[u][q].v[e]) : v);
                        }
                        *reinterpret_cast<Pack<T, E>*>(y + yo[u] + q * E) = o;
                    }
                } else {  // the last block of a flat tensor (rows of a strided one are multiples of 8)
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int64_t at = b * 8 + i;
                        if (at < n) {
                            const uint32_t h = (i & 1) ? bits[i >> 1] >> 16 : bits[i >> 1] & 0xffffu;
                            const float v = h >= a.threshold ? to_f32(x[at]) * a.scale : 0.0f;
                            y[at] = from_f32<T>(res ? v + to_f32(res[at]) : v);
                        }
                    }
                }
            }
        } else {
#pragma unroll 1
            for (int u = 0; u < UNR; ++u) {
                const int64_t b = b0 + u * stride;
                if (b >= blocks) break;
                const uint4 w = philox(make_uint4((uint32_t)b, (uint32_t)(b >> 32), (uint32_t)offset, (uint32_t)(offset >> 32)), key);
                const uint32_t bits[4] = {w.x, w.y, w.z, w.w};
                int64_t r = (b * 8) / a.dim;
                int c = (int)(b * 8 - r * a.dim);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    if (r < a.rows) {
                        const uint32_t h = (i & 1) ? bits[i >> 1] >> 16 : bits[i >> 1] & 0xffffu;
                        const float v = h >= a.threshold ? to_f32(x[r * a.xs + c]) * a.scale : 0.0f;
                        y[r * a.ys + c] = from_f32<T>(res ? v + to_f32(res[r * a.rs + c]) : v);
                    }
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

inline cudaStream_t as_stream(void* s) { return reinterpret_cast<cudaStream_t>(s); }
int cuda_rc(cudaError_t e, const char* what) {
    return e == cudaSuccess ? PRISM_OK : fail(PRISM_E_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

constexpr int kNormMaxDim = 16384;
constexpr int kBackCtasPerSm = 2;

// What a row's threads hold, by type, alignment and width: f(T{}, VEC, TEAM, NV) as constants.
template <typename T, typename F>
int with_shape(bool vec, int dim, F&& f) {
    constexpr int V = 16 / sizeof(T);
    using std::integral_constant;
#define SHAPE(VEC, TEAM, NV) \
    return f(integral_constant<int, VEC>{}, integral_constant<int, TEAM>{}, integral_constant<int, NV>{})
    if (vec) {
        if (dim <= 8 * V) SHAPE(V, 8, 1);
        if (dim <= 16 * V) SHAPE(V, 16, 1);
        if (dim <= 32 * V) SHAPE(V, 32, 1);
        if (dim <= 64 * V) SHAPE(V, 32, 2);
        if (dim <= 128 * V) SHAPE(V, 32, 4);
        if (dim <= 512 * V) SHAPE(V, 256, 2);
        if (dim <= 1024 * V) SHAPE(V, 256, 4);
        if (dim <= 2048 * V) SHAPE(V, 256, 8);
        SHAPE(V, 256, 64 / V);
    }
    if (dim <= 64) SHAPE(1, 16, 4);
    if (dim <= 256) SHAPE(1, 32, 8);
    if (dim <= 1024) SHAPE(1, 32, 32);
    if (dim <= 4096) SHAPE(1, 256, 16);
    SHAPE(1, 256, 64);
#undef SHAPE
}

template <typename F>
int with_type(int dtype, F&& f) {
    if (dtype == PRISM_DTYPE_F16) return f(__half{});
    if (dtype == PRISM_DTYPE_BF16) return f(__nv_bfloat16{});
    return f(float{});
}

// 16-byte groups: base and row pitch multiples of 16 bytes
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
int check_stride(const char* who, const char* name, const void* t, int64_t stride, int64_t rows, int dim, int es) {
    if (!t) return PRISM_OK;
    if ((uintptr_t)t % es) return fail(PRISM_E_ALIGN, "%s: %s is not aligned to its type", who, name);
    if (rows > 1 && stride < dim)
        return fail(PRISM_E_ARG, "%s: %s_stride %lld below dim %d", who, name, (long long)stride, dim);
    if (rows > 0 && stride > (int64_t)1 << 40) return fail(PRISM_E_RANGE, "%s: %s_stride %lld", who, name, (long long)stride);
    if (rows > (int64_t)1 << 40) return fail(PRISM_E_RANGE, "%s: rows %lld", who, (long long)rows);
    return PRISM_OK;
}
// outputs may be an input itself (same address and stride), never share bytes with it otherwise
bool bad_alias(const void* out, int64_t so, const void* in, int64_t si, int64_t rows, int64_t dim, int64_t es) {
    if (rows <= 1) so = si = dim;
    if (out == in && so == si) return false;
    return rows_overlap(out, so, in, si, rows, dim, es);
}

// CTAs of the backward kernel: one partial sum each
int back_ctas(const prism_ctx* ctx, int64_t rows, int teams) {
    return (int)std::min<int64_t>((rows + teams - 1) / teams, (int64_t)ctx->sm_count * kBackCtasPerSm);
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
        (rc = check_stride("prism_layer_norm", "y", y, p->y_stride, p->rows, p->dim, es)))
        return rc;
    if (bad_alias(y, p->y_stride, x, p->x_stride, p->rows, p->dim, es))
        return fail(PRISM_E_ARG, "prism_layer_norm: y overlaps x");
    DeviceGuard g(ctx->device);
    NormArgs a{x, weight, bias, y, mean, rstd, p->rows, p->x_stride, p->y_stride, p->dim,
               p->param_dtype == PRISM_DTYPE_F32, p->eps};
    const bool vec = vec_ok(x, p->x_stride, es) && vec_ok(y, p->y_stride, es);
    return with_type(p->dtype, [&](auto tag) {
        using T = decltype(tag);
        return with_shape<T>(vec, p->dim, [&](auto v, auto team, auto nv) {
            constexpr int kTeams = kThreads / decltype(team)::value;
            const int64_t want = (p->rows + kTeams - 1) / kTeams;
            const int grid = (int)std::min<int64_t>(want, (int64_t)ctx->sm_count * 8);
            norm_kernel<T, decltype(v)::value, decltype(team)::value, decltype(nv)::value>
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
    DeviceGuard g(ctx->device);
    if (p->rows == 0) {  // no rows: the sums are zero
        const size_t n = (size_t)p->dim * dtype_bytes(p->param_dtype);
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
    NormBackArgs a{x,  weight, dy, add, mean, rstd, dx, sums ? static_cast<float*>(workspace) : nullptr,
                   p->rows, p->x_stride, p->dy_stride, p->add_stride, p->dx_stride, p->dim,
                   p->param_dtype == PRISM_DTYPE_F32};
    const bool vec = vec_ok(x, p->x_stride, es) && vec_ok(dy, p->dy_stride, es) && vec_ok(add, p->add_stride, es) &&
                     vec_ok(dx, p->dx_stride, es);
    return with_type(p->dtype, [&](auto tag) {
        using T = decltype(tag);
        int grid = 0;
        int rc = with_shape<T>(vec, p->dim, [&](auto v, auto team, auto nv) {
            constexpr int kTeam = decltype(team)::value;
            grid = back_ctas(ctx, p->rows, kThreads / kTeam);
            const size_t smem = sums && kTeam < kThreads ? (size_t)p->dim * 8 : 0;
            norm_back_kernel<T, decltype(v)::value, kTeam, decltype(nv)::value>
                <<<grid, kThreads, smem, as_stream(stream)>>>(a);
            return cuda_rc(cudaGetLastError(), who);
        });
        if (rc || !sums) return rc;
        return cuda_rc(launch_pdl(norm_fold_kernel<T>, dim3((2 * p->dim + 31) / 32), dim3(kThreads), 0, as_stream(stream),
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
