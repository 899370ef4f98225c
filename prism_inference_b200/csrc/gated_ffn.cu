// gated_ffn.cu - the gated feed-forward block, forward and backward, on the sm_100a tensor cores.
//
//   g = x Wg^T + bg,  u = x Wu^T + bu,  h = act(g) u,  y = h Wd^T + bd [+ residual]
//   dh = dy Wd,  du = dh act(g),  dg = dh u act'(g),  dx = dg Wg + du Wu,
//   dWg = dg^T x,  dWu = du^T x,  dWd = dy^T h,  dbg, dbu, dbd = column sums of dg, du, dy
//
// One persistent kernel template over CTA pairs (tcgen05 cta_group::2): a pair owns a 256 x 256 output
// tile, each CTA 128 rows of it, and loads half of the B operand, so an SM reads 32 KB per 64 deep
// step instead of the 48 KB that a CTA by itself would (the 128 x 256 tiles of both would pull 94 bytes
// a clock from L2, which it does not deliver).  Operands come by TMA in the order they lie in memory;
// K-major or MN-major is a bit of the MMA, so nothing is transposed.
//   UP    [g | u] of 128 hidden columns side by side (the leader loads Wg, its peer Wu) -> h
//   DOWN  y = h Wd^T
//   BACK  [g | u] again from x, dh = dy Wd beside them -> dg, du, h
//   XW    dx tiles and dW tiles (split over rows) in one launch: neither fills the GPU alone
// Rows go through in chunks, so the scratch memory does not grow with the batch.
#include <cudaTypedefs.h>

#include <algorithm>

#include "gated_tc.cuh"

namespace prism {
namespace {

enum Kind : int { UP, DOWN, BACK, XW };

constexpr int kEpiWarps = 8;
constexpr int kThreads = 32 * (2 + kEpiWarps);
constexpr int kStageA = 16384, kStageB = 16384, kStage = kStageA + kStageB;
constexpr int kStages = 5;
constexpr int kStageOut = 6144;  // a warp's store staging: three 32 x 32 16-bit boxes or one of fp32
constexpr int kBiasBytes = kEpiWarps * 1024;
constexpr int kSmem = kStages * kStage + kEpiWarps * kStageOut + kBiasBytes + 512 + 1024;

struct Bars {
    uint64_t full[kStages], empty[kStages], acc_full[2], acc_empty[2];
    uint32_t tmem_base;
    int abort;
};

struct Maps {
    CUtensorMap a0, a1, b0, b1, b2, out, p_k, p_mn, x_mn, dy_mn, dw;
};

struct Args {
    int rows, dim, hidden;      // rows of this chunk
    int m_tiles, n_tiles;       // 256-row tiles; column tiles (128 hidden for UP / BACK, bn else)
    int bn;                     // N of an output tile over dim: 256 or 128
    int units, x_units;         // XW: the first x_units are dx tiles, the others dW tiles
    int w_tiles, k_per, k_all;  // XW: 256-row tiles of one weight's hidden axis; row blocks a split, in all
    int act, bf16;
    const void *b_gate, *b_up, *b_down;
    const void* residual;
    int64_t residual_stride;
    uint32_t* err;
};

template <typename T>
PRISM_DEV float ld_bias(const void* b, int i, int n) {
    return b && i < n ? to_f32(static_cast<const T*>(b)[i]) : 0.0f;
}

// one unit of work, the same on every role
struct Unit {
    int mt, nt, seg, k0, nkb;  // seg: XW's dW units: 0 dWg, 1 dWu, 2 dWd^T; -1: dx
    int split;
};
template <int KIND>
PRISM_DEV Unit unit_of(const Args& a, int u) {
    Unit r;
    r.seg = -1;
    r.k0 = 0;
    r.split = 0;
    const int kd = (a.dim + 63) / 64, kh = (a.hidden + 63) / 64;
    if (KIND != XW || u < a.x_units) {
        r.mt = u / a.n_tiles;
        r.nt = u % a.n_tiles;
        r.nkb = KIND == UP ? kd : KIND == DOWN ? kh : KIND == BACK ? 2 * kd : 2 * kh;
    } else {
        u -= a.x_units;
        const int per = 3 * a.w_tiles * a.n_tiles;
        r.split = u / per;
        u %= per;
        r.nt = u % a.n_tiles;
        u /= a.n_tiles;
        r.mt = u % a.w_tiles;
        r.seg = u / a.w_tiles;
        r.k0 = r.split * a.k_per;
        r.nkb = min(a.k_per, a.k_all - r.k0);
    }
    return r;
}

// A 32 x 32 box of a warp's rows: this lane's row as 16 packed pairs into 64-byte swizzled rows.
PRISM_DEV void stage_row64(unsigned char* buf, int lane, const uint32_t (&v)[16]) {
#pragma unroll
    for (int q = 0; q < 4; ++q)
        *reinterpret_cast<uint4*>(buf + sw64_off(lane, q)) = make_uint4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
}

template <typename T, int ACT>
PRISM_DEV void gate_cols(const uint32_t (&g)[32], const uint32_t (&u)[32], const float* bg, const float* bu, uint32_t (&out)[16]) {
#pragma unroll
    for (int j = 0; j < 16; ++j) {
        const float2 b0 = reinterpret_cast<const float2*>(bg)[j], b1 = reinterpret_cast<const float2*>(bu)[j];
        const float h0 = gate<ACT>(__uint_as_float(g[2 * j]) + b0.x) * (__uint_as_float(u[2 * j]) + b1.x);
        const float h1 = gate<ACT>(__uint_as_float(g[2 * j + 1]) + b0.y) * (__uint_as_float(u[2 * j + 1]) + b1.y);
        out[j] = pack2<T>(h0, h1);
    }
}
// dg over g's registers' first half, du, h: packed
template <typename T, int ACT>
PRISM_DEV void grad_cols(const uint32_t (&g)[32], const uint32_t (&u)[32], const uint32_t (&dh)[32], const float* bg,
                         const float* bu, uint32_t (&dg)[16], uint32_t (&du)[16], uint32_t (&h)[16]) {
#pragma unroll
    for (int j = 0; j < 16; ++j) {
        const float2 b0 = reinterpret_cast<const float2*>(bg)[j], b1 = reinterpret_cast<const float2*>(bu)[j];
        float pg[2], pu[2], ph[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const float gv = __uint_as_float(g[2 * j + e]) + (e ? b0.y : b0.x);
            const float uv = __uint_as_float(u[2 * j + e]) + (e ? b1.y : b1.x);
            const float dv = __uint_as_float(dh[2 * j + e]);
            float a, d;
            gate_grad<ACT>(gv, a, d);
            pg[e] = dv * uv * d;
            pu[e] = dv * a;
            ph[e] = a * uv;
        }
        dg[j] = pack2<T>(pg[0], pg[1]);
        du[j] = pack2<T>(pu[0], pu[1]);
        h[j] = pack2<T>(ph[0], ph[1]);
    }
}

template <typename T, int KIND>
__global__ void __launch_bounds__(kThreads, 1) __cluster_dims__(2, 1, 1)
    gated_kernel(const Args a, const __grid_constant__ Maps maps) {
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = smem_align1k(smem_raw);
    unsigned char* s_out = smem + kStages * kStage;
    float* s_bias = reinterpret_cast<float*>(s_out + kEpiWarps * kStageOut);
    Bars* bars = reinterpret_cast<Bars*>(s_out + kEpiWarps * kStageOut + kBiasBytes);
    volatile int* abort = &bars->abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)cluster_rank(), pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    constexpr int kSlots = KIND == BACK ? 1 : 2;  // BACK's g | u | dh take 384 of the 512 columns
    constexpr bool bf16 = sizeof(T) == 2 && !std::is_same<T, __half>::value;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&bars->full[s], 1);
            mbar_init(&bars->empty[s], 1);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(&bars->acc_full[s], 1);
            mbar_init(&bars->acc_empty[s], 2 * kEpiWarps);  // used in the leader: both CTAs' epilogue warps
        }
        bars->abort = 0;
        fence_barrier_init();
        fence_async_shared();
    }
    __syncwarp();
    if (warp == 1) tmem_alloc_pair(&bars->tmem_base, 512);
    tc_fence_before();
    __syncthreads();
    cluster_sync();
    tc_fence_after();
    const uint32_t tmem = bars->tmem_base;
    grid_dep_wait();

    if (warp == 0) {
        // ---- producer (both CTAs): this CTA's rows of A, its half of B, all on the leader's barrier
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int u = pair; u < a.units && ok; u += pairs) {
            const Unit t = unit_of<KIND>(a, u);
            const int kd = (a.dim + 63) / 64, kh = (a.hidden + 63) / 64;
            const int bh = a.bn / 2;  // this CTA's share of an N tile over dim
            for (int kb = 0; kb < t.nkb; ++kb) {
                if (!mbar_wait_w(&bars->empty[stage], phase ^ 1, abort)) { ok = false; break; }
                if (lane == 0) {
                    const uint32_t sa = smem_u32(smem + stage * kStage), sb = sa + kStageA;
                    const uint32_t bar = peer_addr(smem_u32(&bars->full[stage]), 0);
                    uint32_t bytes;
                    const int row = t.mt * 256 + rank * 128;
                    if (KIND == UP || (KIND == BACK && kb < kd)) {
                        bytes = kStageA + kStageB;
                        if (rank == 0) mbar_expect_tx(&bars->full[stage], 2 * bytes);
                        tma_load_2d_pair(sa, &maps.a0, bar, kb * 64, row);
                        tma_load_2d_pair(sb, rank ? &maps.b1 : &maps.b0, bar, kb * 64, t.nt * 128);
                    } else if (KIND == BACK) {
                        bytes = kStageA + kStageB / 2;
                        if (rank == 0) mbar_expect_tx(&bars->full[stage], 2 * bytes);
                        tma_load_2d_pair(sa, &maps.a1, bar, (kb - kd) * 64, row);
                        tma_load_2d_pair(sb, &maps.b2, bar, t.nt * 128 + rank * 64, (kb - kd) * 64);
                    } else if (KIND == DOWN) {
                        bytes = kStageA + bh * 128;
                        if (rank == 0) mbar_expect_tx(&bars->full[stage], 2 * bytes);
                        tma_load_2d_pair(sa, &maps.a0, bar, kb * 64, row);
                        tma_load_2d_pair(sb, &maps.b0, bar, kb * 64, t.nt * a.bn + rank * bh);
                    } else if (t.seg < 0) {
                        bytes = kStageA + bh * 128;
                        if (rank == 0) mbar_expect_tx(&bars->full[stage], 2 * bytes);
                        const int s = kb >= kh, k = (kb - s * kh) * 64;
                        tma_load_3d_pair(sa, &maps.p_k, bar, k, row, s);
                        for (int n = 0; n < bh; n += 64)
                            tma_load_2d_pair(sb + n * 128, s ? &maps.b1 : &maps.b0, bar, t.nt * a.bn + rank * bh + n, k);
                    } else {
                        bytes = kStageA + bh * 128;
                        if (rank == 0) mbar_expect_tx(&bars->full[stage], 2 * bytes);
                        const int k = (t.k0 + kb) * 64;
                        for (int m = 0; m < 128; m += 64) tma_load_3d_pair(sa + m * 128, &maps.p_mn, bar, row + m, k, t.seg);
                        for (int n = 0; n < bh; n += 64)
                            tma_load_2d_pair(sb + n * 128, t.seg == 2 ? &maps.dy_mn : &maps.x_mn, bar,
                                             t.nt * a.bn + rank * bh + n, k);
                    }
                }
                __syncwarp();
                if (++stage == kStages) {
                    stage = 0;
                    phase ^= 1;
                }
            }
        }
    } else if (warp == 1) {
        // ---- MMA issuer: the leader's, for both CTAs
        if (rank == 0) {
            int stage = 0, it = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int u = pair; u < a.units && ok; u += pairs, ++it) {
                const Unit t = unit_of<KIND>(a, u);
                const int slot = it % kSlots;
                const uint32_t acc = tmem + slot * 256;
                if (!mbar_wait_cl(&bars->acc_empty[slot], ((it / kSlots) & 1) ^ 1, abort)) ok = false;
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tc_fence_after();
                const int kd = (a.dim + 63) / 64;
                for (int kb = 0; kb < t.nkb; ++kb) {
                    if (!mbar_wait_w(&bars->full[stage], phase, abort)) { ok = false; break; }
                    tc_fence_after();
                    const uint32_t sa = smem_u32(smem + stage * kStage), sb = sa + kStageA;
                    if (KIND == XW && t.seg >= 0) {
                        const uint32_t id = idesc_pair(256, a.bn, bf16, 1, 1);
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            mma_pair_ss_w(acc, sdesc_mn(sa + k * 2048, 8192), sdesc_mn(sb + k * 2048, 8192), id, (kb | k) != 0);
                    } else if (KIND == XW) {
                        const uint32_t id = idesc_pair(256, a.bn, bf16, 0, 1);
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            mma_pair_ss_w(acc, sdesc(sa + k * 32, SW128), sdesc_mn(sb + k * 2048, 8192), id, (kb | k) != 0);
                    } else if (KIND == BACK && kb >= kd) {
                        const uint32_t id = idesc_pair(256, 128, bf16, 0, 1);
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            mma_pair_ss_w(acc + 256, sdesc(sa + k * 32, SW128), sdesc_mn(sb + k * 2048, 8192), id,
                                          (kb - kd) | k);
                    } else {
                        const uint32_t id = idesc_pair(256, KIND == DOWN ? a.bn : 256, bf16, 0, 0);
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            mma_pair_ss_w(acc, sdesc(sa + k * 32, SW128), sdesc(sb + k * 32, SW128), id, (kb | k) != 0);
                    }
                    mma_commit_pair_w(&bars->empty[stage]);
                    if (++stage == kStages) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
                if (!ok) break;
                mma_commit_pair_w(&bars->acc_full[slot]);
            }
        }
    } else {
        // ---- epilogue: warp w reads TMEM lanes 32 (w % 4) .., half of the columns
        const int quad = warp & 3, half = (warp - 2) >> 2;
        unsigned char* buf = s_out + (warp - 2) * kStageOut;
        const uint32_t sbuf = smem_u32(buf);
        float* bias = s_bias + (warp - 2) * 256;
        const uint32_t lane_addr = (uint32_t)(quad * 32) << 16;
        const uint32_t acc_empty0 = peer_addr(smem_u32(&bars->acc_empty[0]), 0);
        const uint32_t acc_empty1 = peer_addr(smem_u32(&bars->acc_empty[1]), 0);
        int it = 0;
        for (int u = pair; u < a.units; u += pairs, ++it) {
            const Unit t = unit_of<KIND>(a, u);
            const int slot = it % kSlots;
            const int row = t.mt * 256 + rank * 128 + quad * 32;
            constexpr bool kGate = KIND == UP || KIND == BACK;
            const int cols = kGate ? 64 : a.bn / 2;  // this warp's
            const int col0 = kGate ? t.nt * 128 + half * 64 : t.nt * a.bn + half * cols;
            // biases of this warp's columns
            if (kGate) {
                for (int i = lane; i < 64; i += 32) {
                    bias[i] = ld_bias<T>(a.b_gate, col0 + i, a.hidden);
                    bias[64 + i] = ld_bias<T>(a.b_up, col0 + i, a.hidden);
                }
            } else if (KIND == DOWN) {
                for (int i = lane; i < cols; i += 32) bias[i] = ld_bias<T>(a.b_down, col0 + i, a.dim);
            }
            __syncwarp();
            const bool got = mbar_wait_w(&bars->acc_full[slot], (it / kSlots) & 1, abort);
            if (!got) break;
            tc_fence_after();
            const uint32_t acc = tmem + lane_addr + slot * 256;
            for (int g = 0; g < cols; g += 32) {
                const int c = col0 + g;
                if (kGate) {
                    uint32_t rg[32], ru[32];
                    tmem_ld32(acc + half * 64 + g, rg);
                    tmem_ld32(acc + 128 + half * 64 + g, ru);
                    if (KIND == UP) {
                        uint32_t o[16];
                        tmem_ld_wait();
                        if (a.act == kActSilu) gate_cols<T, kActSilu>(rg, ru, bias + g, bias + 64 + g, o);
                        else if (a.act == kActGelu) gate_cols<T, kActGelu>(rg, ru, bias + g, bias + 64 + g, o);
                        else gate_cols<T, kActRelu>(rg, ru, bias + g, bias + 64 + g, o);
                        if (lane == 0) tma_store_wait_read<0>();
                        __syncwarp();
                        stage_row64(buf, lane, o);
                        fence_async_shared();
                        __syncwarp();
                        if (lane == 0 && c < a.hidden && row < a.rows) {
                            tma_store_2d(&maps.out, sbuf, c, row);
                            tma_store_commit();
                        }
                    } else {
                        uint32_t rd[32], dg[16], du[16], h[16];
                        tmem_ld32(acc + 256 + half * 64 + g, rd);
                        tmem_ld_wait();
                        if (a.act == kActSilu) grad_cols<T, kActSilu>(rg, ru, rd, bias + g, bias + 64 + g, dg, du, h);
                        else if (a.act == kActGelu) grad_cols<T, kActGelu>(rg, ru, rd, bias + g, bias + 64 + g, dg, du, h);
                        else grad_cols<T, kActRelu>(rg, ru, rd, bias + g, bias + 64 + g, dg, du, h);
                        if (lane == 0) tma_store_wait_read<0>();
                        __syncwarp();
                        stage_row64(buf, lane, dg);
                        stage_row64(buf + 2048, lane, du);
                        stage_row64(buf + 4096, lane, h);
                        fence_async_shared();
                        __syncwarp();
                        if (lane == 0 && c < a.hidden && row < a.rows) {
#pragma unroll
                            for (int s = 0; s < 3; ++s) tma_store_3d(&maps.out, sbuf + 2048 * s, c, row, s);
                            tma_store_commit();
                        }
                    }
                } else {
                    uint32_t r[32];
                    tmem_ld32(acc + half * cols + g, r);
                    tmem_ld_wait();
                    if (KIND == XW && t.seg >= 0) {
                        if (lane == 0) tma_store_wait_read<0>();
                        __syncwarp();
#pragma unroll
                        for (int q = 0; q < 8; ++q)
                            *reinterpret_cast<uint4*>(buf + sw128_off(lane, q)) =
                                make_uint4(r[4 * q], r[4 * q + 1], r[4 * q + 2], r[4 * q + 3]);
                        fence_async_shared();
                        __syncwarp();
                        if (lane == 0 && c < a.dim && row < a.hidden) {
                            tma_add_3d(&maps.dw, sbuf, c, row, t.split * 3 + t.seg);
                            tma_store_commit();
                        }
                    } else {
                        if (KIND == DOWN) {
                            const bool in = row + lane < a.rows;
                            const T* res = static_cast<const T*>(a.residual) + (int64_t)(row + lane) * a.residual_stride + c;
#pragma unroll
                            for (int q = 0; q < 4; ++q) {
                                // dim is a multiple of 8: groups of 8 columns are inside or outside
                                uint4 v = make_uint4(0, 0, 0, 0);
                                if (a.residual && in && c + 8 * q < a.dim) v = *reinterpret_cast<const uint4*>(res + 8 * q);
                                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                                for (int j = 0; j < 4; ++j) {
                                    float f0, f1;
                                    unpack2<T>(w[j], f0, f1);
                                    const int i = 8 * q + 2 * j;
                                    r[i] = __float_as_uint(__uint_as_float(r[i]) + bias[g + i] + f0);
                                    r[i + 1] = __float_as_uint(__uint_as_float(r[i + 1]) + bias[g + i + 1] + f1);
                                }
                            }
                        }
                        uint32_t o[16];
#pragma unroll
                        for (int j = 0; j < 16; ++j) o[j] = pack2<T>(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1]));
                        if (lane == 0) tma_store_wait_read<0>();
                        __syncwarp();
                        stage_row64(buf, lane, o);
                        fence_async_shared();
                        __syncwarp();
                        if (lane == 0 && c < a.dim && row < a.rows) {
                            tma_store_2d(&maps.out, sbuf, c, row);
                            tma_store_commit();
                        }
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_peer(slot ? acc_empty1 : acc_empty0);
        }
        if (lane == 0) tma_store_wait0();
    }
    if (*abort && lane == 0) atomicOr(a.err, ERR_TIMEOUT);
    __syncwarp();
    tc_fence_before();
    cluster_sync();
    if (warp == 1) tmem_dealloc_pair(tmem, 512);
}

// ---- column sums (bias gradients) ----------------------------------------------------------------
// out[c] (+)= sum over rows of in[row][c], fp32: one CTA per 64 columns and row slice, 32 threads across
// column pairs, 8 down the rows; partial sums [slice][cols].
template <typename T>
__global__ void __launch_bounds__(256)
    col_sum_kernel(const T* in, int64_t stride, int rows, int cols, float* part, int first) {
    __shared__ float2 red[8][32];
    grid_dep_wait();
    const int lane = threadIdx.x & 31, k = threadIdx.x >> 5;
    const int c = blockIdx.x * 64 + 2 * lane;
    float s0 = 0.0f, s1 = 0.0f;
    if (c < cols)
        for (int r = blockIdx.y * 8 + k; r < rows; r += 8 * gridDim.y) {
            float a, b;
            unpack2<T>(*reinterpret_cast<const uint32_t*>(in + r * stride + c), a, b);
            s0 += a;
            s1 += b;
        }
    red[k][lane] = make_float2(s0, s1);
    __syncthreads();
    if (k == 0 && c < cols) {
        s0 = s1 = 0.0f;
        for (int i = 0; i < 8; ++i) {
            s0 += red[i][lane].x;
            s1 += red[i][lane].y;
        }
        float* p = part + (int64_t)blockIdx.y * cols + c;
        p[0] = first ? s0 : p[0] + s0;
        p[1] = first ? s1 : p[1] + s1;
    }
}
template <typename T>
__global__ void __launch_bounds__(256) col_fold_kernel(const float* part, int n_part, int cols, T* out) {
    grid_dep_wait();
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= cols) return;
    float s = 0.0f;
    for (int p = 0; p < n_part; ++p) s += part[(int64_t)p * cols + c];
    out[c] = from_f32<T>(s);
}

// dW from the splits' sums [split][3][hidden][dim]: 32 x 32 tiles, the third weight transposed.
template <typename T>
__global__ void __launch_bounds__(256)
    dw_fold_kernel(const float* part, int splits, int hidden, int dim, T* dwg, T* dwu, T* dwd) {
    __shared__ float tile[32][33];
    grid_dep_wait();
    const int seg = blockIdx.z, h0 = blockIdx.y * 32, d0 = blockIdx.x * 32, tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    T* out = seg == 0 ? dwg : seg == 1 ? dwu : dwd;
    if (!out) return;
    for (int i = ty; i < 32; i += 8) {
        const int h = h0 + i, d = d0 + tx;
        float s = 0.0f;
        if (h < hidden && d < dim) {
            for (int k = 0; k < splits; ++k) s += part[(((int64_t)k * 3 + seg) * hidden + h) * dim + d];
            if (seg < 2) out[(int64_t)h * dim + d] = from_f32<T>(s);
        }
        tile[i][tx] = s;
    }
    if (seg < 2) return;
    __syncthreads();
    for (int i = ty; i < 32; i += 8) {
        const int d = d0 + i, h = h0 + tx;
        if (h < hidden && d < dim) out[(int64_t)d * hidden + h] = from_f32<T>(tile[tx][i]);
    }
}

// ---- host ------------------------------------------------------------------------------------------

#define fail prism::set_error

inline cudaStream_t as_stream(void* s) { return reinterpret_cast<cudaStream_t>(s); }
int cuda_rc(cudaError_t e, const char* what) {
    return e == cudaSuccess ? PRISM_OK : fail(PRISM_E_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

PFN_cuTensorMapEncodeTiled_v12000 encode_tiled() {
    static const PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
    }();
    return fn;
}

// [planes][rows][cols] with `stride` elements a row; box {box_cols, box_rows, 1}
int make_map(CUtensorMap* m, const void* base, int dtype, int64_t cols, int64_t rows, int64_t planes, int64_t stride,
             int box_cols, int box_rows, CUtensorMapSwizzle swizzle) {
    auto fn = encode_tiled();
    if (!fn) return fail(PRISM_E_CUDA, "cuTensorMapEncodeTiled is not available");
    const int es = dtype_bytes(dtype);
    const CUtensorMapDataType type = dtype == PRISM_DTYPE_F16    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                     : dtype == PRISM_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                                 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32;
    cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)std::max<int64_t>(1, planes)};
    cuuint64_t strides[2] = {(cuuint64_t)(stride * es), (cuuint64_t)(stride * es * rows)};
    cuuint32_t box[3] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows, 1};
    cuuint32_t estr[3] = {1, 1, 1};
    CUresult r = fn(m, type, planes ? 3 : 2, const_cast<void*>(base), dims, strides, box, estr,
                    CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(PRISM_E_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
    return PRISM_OK;
}
constexpr CUtensorMapSwizzle kSw128 = CU_TENSOR_MAP_SWIZZLE_128B, kSw64 = CU_TENSOR_MAP_SWIZZLE_64B;

template <typename T, int KIND>
int launch(const prism_ctx* ctx, const Args& a, const Maps& m, cudaStream_t s, const char* who) {
    auto k = gated_kernel<T, KIND>;
    cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e != cudaSuccess) return cuda_rc(e, who);
    const int pairs = std::min(a.units, ctx->sm_count / 2);
    return cuda_rc(launch_pdl(k, dim3(2 * pairs), dim3(kThreads), kSmem, s, a, m), who);
}

// Rows that go through at a time: a row tile for every CTA pair.
int64_t chunk_rows(const prism_ctx* ctx, int64_t rows) { return std::min<int64_t>(rows, (int64_t)(ctx->sm_count / 2) * 256); }

inline int64_t up_to(int64_t n, int64_t m) { return (n + m - 1) / m * m; }

// scratch of the backward pass: p [3][rows][hidden] 16-bit, dw [splits][3][hidden][dim] fp32, column sums
struct BackPlan {
    int64_t chunk;
    int splits, slices;
    size_t p_bytes, dw_bytes, sum_bytes;
    size_t total() const { return p_bytes + dw_bytes + sum_bytes; }
};
BackPlan back_plan(const prism_ctx* ctx, const prism_gated_params* p) {
    BackPlan b;
    b.chunk = chunk_rows(ctx, p->rows);
    const int bn = p->dim <= 128 ? 128 : 256;
    const int64_t tiles = 3 * ((p->hidden + 255) / 256) * (int64_t)((p->dim + bn - 1) / bn);
    const int64_t kb = (b.chunk + 63) / 64;
    b.splits = (int)std::max<int64_t>(1, std::min<int64_t>(kb, (ctx->sm_count / 2) / tiles));
    b.slices = (int)std::max<int64_t>(1, std::min<int64_t>(64, b.chunk / 64));
    b.p_bytes = (size_t)up_to(3 * b.chunk * p->hidden * 2, 1024);
    b.dw_bytes = (size_t)up_to((int64_t)b.splits * 3 * p->hidden * p->dim * 4, 1024);
    b.sum_bytes = (size_t)b.slices * (2 * (size_t)p->hidden + p->dim) * 4;
    return b;
}

int check_gated(const char* who, const prism_gated_params* p) {
    if (p->dtype != PRISM_DTYPE_F16 && p->dtype != PRISM_DTYPE_BF16)
        return fail(dtype_known(p->dtype) ? PRISM_E_UNSUPPORTED : PRISM_E_ARG, "%s: dtype %d (fp16 or bf16)", who, p->dtype);
    if (p->activation < PRISM_ACT_GELU || p->activation > PRISM_ACT_RELU)
        return fail(PRISM_E_ARG, "%s: activation %d", who, p->activation);
    if (p->rows < 0 || p->dim <= 0 || p->hidden <= 0)
        return fail(PRISM_E_ARG, "%s: rows %lld, dim %d, hidden %d", who, (long long)p->rows, p->dim, p->hidden);
    if (p->dim % 8 || p->hidden % 8)
        return fail(PRISM_E_UNSUPPORTED, "%s: dim %d and hidden %d have to be multiples of 8", who, p->dim, p->hidden);
    if (p->dim > 16384 || p->hidden > 65536)
        return fail(PRISM_E_UNSUPPORTED, "%s: dim %d above 16384 or hidden %d above 65536", who, p->dim, p->hidden);
    if (p->rows > (int64_t)1 << 40) return fail(PRISM_E_RANGE, "%s: rows %lld", who, (long long)p->rows);
    return PRISM_OK;
}
// rows that TMA or 16-byte accesses reach: base and stride in 16 bytes
int check_rows(const char* who, const char* name, const void* t, int64_t stride, int64_t rows, int dim) {
    if (!t) return PRISM_OK;
    if (rows > 1 && stride < dim) return fail(PRISM_E_ARG, "%s: %s_stride %lld below dim %d", who, name, (long long)stride, dim);
    if (((uintptr_t)t & 15) || (rows > 1 && stride % 8))
        return fail(PRISM_E_ALIGN, "%s: %s and its stride have to be multiples of 16 bytes", who, name);
    if (rows > 1 && stride > (int64_t)1 << 36) return fail(PRISM_E_RANGE, "%s: %s_stride %lld", who, name, (long long)stride);
    return PRISM_OK;
}
int check_weight(const char* who, const char* name, const void* t, bool needed, int align = 16) {
    if (!t) return needed ? fail(PRISM_E_ARG, "%s: %s is NULL", who, name) : PRISM_OK;
    if ((uintptr_t)t % align) return fail(PRISM_E_ALIGN, "%s: %s is not %d-byte aligned", who, name, align);
    return PRISM_OK;
}
int64_t row_stride(int64_t stride, int64_t rows, int dim) { return rows > 1 ? stride : dim; }

template <typename T>
int forward(const prism_ctx* ctx, const prism_gated_params* p, const prism_gated_weights* w, const void* x,
            const void* residual, void* y, void* ws, cudaStream_t s) {
    const char* who = "prism_gated_ffn";
    const int64_t chunk = chunk_rows(ctx, p->rows);
    const int64_t xs = row_stride(p->x_stride, p->rows, p->dim), ys = row_stride(p->y_stride, p->rows, p->dim);
    const int64_t rs = row_stride(p->residual_stride, p->rows, p->dim);
    int rc;
    for (int64_t r0 = 0; r0 < p->rows; r0 += chunk) {
        const int rows = (int)std::min(chunk, p->rows - r0);
        const T* xc = static_cast<const T*>(x) + r0 * xs;
        T* yc = static_cast<T*>(y) + r0 * ys;
        Args a = {};
        a.rows = rows;
        a.dim = p->dim;
        a.hidden = p->hidden;
        a.act = p->activation;
        a.b_gate = w->b_gate;
        a.b_up = w->b_up;
        a.b_down = w->b_down;
        a.residual = residual ? static_cast<const T*>(residual) + r0 * rs : nullptr;
        a.residual_stride = rs;
        a.err = ctx->err;
        a.bn = p->dim <= 128 ? 128 : 256;
        a.m_tiles = (rows + 255) / 256;
        a.n_tiles = (p->hidden + 127) / 128;
        a.units = a.m_tiles * a.n_tiles;
        Maps m;
        if ((rc = make_map(&m.a0, xc, p->dtype, p->dim, rows, 0, xs, 64, 128, kSw128)) ||
            (rc = make_map(&m.b0, w->w_gate, p->dtype, p->dim, p->hidden, 0, p->dim, 64, 128, kSw128)) ||
            (rc = make_map(&m.b1, w->w_up, p->dtype, p->dim, p->hidden, 0, p->dim, 64, 128, kSw128)) ||
            (rc = make_map(&m.out, ws, p->dtype, p->hidden, rows, 0, p->hidden, 32, 32, kSw64)) ||
            (rc = launch<T, UP>(ctx, a, m, s, who)))
            return rc;
        a.n_tiles = (p->dim + a.bn - 1) / a.bn;
        a.units = a.m_tiles * a.n_tiles;
        if ((rc = make_map(&m.a0, ws, p->dtype, p->hidden, rows, 0, p->hidden, 64, 128, kSw128)) ||
            (rc = make_map(&m.b0, w->w_down, p->dtype, p->hidden, p->dim, 0, p->hidden, 64, a.bn / 2, kSw128)) ||
            (rc = make_map(&m.out, yc, p->dtype, p->dim, rows, 0, ys, 32, 32, kSw64)) ||
            (rc = launch<T, DOWN>(ctx, a, m, s, who)))
            return rc;
    }
    return PRISM_OK;
}

template <typename T>
int backward(const prism_ctx* ctx, const prism_gated_params* p, const prism_gated_weights* w, const void* x, const void* dy,
             void* dx, const prism_gated_grads* d, void* ws, cudaStream_t s) {
    const char* who = "prism_gated_ffn_backward";
    const BackPlan b = back_plan(ctx, p);
    const int64_t xs = row_stride(p->x_stride, p->rows, p->dim), dys = row_stride(p->dy_stride, p->rows, p->dim);
    const int64_t dxs = row_stride(p->dx_stride, p->rows, p->dim);
    T* pbuf = static_cast<T*>(ws);
    float* dw = reinterpret_cast<float*>(static_cast<char*>(ws) + b.p_bytes);
    float* sum_h = reinterpret_cast<float*>(static_cast<char*>(ws) + b.p_bytes + b.dw_bytes);
    float* sum_d = sum_h + (size_t)b.slices * 2 * p->hidden;
    int rc;
    if ((rc = cuda_rc(cudaMemsetAsync(dw, 0, b.dw_bytes, s), who))) return rc;
    for (int64_t r0 = 0; r0 < p->rows; r0 += b.chunk) {
        const int rows = (int)std::min(b.chunk, p->rows - r0);
        const T* xc = static_cast<const T*>(x) + r0 * xs;
        const T* dyc = static_cast<const T*>(dy) + r0 * dys;
        Args a = {};
        a.rows = rows;
        a.dim = p->dim;
        a.hidden = p->hidden;
        a.act = p->activation;
        a.b_gate = w->b_gate;
        a.b_up = w->b_up;
        a.err = ctx->err;
        a.bn = p->dim <= 128 ? 128 : 256;
        a.m_tiles = (rows + 255) / 256;
        a.n_tiles = (p->hidden + 127) / 128;
        a.units = a.m_tiles * a.n_tiles;
        Maps m;
        if ((rc = make_map(&m.a0, xc, p->dtype, p->dim, rows, 0, xs, 64, 128, kSw128)) ||
            (rc = make_map(&m.a1, dyc, p->dtype, p->dim, rows, 0, dys, 64, 128, kSw128)) ||
            (rc = make_map(&m.b0, w->w_gate, p->dtype, p->dim, p->hidden, 0, p->dim, 64, 128, kSw128)) ||
            (rc = make_map(&m.b1, w->w_up, p->dtype, p->dim, p->hidden, 0, p->dim, 64, 128, kSw128)) ||
            (rc = make_map(&m.b2, w->w_down, p->dtype, p->hidden, p->dim, 0, p->hidden, 64, 64, kSw128)) ||
            (rc = make_map(&m.out, pbuf, p->dtype, p->hidden, rows, 3, p->hidden, 32, 32, kSw64)) ||
            (rc = launch<T, BACK>(ctx, a, m, s, who)))
            return rc;
        // column sums of dg and du (one after the other in pbuf) and of dy
        const dim3 gh((p->hidden + 63) / 64, b.slices), gd((p->dim + 63) / 64, b.slices);
        for (int k = 0; k < 2; ++k)
            if (k ? d->db_up : d->db_gate)
                if ((rc = cuda_rc(launch_pdl(col_sum_kernel<T>, gh, dim3(256), 0, s, (const T*)(pbuf + (int64_t)k * rows * p->hidden),
                                             (int64_t)p->hidden, rows, p->hidden, sum_h + (size_t)k * b.slices * p->hidden,
                                             (int)(r0 == 0)), who)))
                    return rc;
        if (d->db_down && (rc = cuda_rc(launch_pdl(col_sum_kernel<T>, gd, dim3(256), 0, s, dyc, dys, rows, p->dim, sum_d,
                                                   (int)(r0 == 0)), who)))
            return rc;
        a.n_tiles = (p->dim + a.bn - 1) / a.bn;
        a.x_units = a.m_tiles * a.n_tiles;
        a.w_tiles = (p->hidden + 255) / 256;
        a.k_all = (rows + 63) / 64;
        a.k_per = (a.k_all + b.splits - 1) / b.splits;
        const int splits = (a.k_all + a.k_per - 1) / a.k_per;
        a.units = a.x_units + 3 * a.w_tiles * a.n_tiles * splits;
        if ((rc = make_map(&m.p_k, pbuf, p->dtype, p->hidden, rows, 3, p->hidden, 64, 128, kSw128)) ||
            (rc = make_map(&m.p_mn, pbuf, p->dtype, p->hidden, rows, 3, p->hidden, 64, 64, kSw128)) ||
            (rc = make_map(&m.b0, w->w_gate, p->dtype, p->dim, p->hidden, 0, p->dim, 64, 64, kSw128)) ||
            (rc = make_map(&m.b1, w->w_up, p->dtype, p->dim, p->hidden, 0, p->dim, 64, 64, kSw128)) ||
            (rc = make_map(&m.x_mn, xc, p->dtype, p->dim, rows, 0, xs, 64, 64, kSw128)) ||
            (rc = make_map(&m.dy_mn, dyc, p->dtype, p->dim, rows, 0, dys, 64, 64, kSw128)) ||
            (rc = make_map(&m.out, static_cast<T*>(dx) + r0 * dxs, p->dtype, p->dim, rows, 0, dxs, 32, 32, kSw64)) ||
            (rc = make_map(&m.dw, dw, PRISM_DTYPE_F32, p->dim, p->hidden, 3 * (int64_t)b.splits, p->dim, 32, 32, kSw128)) ||
            (rc = launch<T, XW>(ctx, a, m, s, who)))
            return rc;
    }
    if ((rc = cuda_rc(launch_pdl(dw_fold_kernel<T>, dim3((p->dim + 31) / 32, (p->hidden + 31) / 32, 3), dim3(256), 0, s,
                                 (const float*)dw, b.splits, p->hidden, p->dim, static_cast<T*>(d->dw_gate),
                                 static_cast<T*>(d->dw_up), static_cast<T*>(d->dw_down)), who)))
        return rc;
    const struct { void* out; const float* part; int cols; } sums[3] = {
        {d->db_gate, sum_h, p->hidden}, {d->db_up, sum_h + (size_t)b.slices * p->hidden, p->hidden}, {d->db_down, sum_d, p->dim}};
    for (const auto& f : sums)
        if (f.out && (rc = cuda_rc(launch_pdl(col_fold_kernel<T>, dim3((f.cols + 255) / 256), dim3(256), 0, s, f.part, b.slices,
                                              f.cols, static_cast<T*>(f.out)), who)))
            return rc;
    return PRISM_OK;
}

}  // namespace
}  // namespace prism

using namespace prism;

extern "C" int prism_gated_ffn_workspace(prism_ctx* ctx, const prism_gated_params* p, int backward, size_t* bytes) {
    if (!ctx || !p || !bytes) return fail(PRISM_E_ARG, "prism_gated_ffn_workspace: NULL argument");
    int rc = check_gated("prism_gated_ffn_workspace", p);
    if (rc) return rc;
    *bytes = p->rows == 0 ? 0 : backward ? back_plan(ctx, p).total() : (size_t)chunk_rows(ctx, p->rows) * p->hidden * 2;
    return PRISM_OK;
}

static int check_workspace(const char* who, prism_ctx* ctx, const prism_gated_params* p, int backward, void* ws, size_t bytes) {
    size_t need = 0;
    int rc = prism_gated_ffn_workspace(ctx, p, backward, &need);
    if (rc) return rc;
    if (need && (!ws || bytes < need))
        return fail(PRISM_E_ARG, "%s: workspace of %zu bytes, %zu needed", who, ws ? bytes : (size_t)0, need);
    if ((uintptr_t)ws & 15) return fail(PRISM_E_ALIGN, "%s: workspace is not 16-byte aligned", who);
    return PRISM_OK;
}

extern "C" int prism_gated_ffn(prism_ctx* ctx, const prism_gated_params* p, const prism_gated_weights* w, const void* x,
                               const void* residual, void* y, void* workspace, size_t workspace_bytes, void* stream) {
    const char* who = "prism_gated_ffn";
    if (!ctx || !p || !w) return fail(PRISM_E_ARG, "%s: NULL argument", who);
    int rc = check_gated(who, p);
    if (rc || p->rows == 0) return rc;
    if (!x || !y) return fail(PRISM_E_ARG, "%s: NULL argument", who);
    if ((rc = check_rows(who, "x", x, p->x_stride, p->rows, p->dim)) ||
        (rc = check_rows(who, "residual", residual, p->residual_stride, p->rows, p->dim)) ||
        (rc = check_rows(who, "y", y, p->y_stride, p->rows, p->dim)) || (rc = check_weight(who, "w_gate", w->w_gate, true)) ||
        (rc = check_weight(who, "w_up", w->w_up, true)) || (rc = check_weight(who, "w_down", w->w_down, true)) ||
        (rc = check_weight(who, "b_gate", w->b_gate, false, 2)) || (rc = check_weight(who, "b_up", w->b_up, false, 2)) ||
        (rc = check_weight(who, "b_down", w->b_down, false, 2)) ||
        (rc = check_workspace(who, ctx, p, 0, workspace, workspace_bytes)))
        return rc;
    const int64_t ys = row_stride(p->y_stride, p->rows, p->dim), xs = row_stride(p->x_stride, p->rows, p->dim);
    const int64_t rs = row_stride(p->residual_stride, p->rows, p->dim);
    if (rows_overlap(y, ys, x, xs, p->rows, p->dim, 2) ||
        (!(y == residual && ys == rs) && rows_overlap(y, ys, residual, rs, p->rows, p->dim, 2)))
        return fail(PRISM_E_ARG, "%s: y overlaps an input", who);
    DeviceGuard g(ctx->device);
    return p->dtype == PRISM_DTYPE_F16 ? forward<__half>(ctx, p, w, x, residual, y, workspace, as_stream(stream))
                                       : forward<__nv_bfloat16>(ctx, p, w, x, residual, y, workspace, as_stream(stream));
}

extern "C" int prism_gated_ffn_backward(prism_ctx* ctx, const prism_gated_params* p, const prism_gated_weights* w,
                                        const void* x, const void* dy, void* dx, const prism_gated_grads* d, void* workspace,
                                        size_t workspace_bytes, void* stream) {
    const char* who = "prism_gated_ffn_backward";
    if (!ctx || !p || !w || !d) return fail(PRISM_E_ARG, "%s: NULL argument", who);
    int rc = check_gated(who, p);
    if (rc) return rc;
    if ((rc = check_weight(who, "dw_gate", d->dw_gate, false, 2)) || (rc = check_weight(who, "dw_up", d->dw_up, false, 2)) ||
        (rc = check_weight(who, "dw_down", d->dw_down, false, 2)) || (rc = check_weight(who, "db_gate", d->db_gate, false, 2)) ||
        (rc = check_weight(who, "db_up", d->db_up, false, 2)) || (rc = check_weight(who, "db_down", d->db_down, false, 2)))
        return rc;
    DeviceGuard g(ctx->device);
    cudaStream_t s = as_stream(stream);
    if (p->rows == 0) {  // no rows: the sums are zero
        const size_t nw = (size_t)p->hidden * p->dim * 2;
        const struct { void* t; size_t n; } all[6] = {{d->dw_gate, nw}, {d->dw_up, nw}, {d->dw_down, nw},
                                                      {d->db_gate, (size_t)p->hidden * 2}, {d->db_up, (size_t)p->hidden * 2},
                                                      {d->db_down, (size_t)p->dim * 2}};
        for (const auto& t : all)
            if (t.t && (rc = cuda_rc(cudaMemsetAsync(t.t, 0, t.n, s), who))) return rc;
        return PRISM_OK;
    }
    if (!x || !dy || !dx) return fail(PRISM_E_ARG, "%s: NULL argument", who);
    if ((rc = check_rows(who, "x", x, p->x_stride, p->rows, p->dim)) || (rc = check_rows(who, "dy", dy, p->dy_stride, p->rows, p->dim)) ||
        (rc = check_rows(who, "dx", dx, p->dx_stride, p->rows, p->dim)) || (rc = check_weight(who, "w_gate", w->w_gate, true)) ||
        (rc = check_weight(who, "w_up", w->w_up, true)) || (rc = check_weight(who, "w_down", w->w_down, true)) ||
        (rc = check_weight(who, "b_gate", w->b_gate, false, 2)) || (rc = check_weight(who, "b_up", w->b_up, false, 2)) ||
        (rc = check_workspace(who, ctx, p, 1, workspace, workspace_bytes)))
        return rc;
    const int64_t xs = row_stride(p->x_stride, p->rows, p->dim), dys = row_stride(p->dy_stride, p->rows, p->dim);
    const int64_t dxs = row_stride(p->dx_stride, p->rows, p->dim);
    if (rows_overlap(dx, dxs, x, xs, p->rows, p->dim, 2) || rows_overlap(dx, dxs, dy, dys, p->rows, p->dim, 2))
        return fail(PRISM_E_ARG, "%s: dx overlaps an input", who);
    return p->dtype == PRISM_DTYPE_F16 ? backward<__half>(ctx, p, w, x, dy, dx, d, workspace, s)
                                       : backward<__nv_bfloat16>(ctx, p, w, x, dy, dx, d, workspace, s);
}
