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
//   BACK  dh = dy Wd and [g | u] again from x -> dg, du, h, and the bias gradients' sums on the way
//   XW    dx tiles and dW tiles (split over rows) in one launch: neither fills the GPU alone
// Rows go through in chunks, so the scratch memory stays bounded.
#include <algorithm>

#include "gated_fused.cuh"
#include "gated_small.cuh"
#include "tensor_map.cuh"

namespace prism {
namespace {

enum Kind : int { UP, DOWN, BACK, XW };

constexpr int kStageA = 16384, kStageB = 16384, kStage = kStageA + kStageB;
constexpr int kOut = 4096;  // a warp's store staging: two 32 x 32 16-bit boxes or one of fp32
// Epilogue warps and operand stages.  BACK's epilogue works out some 20 instructions a value between
// its TMEM loads: 16 warps hide what 8 could not (13,000 cycles a unit against some 3100 of MMAs).
template <int KIND>
struct Cfg {
    static constexpr int kEpiWarps = KIND == BACK ? 16 : 8;
    static constexpr int kThreads = 32 * (2 + kEpiWarps);
    static constexpr int kStages = KIND == BACK ? 4 : 5;
    static constexpr int kBias = KIND == BACK ? 256 : 512;  // bytes a warp
    static constexpr int kSmem = kStages * kStage + kEpiWarps * (kOut + kBias) + 512 + 1024;
};
constexpr int kMaxStages = 5;

struct Bars {
    uint64_t full[kMaxStages], empty[kMaxStages], acc_full[2], acc_empty[2];
    uint32_t tmem_base;
    int abort;
};

struct Maps {
    CUtensorMap a0, a1, b0, b1, b2, out, p_k, p_mn, x_mn, dy_mn, dw;
};

struct Args {
    int rows, dim, hidden;      // rows of this chunk
    int m_tiles, n_tiles;       // 256-row tiles; column tiles (128 hidden for UP / BACK, bn else)
    int bn;                     // N of an output tile over dim: 256 (128: XW's dW tiles where dim <= 128)
    int units, x_units;         // XW: the first x_units are dx tiles, the others dW tiles
    int w_each[2];              // XW: dW tiles a pair takes, where it has one dx tile more than the others [1] or not
    int w_tiles, k_per, k_all;  // XW: 256-row tiles of one weight's hidden axis; row blocks a split, in all
    int act;
    int first;                  // the first chunk: sums over rows start here
    float *sums, *sums_dy;      // column sums of dg and du (BACK) and of dy (XW): [CTAs][4][2 hidden], [splits][16][dim]
    const void* dy;             // XW: rows for the sums
    int64_t dy_stride;
    const void *b_gate, *b_up, *b_down;
    const void* residual;
    int64_t residual_stride;
    uint32_t* err;
};

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

// The units of a pair, the same on every role: every pairs-th one.  XW's dW tiles go round the pairs w_each[1]
// times, then round those that have a dx tile less up to w_each[0] times (the two differ in depth: 2051
// rows of 1000 x 2744 in plain turns left the last pairs idle a third of the time, 140 against 128 us).
// Turns, not runs, so that pairs work on neighbouring tiles at a time and share their operands in L2.
template <int KIND>
struct Walk {
    int pair, pairs, n, n_x, x_units, more, w_all;
    PRISM_DEV static int turns(int units, int first, int step) { return units > first ? (units - first + step - 1) / step : 0; }
    PRISM_DEV Walk(const Args& a, int pair_, int pairs_) : pair(pair_), pairs(pairs_), x_units(a.x_units) {
        n = n_x = turns(KIND == XW ? a.x_units : a.units, pair, pairs);
        if (KIND == XW) {
            const int n_w = a.units - a.x_units;
            more = a.x_units % pairs;  // pairs with a dx tile more come first
            w_all = a.w_each[1];
            n += min(w_all, turns(n_w, pair, pairs));
            if (pair >= more) n += min(a.w_each[0] - w_all, turns(n_w - w_all * pairs, pair - more, pairs - more));
        }
    }
    PRISM_DEV int unit(int i) const {
        if (KIND != XW || i < n_x) return pair + i * pairs;
        i -= n_x;
        return x_units + (i < w_all ? i * pairs + pair : w_all * pairs + (i - w_all) * (pairs - more) + pair - more);
    }
};

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
template <typename T, int KIND>
__global__ void __launch_bounds__(Cfg<KIND>::kThreads, 1) __cluster_dims__(2, 1, 1)
    gated_kernel(const Args a, const __grid_constant__ Maps maps) {
    constexpr int kStages = Cfg<KIND>::kStages, kEpiWarps = Cfg<KIND>::kEpiWarps;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = smem_align1k(smem_raw);
    unsigned char* s_out = smem + kStages * kStage;
    unsigned char* s_bias = s_out + kEpiWarps * kOut;
    Bars* bars = reinterpret_cast<Bars*>(s_bias + kEpiWarps * Cfg<KIND>::kBias);
    volatile int* abort = &bars->abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)cluster_rank(), pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    // Accumulators: two of 256 columns.  BACK has [g | u] in columns 0 .. 255 and dh in one of two slots
    // of 128 behind them, so that a unit's dh is computed while the epilogue still reads the unit before.
    constexpr int slots = KIND == BACK ? 1 : 2;
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
    const Walk<KIND> walk(a, pair, pairs);
    grid_dep_wait();

    if (warp == 0) {
        // ---- producer (both CTAs): this CTA's rows of A, its half of B, all on the leader's barrier
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int i = 0; i < walk.n && ok; ++i) {
            const Unit t = unit_of<KIND>(a, walk.unit(i));
            const int kd = (a.dim + 63) / 64, kh = (a.hidden + 63) / 64;
            const int bh = a.bn / 2;  // this CTA's share of an N tile over dim
            for (int kb = 0; kb < t.nkb; ++kb) {
                if (!mbar_wait_w(&bars->empty[stage], phase ^ 1, abort)) { ok = false; break; }
                if (lane == 0) {
                    const uint32_t sa = smem_u32(smem + stage * kStage), sb = sa + kStageA;
                    const uint32_t bar = peer_addr(smem_u32(&bars->full[stage]), 0);
                    uint32_t bytes;
                    const int row = t.mt * 256 + rank * 128;
                    if (KIND == UP || (KIND == BACK && kb >= kd)) {
                        const int k = (KIND == BACK ? kb - kd : kb) * 64;
                        bytes = kStageA + kStageB;
                        if (rank == 0) mbar_expect_tx(&bars->full[stage], 2 * bytes);
                        tma_load_2d_pair(sa, &maps.a0, bar, k, row);
                        tma_load_2d_pair(sb, rank ? &maps.b1 : &maps.b0, bar, k, t.nt * 128);
                    } else if (KIND == BACK) {
                        bytes = kStageA + kStageB / 2;
                        if (rank == 0) mbar_expect_tx(&bars->full[stage], 2 * bytes);
                        tma_load_2d_pair(sa, &maps.a1, bar, kb * 64, row);
                        tma_load_2d_pair(sb, &maps.b2, bar, t.nt * 128 + rank * 64, kb * 64);
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
            const uint32_t id_k = idesc_pair(256, KIND == DOWN ? a.bn : 256, bf16, 0, 0);        // both K-major
            const uint32_t id_x = idesc_pair(256, KIND == BACK ? 128 : a.bn, bf16, 0, 1), id_w = idesc_pair(256, a.bn, bf16, 1, 1);
            for (; it < walk.n && ok; ++it) {
                const Unit t = unit_of<KIND>(a, walk.unit(it));
                const int slot = it % slots;
                const uint32_t acc = tmem + slot * 256;
                if (KIND != BACK) {
                    ok = mbar_wait_w(&bars->acc_empty[slot], ((it / slots) & 1) ^ 1, abort);
                    if (!ok) break;
                    tc_fence_after();
                }
                const int kd = (a.dim + 63) / 64;
                for (int kb = 0; kb < t.nkb; ++kb) {
                    if (KIND == BACK && kb == kd) {  // dh is on its way; g and u need the last unit's read
                        ok = mbar_wait_w(&bars->acc_empty[0], (it & 1) ^ 1, abort);
                        if (!ok) break;
                        tc_fence_after();
                    }
                    if (!mbar_wait_w(&bars->full[stage], phase, abort)) { ok = false; break; }
                    tc_fence_after();
                    const uint32_t sa = smem_u32(smem + stage * kStage), sb = sa + kStageA;
                    if (KIND == XW && t.seg >= 0)
                        mma_pair_x4<128, 128>(acc, desc_lo(sa, 8192), kDescHi128, desc_lo(sb, 8192), kDescHi128, id_w, kb);
                    else if (KIND == XW)
                        mma_pair_x4<2, 128>(acc, desc_lo(sa), kDescHi128, desc_lo(sb, 8192), kDescHi128, id_x, kb);
                    else if (KIND == BACK && kb < kd)
                        mma_pair_x4<2, 128>(acc + 256 + (it & 1) * 128, desc_lo(sa), kDescHi128, desc_lo(sb, 8192), kDescHi128, id_x, kb);
                    else
                        mma_pair_x4<2, 2>(acc, desc_lo(sa), kDescHi128, desc_lo(sb), kDescHi128, id_k, KIND == BACK ? kb - kd : kb);
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
        // (a quarter in BACK)
        const int quad = warp & 3, half = (warp - 2) >> 2;
        unsigned char* buf = s_out + (warp - 2) * kOut;
        const uint32_t sbuf = smem_u32(buf);
        float* bias = reinterpret_cast<float*>(s_bias + (warp - 2) * Cfg<KIND>::kBias);
        const uint32_t lane_addr = (uint32_t)(quad * 32) << 16;
        const uint32_t acc_empty0 = peer_addr(smem_u32(&bars->acc_empty[0]), 0);
        const uint32_t acc_empty1 = peer_addr(smem_u32(&bars->acc_empty[1]), 0);
        // BACK: column sums of this warp's rows of dg and du.  Each warp has columns of its own.
        float* sums = KIND == BACK ? a.sums + ((int64_t)blockIdx.x * 4 + quad) * (2 * a.hidden) : nullptr;
        float next_g = 0.0f, next_u = 0.0f;  // BACK: the next unit's biases of column `lane`
        if (KIND == BACK) {
            if (a.first) {
                for (int c = lane; c < a.hidden; c += 32)
                    if (((c >> 5) & 3) == half) sums[c] = sums[a.hidden + c] = 0.0f;
            }
            const int c = pair % a.n_tiles * 128 + half * 32 + lane;
            next_g = ld_bias<T>(a.b_gate, c, a.hidden);
            next_u = ld_bias<T>(a.b_up, c, a.hidden);
        }
        __syncwarp();
        int it = 0;
        for (; it < walk.n; ++it) {
            const Unit t = unit_of<KIND>(a, walk.unit(it));
            const int slot = it % slots;
            const int row = t.mt * 256 + rank * 128 + quad * 32;
            const int cols = KIND == BACK ? 32 : KIND == UP ? 64 : a.bn / 2;  // this warp's
            const int col0 = (KIND == BACK || KIND == UP ? t.nt * 128 : t.nt * a.bn) + half * cols;
            // biases of this warp's columns
            if (KIND == BACK) {
                __syncwarp();
                bias[lane] = next_g;
                bias[32 + lane] = next_u;
                const int c = walk.unit(it + 1) % a.n_tiles * 128 + half * 32 + lane;
                if (it + 1 < walk.n) {
                    next_g = ld_bias<T>(a.b_gate, c, a.hidden);
                    next_u = ld_bias<T>(a.b_up, c, a.hidden);
                }
            } else if (KIND == UP) {
                for (int i = lane; i < 64; i += 32) {
                    bias[i] = ld_bias<T>(a.b_gate, col0 + i, a.hidden);
                    bias[64 + i] = ld_bias<T>(a.b_up, col0 + i, a.hidden);
                }
            } else if (KIND == DOWN) {
                for (int i = lane; i < cols; i += 32) bias[i] = ld_bias<T>(a.b_down, col0 + i, a.dim);
            }
            if (KIND == XW && a.sums_dy && t.seg == 2 && t.mt == 0) {
                // dy's column sums over the split's rows while the products over the same rows run (and bring them to
                // L2): every 16th row a warp, 8 columns a lane
                const int c = t.nt * a.bn + 8 * lane, r1 = min(a.rows, (t.k0 + t.nkb) * 64);
                if (8 * lane < a.bn && c < a.dim) {
                    const T* dy = static_cast<const T*>(a.dy) + c;
                    float s[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
                    const int w = rank * kEpiWarps + warp - 2;
                    for (int r = t.k0 * 64 + w; r < r1; r += 16 * 8) {
                        uint4 v[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            v[i] = r + 16 * i < r1 ? *reinterpret_cast<const uint4*>(dy + (int64_t)(r + 16 * i) * a.dy_stride)
                                                   : make_uint4(0, 0, 0, 0);
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const uint32_t q[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                float f0, f1;
                                unpack2<T>(q[j], f0, f1);
                                s[2 * j] += f0;
                                s[2 * j + 1] += f1;
                            }
                        }
                    }
                    float4* out = reinterpret_cast<float4*>(a.sums_dy + ((int64_t)t.split * 16 + w) * a.dim + c);
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        float4 o = make_float4(s[4 * j], s[4 * j + 1], s[4 * j + 2], s[4 * j + 3]);
                        if (!a.first) {
                            const float4 p = out[j];
                            o.x += p.x, o.y += p.y, o.z += p.z, o.w += p.w;
                        }
                        out[j] = o;
                    }
                }
            }
            __syncwarp();
            const bool got = mbar_wait_w(&bars->acc_full[slot], (it / slots) & 1, abort);
            if (!got) break;
            tc_fence_after();
            const uint32_t acc = tmem + lane_addr + slot * 256;
            if (KIND == BACK) {
                uint32_t h[16];
                if (lane == 0) tma_store_wait_read<0>();
                __syncwarp();
#pragma unroll
                for (int g = 0; g < 32; g += 16) {
                    uint32_t rg[16], ru[16], rd[16];
                    uint64_t dg[8], du[8];
                    tmem_ld16(acc + half * 32 + g, rg);
                    tmem_ld16(acc + 128 + half * 32 + g, ru);
                    tmem_ld16(acc + 256 + (it & 1) * 128 + half * 32 + g, rd);
                    tmem_ld_wait();
                    if (g) {  // everything read: the next unit's products may come
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive_pair(acc_empty0);
                    }
                    if (a.act == kActSilu) grad_cols<T, kActSilu>(rg, ru, rd, bias + g, bias + 32 + g, dg, du, h + g / 2);
                    else if (a.act == kActGelu) grad_cols<T, kActGelu>(rg, ru, rd, bias + g, bias + 32 + g, dg, du, h + g / 2);
                    else grad_cols<T, kActRelu>(rg, ru, rd, bias + g, bias + 32 + g, dg, du, h + g / 2);
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        *reinterpret_cast<uint4*>(buf + sw64_off(lane, g / 8 + q)) = pack8<T>(dg + 4 * q);
                        *reinterpret_cast<uint4*>(buf + 2048 + sw64_off(lane, g / 8 + q)) = pack8<T>(du + 4 * q);
                    }
                    // one warp adds to an address, in the order of its units: the same bits every time
                    const float sg = column_sum(dg, lane), su = column_sum(du, lane);
                    const int c = col0 + g + (lane >> 1);
                    if (c < a.hidden) atomicAdd(sums + (lane & 1 ? a.hidden : 0) + c, lane & 1 ? su : sg);
                }
                const bool store = lane == 0 && col0 < a.hidden && row < a.rows;
                fence_async_shared();
                __syncwarp();
                if (store) {
                    tma_store_3d(&maps.out, sbuf, col0, row, 0);
                    tma_store_3d(&maps.out, sbuf + 2048, col0, row, 1);
                    tma_store_commit();
                    tma_store_wait_read<0>();
                }
                __syncwarp();
                stage_row64(buf, lane, h);
                fence_async_shared();
                __syncwarp();
                if (store) {
                    tma_store_3d(&maps.out, sbuf, col0, row, 2);
                    tma_store_commit();
                }
                continue;
            }
            for (int g = 0; g < cols; g += 32) {
                const int c = col0 + g;
                if (KIND == UP) {
                    uint32_t rg[32], ru[32], o[16];
                    tmem_ld32(acc + half * 64 + g, rg);
                    tmem_ld32(acc + 128 + half * 64 + g, ru);
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
                            // one add to an address and launch: the same order, the same bits every time
                            if (a.first) tma_store_3d(&maps.dw, sbuf, c, row, t.split * 3 + t.seg);
                            else tma_add_3d(&maps.dw, sbuf, c, row, t.split * 3 + t.seg);
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
            if (lane == 0) mbar_arrive_pair(slot ? acc_empty1 : acc_empty0);
        }
        if (lane == 0) tma_store_wait0();
    }
    if (*abort && lane == 0) atomicOr(a.err, ERR_TIMEOUT);
    __syncwarp();
    tc_fence_before();
    cluster_sync();
    if (warp == 1) tmem_dealloc_pair(tmem, 512);
}

// ---- joining the partial sums ------------------------------------------------------------------
// dW from the splits' sums [split][3][hidden][dim] by 32 x 32 tiles, four columns a thread, the third
// weight transposed; behind those CTAs, db from the warps' column sums [n_sums][2 hidden] and
// [n_dy][dim], 32 columns a CTA: 32 threads deep, each over every 32nd row, then the 32 in order.  Bound
// by latency: single loads 8 deep took 45 us for 592 rows of sums, this 12.
PRISM_DEV float4 operator+(const float4& a, const float4& b) { return make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w); }
template <typename T>
PRISM_DEV void store4(T* out, const float4& v) { *reinterpret_cast<uint2*>(out) = make_uint2(pack2<T>(v.x, v.y), pack2<T>(v.z, v.w)); }

template <typename T>
__global__ void __launch_bounds__(256)
    fold_kernel(const float* dw, int splits, const float* sums, int n_sums, const float* sums_dy, int n_dy, int hidden, int dim,
                T* dwg, T* dwu, T* dwd, T* dbg, T* dbu, T* dbd, int aligned) {
    __shared__ float tile[32][33];
    __shared__ float4 red[32][8];
    grid_dep_wait();
    const int tx = threadIdx.x & 7, ty = threadIdx.x >> 3;  // columns 4 tx .., row ty
    const int dt = (dim + 31) / 32, ht = (hidden + 31) / 32;
    int b = blockIdx.x;
    float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (b >= 3 * dt * ht) {
        // dim and hidden are multiples of 8: four columns are of one vector
        const int cols = 2 * hidden + dim, c = (b - 3 * dt * ht) * 32 + 4 * tx;
        const float* src = c < 2 * hidden ? sums + c : sums_dy + c - 2 * hidden;
        const int n = c < 2 * hidden ? n_sums : c < cols ? n_dy : 0, pitch = c < 2 * hidden ? 2 * hidden : dim;
#pragma unroll 4
        for (int p = ty; p < n; p += 32) s = s + *reinterpret_cast<const float4*>(src + (int64_t)p * pitch);
        red[ty][tx] = s;
        __syncthreads();
        if (ty == 0 && c < cols) {
            s = red[0][tx];
#pragma unroll
            for (int i = 1; i < 32; ++i) s = s + red[i][tx];
            T* out = c < hidden ? dbg : c < 2 * hidden ? dbu : dbd;
            if (out) {
                out += c < hidden ? c : c < 2 * hidden ? c - hidden : c - 2 * hidden;
                out[0] = from_f32<T>(s.x), out[1] = from_f32<T>(s.y), out[2] = from_f32<T>(s.z), out[3] = from_f32<T>(s.w);
            }
        }
        return;
    }
    const int d0 = b % dt * 32;
    b /= dt;
    const int h0 = b % ht * 32, seg = b / ht;
    T* out = seg == 0 ? dwg : seg == 1 ? dwu : dwd;
    if (!out) return;
    const int h = h0 + ty, d = d0 + 4 * tx;
    if (h < hidden && d < dim) {
        const float* p = dw + ((int64_t)seg * hidden + h) * dim + d;
#pragma unroll 4
        for (int k = 0; k < splits; ++k) s = s + *reinterpret_cast<const float4*>(p + (int64_t)k * 3 * hidden * dim);
        if (seg < 2) {
            T* o = out + (int64_t)h * dim + d;
            if (aligned) store4<T>(o, s);
            else o[0] = from_f32<T>(s.x), o[1] = from_f32<T>(s.y), o[2] = from_f32<T>(s.z), o[3] = from_f32<T>(s.w);
        }
    }
    if (seg < 2) return;
    tile[ty][4 * tx] = s.x, tile[ty][4 * tx + 1] = s.y, tile[ty][4 * tx + 2] = s.z, tile[ty][4 * tx + 3] = s.w;
    __syncthreads();
    if (d0 + ty < dim && h0 + 4 * tx < hidden) {
        T* o = out + (int64_t)(d0 + ty) * hidden + h0 + 4 * tx;
        s = make_float4(tile[4 * tx][ty], tile[4 * tx + 1][ty], tile[4 * tx + 2][ty], tile[4 * tx + 3][ty]);
        if (aligned) store4<T>(o, s);
        else o[0] = from_f32<T>(s.x), o[1] = from_f32<T>(s.y), o[2] = from_f32<T>(s.z), o[3] = from_f32<T>(s.w);
    }
}

// ---- host ------------------------------------------------------------------------------------------

#define fail prism::set_error

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
    static std::atomic<uint64_t> done{0};
    cudaError_t e = allow_smem(k, Cfg<KIND>::kSmem, ctx->device, done);
    if (e != cudaSuccess) return cuda_rc(e, who);
    const int pairs = std::min(a.units, ctx->sm_count / 2);
    return cuda_rc(launch_pdl(k, dim3(2 * pairs), dim3(Cfg<KIND>::kThreads), Cfg<KIND>::kSmem, s, a, m), who);
}

// Rows that go through at a time: whole waves of a row tile for every CTA pair, as many as keep
// `row_bytes` of scratch a row within 1 GiB, one at least (also where that is more than 1 GiB).  (130,560 x 256, hidden 1024, backward: 635 us
// by single waves, whose scratch half stays in L2, 559 us in one piece: launches and their first
// loads cost more than L2 gives.)
int64_t chunk_rows(const prism_ctx* ctx, int64_t rows, int64_t row_bytes) {
    const int64_t wave = (int64_t)(ctx->sm_count / 2) * 256;
    return std::min<int64_t>(rows, wave * std::max<int64_t>(1, (1ll << 30) / row_bytes / wave));
}

inline int64_t up_to(int64_t n, int64_t m) { return (n + m - 1) / m * m; }

// scratch of the backward pass: p [3][rows][hidden] 16-bit, dw [splits][3][hidden][dim] fp32, column sums
struct BackPlan {
    bool fused;
    int64_t chunk;
    int splits, pairs;            // pairs: of BACK's first launch
    int n_sums, n_dy;             // rows of the column sums of dg and du (a warp's) and of dy (a CTA's or a split's warp's)
    size_t p_bytes, dw_bytes, sum_bytes;
    size_t total() const { return p_bytes + dw_bytes + sum_bytes; }
};
BackPlan back_plan(const prism_ctx* ctx, const prism_gated_params* p) {
    BackPlan b;
    b.chunk = chunk_rows(ctx, p->rows, 6 * (int64_t)p->hidden);
    const int bn = p->dim <= 128 ? 128 : 256;
    const int64_t tiles = 3 * ((p->hidden + 255) / 256) * (int64_t)((p->dim + bn - 1) / bn);
    const int64_t kb = (b.chunk + 63) / 64;
    b.splits = (int)std::max<int64_t>(1, std::min<int64_t>(kb, (ctx->sm_count / 2) / tiles));
    b.fused = p->dim <= kFusedMaxDim;
    b.pairs = (int)std::min<int64_t>(ctx->sm_count / 2, (b.chunk + 255) / 256 * (b.fused ? 1 : (p->hidden + 127) / 128));
    b.p_bytes = (size_t)up_to(3 * b.chunk * p->hidden * 2, 1024);
    b.dw_bytes = (size_t)up_to((int64_t)b.splits * 3 * p->hidden * p->dim * 4, 1024);
    b.n_sums = 8 * b.pairs;
    b.n_dy = b.fused ? 2 * b.pairs : 16 * b.splits;
    b.sum_bytes = (b.n_sums * 2 * (size_t)p->hidden + b.n_dy * (size_t)p->dim) * 4;
    return b;
}

// XW's dW tiles over `pairs` CTA pairs: the least depth a pair that holds them all.
void share_out(Args& a, int pairs) {
    const int64_t kx = 2 * ((a.hidden + 63) / 64), n_w = a.units - a.x_units, more = a.x_units % pairs, all = a.x_units / pairs;
    const auto each = [&](int64_t depth, int64_t dx) { return std::max<int64_t>(0, (depth - dx * kx) / a.k_per); };
    int64_t lo = 0, hi = (all + 1) * kx + n_w * a.k_per;  // lo: too little, hi: enough
    while (hi - lo > 1) {
        const int64_t mid = (lo + hi) / 2;
        (more * each(mid, all + 1) + (pairs - more) * each(mid, all) >= n_w ? hi : lo) = mid;
    }
    a.w_each[1] = (int)std::min(n_w, each(hi, all + 1));
    a.w_each[0] = (int)std::max<int64_t>(a.w_each[1], std::min(n_w, each(hi, all)));
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
    if (rows > 1 && (stride > (int64_t)1 << 36 || !extent_ok(rows, stride)))
        return fail(PRISM_E_RANGE, "%s: %s_stride %lld", who, name, (long long)stride);
    return PRISM_OK;
}
int check_weight(const char* who, const char* name, const void* t, bool needed, int align = 16) {
    if (!t) return needed ? fail(PRISM_E_ARG, "%s: %s is NULL", who, name) : PRISM_OK;
    if ((uintptr_t)t % align) return fail(PRISM_E_ALIGN, "%s: %s is not %d-byte aligned", who, name, align);
    return PRISM_OK;
}
int64_t row_stride(int64_t stride, int64_t rows, int dim) { return rows > 1 ? stride : dim; }

// rows of one fused forward launch: 32-bit row coordinates with room to spare
constexpr int64_t kFusedRows = 1ll << 30;
void fused_args(const prism_ctx* ctx, const prism_gated_params* p, const prism_gated_weights* w, int rows, FusedArgs& a) {
    a.rows = rows;
    a.dim = p->dim;
    a.hidden = p->hidden;
    a.tiles = (rows + 255) / 256;
    a.bn = p->dim <= 128 ? 128 : 256;
    a.act = p->activation;
    a.b_gate = w->b_gate;
    a.b_up = w->b_up;
    a.err = ctx->err;
}
int fused_maps(const prism_gated_params* p, const prism_gated_weights* w, const void* x, int64_t xs, int rows, int step, FusedMaps& m) {
    int rc;
    if ((rc = make_map(&m.x, x, p->dtype, p->dim, rows, 0, xs, 64, 128, kSw128)) ||
        (rc = make_map(&m.wg, w->w_gate, p->dtype, p->dim, p->hidden, 0, p->dim, 64, step, kSw128)))
        return rc;
    return make_map(&m.wu, w->w_up, p->dtype, p->dim, p->hidden, 0, p->dim, 64, step, kSw128);
}

template <typename T>
int forward(const prism_ctx* ctx, const prism_gated_params* p, const prism_gated_weights* w, const void* x,
            const void* residual, void* y, void* ws, cudaStream_t s) {
    const char* who = "prism_gated_ffn";
    const int64_t xs = row_stride(p->x_stride, p->rows, p->dim), ys = row_stride(p->y_stride, p->rows, p->dim);
    const int64_t rs = row_stride(p->residual_stride, p->rows, p->dim);
    int rc;
    if (is_small(p->rows, p->dim, p->hidden)) {
        SmallArgs a{(int)p->rows, p->dim, p->hidden, p->activation, x, w->w_gate, w->b_gate, w->w_up, w->b_up, w->w_down, w->b_down,
                    residual, xs, rs, ys, static_cast<float*>(ws), y};
        return cuda_rc(launch_gated_small(std::is_same<T, __nv_bfloat16>::value, a, s), who);
    }
    // dim <= 256: one kernel; 522,240 x 256, hidden 1024: 627 us against 1258 of the two that follow
    for (int64_t r0 = 0; p->dim <= kFusedMaxDim && r0 < p->rows; r0 += kFusedRows) {
        const int rows = (int)std::min(kFusedRows, p->rows - r0);
        FusedArgs a = {};
        FusedMaps m;
        fused_args(ctx, p, w, rows, a);
        a.b_down = w->b_down;
        a.residual = residual != nullptr;
        if ((rc = residual ? make_map(&m.residual, static_cast<const T*>(residual) + r0 * rs, p->dtype, p->dim, rows, 0, rs, 32, 32, kSw64)
                           : PRISM_OK) ||
            (rc = fused_maps(p, w, static_cast<const T*>(x) + r0 * xs, xs, rows, 128, m)) ||
            (rc = make_map(&m.wd, w->w_down, p->dtype, p->hidden, p->dim, 0, p->hidden, 64, a.bn / 2, kSw128)) ||
            (rc = make_map(&m.out, static_cast<T*>(y) + r0 * ys, p->dtype, p->dim, rows, 0, ys, 32, 32, kSw64)) ||
            (rc = cuda_rc(launch_gated_fused(std::is_same<T, __nv_bfloat16>::value, false, a, m, ctx, s), who)))
            return rc;
    }
    if (p->dim <= kFusedMaxDim) return PRISM_OK;
    const int64_t chunk = chunk_rows(ctx, p->rows, 2 * (int64_t)p->hidden);
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
        a.bn = 256;
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
    float* sums = reinterpret_cast<float*>(static_cast<char*>(ws) + b.p_bytes + b.dw_bytes);
    const bool grads = d->dw_gate || d->db_gate || d->dw_up || d->db_up || d->dw_down || d->db_down;
    float* sums_dy = sums + (size_t)b.n_sums * 2 * p->hidden;
    int rc, splits = 1;
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
        a.first = r0 == 0;
        a.sums = sums;
        a.sums_dy = sums_dy;
        a.dy = dyc;
        a.dy_stride = dys;
        a.bn = p->dim <= 128 ? 128 : 256;
        a.m_tiles = (rows + 255) / 256;
        a.n_tiles = (p->hidden + 127) / 128;
        a.units = a.m_tiles * a.n_tiles;
        Maps m;
        T* dxc = static_cast<T*>(dx) + r0 * dxs;
        if (b.fused) {  // 56 us for 18,944 x 256, hidden 1024, against 64 of BACK and of XW's dx tiles
            FusedArgs f = {};
            FusedMaps fm;
            fused_args(ctx, p, w, rows, f);
            f.first = r0 == 0;
            f.sums = sums;
            f.sums_dy = sums_dy;
            if ((rc = fused_maps(p, w, xc, xs, rows, 64, fm)) ||
                (rc = make_map(&fm.dy, dyc, p->dtype, p->dim, rows, 0, dys, 64, 128, kSw128)) ||
                (rc = make_map(&fm.wd, w->w_down, p->dtype, p->hidden, p->dim, 0, p->hidden, 32, 128, kSw64)) ||
                (rc = make_map(&fm.wg_mn, w->w_gate, p->dtype, p->dim, p->hidden, 0, p->dim, 64, 64, kSw128)) ||
                (rc = make_map(&fm.wu_mn, w->w_up, p->dtype, p->dim, p->hidden, 0, p->dim, 64, 64, kSw128)) ||
                (rc = make_map(&fm.p, pbuf, p->dtype, p->hidden, rows, 3, p->hidden, 64, 32, kSw128)) ||
                (rc = make_map(&fm.out, dxc, p->dtype, p->dim, rows, 0, dxs, 32, 32, kSw64)) ||
                (rc = cuda_rc(launch_gated_fused(std::is_same<T, __nv_bfloat16>::value, true, f, fm, ctx, s), who)))
                return rc;
            a.sums_dy = nullptr;
            if (!grads) continue;
        } else {
            if ((rc = make_map(&m.a0, xc, p->dtype, p->dim, rows, 0, xs, 64, 128, kSw128)) ||
                (rc = make_map(&m.a1, dyc, p->dtype, p->dim, rows, 0, dys, 64, 128, kSw128)) ||
                (rc = make_map(&m.b0, w->w_gate, p->dtype, p->dim, p->hidden, 0, p->dim, 64, 128, kSw128)) ||
                (rc = make_map(&m.b1, w->w_up, p->dtype, p->dim, p->hidden, 0, p->dim, 64, 128, kSw128)) ||
                (rc = make_map(&m.b2, w->w_down, p->dtype, p->hidden, p->dim, 0, p->hidden, 64, 64, kSw128)) ||
                (rc = make_map(&m.out, pbuf, p->dtype, p->hidden, rows, 3, p->hidden, 32, 32, kSw64)) ||
                (rc = launch<T, BACK>(ctx, a, m, s, who)))
                return rc;
        }
        a.n_tiles = (p->dim + a.bn - 1) / a.bn;
        a.x_units = b.fused ? 0 : a.m_tiles * a.n_tiles;
        a.w_tiles = (p->hidden + 255) / 256;
        a.k_all = (rows + 63) / 64;
        a.k_per = (int)((up_to(b.chunk, 64) / 64 + b.splits - 1) / b.splits);
        const int here = (a.k_all + a.k_per - 1) / a.k_per;
        if (r0 == 0) splits = here;  // the first chunk is the largest: it writes every split's sums
        a.units = a.x_units + 3 * a.w_tiles * a.n_tiles * here;
        share_out(a, std::min(a.units, ctx->sm_count / 2));
        if ((rc = make_map(&m.p_k, pbuf, p->dtype, p->hidden, rows, 3, p->hidden, 64, 128, kSw128)) ||
            (rc = make_map(&m.p_mn, pbuf, p->dtype, p->hidden, rows, 3, p->hidden, 64, 64, kSw128)) ||
            (rc = make_map(&m.b0, w->w_gate, p->dtype, p->dim, p->hidden, 0, p->dim, 64, 64, kSw128)) ||
            (rc = make_map(&m.b1, w->w_up, p->dtype, p->dim, p->hidden, 0, p->dim, 64, 64, kSw128)) ||
            (rc = make_map(&m.x_mn, xc, p->dtype, p->dim, rows, 0, xs, 64, 64, kSw128)) ||
            (rc = make_map(&m.dy_mn, dyc, p->dtype, p->dim, rows, 0, dys, 64, 64, kSw128)) ||
            (rc = make_map(&m.out, dxc, p->dtype, p->dim, rows, 0, dxs, 32, 32, kSw64)) ||
            (rc = make_map(&m.dw, dw, PRISM_DTYPE_F32, p->dim, p->hidden, 3 * (int64_t)b.splits, p->dim, 32, 32, kSw128)) ||
            (rc = launch<T, XW>(ctx, a, m, s, who)))
            return rc;
    }
    if (!grads) return PRISM_OK;
    const int aligned = (((uintptr_t)d->dw_gate | (uintptr_t)d->dw_up | (uintptr_t)d->dw_down) & 7) == 0;
    const int blocks = 3 * ((p->dim + 31) / 32) * ((p->hidden + 31) / 32) + (2 * p->hidden + p->dim + 31) / 32;
    return cuda_rc(launch_pdl(fold_kernel<T>, dim3(blocks), dim3(256), 0, s, (const float*)dw, splits, (const float*)sums,
                              b.n_sums, (const float*)sums_dy, b.fused ? b.n_dy : 16 * splits, p->hidden, p->dim, static_cast<T*>(d->dw_gate), static_cast<T*>(d->dw_up),
                              static_cast<T*>(d->dw_down), static_cast<T*>(d->db_gate), static_cast<T*>(d->db_up),
                              static_cast<T*>(d->db_down), aligned), who);
}

}  // namespace
}  // namespace prism

using namespace prism;

extern "C" int prism_gated_ffn_workspace(prism_ctx* ctx, const prism_gated_params* p, int backward, size_t* bytes) {
    if (!ctx || !p || !bytes) return fail(PRISM_E_ARG, "prism_gated_ffn_workspace: NULL argument");
    int rc = check_gated("prism_gated_ffn_workspace", p);
    if (rc) return rc;
    *bytes = p->rows == 0 ? 0
             : backward   ? back_plan(ctx, p).total()
             : is_small(p->rows, p->dim, p->hidden) ? (size_t)p->rows * p->hidden * 4
             : p->dim <= kFusedMaxDim ? 0 : (size_t)chunk_rows(ctx, p->rows, 2 * (int64_t)p->hidden) * p->hidden * 2;
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
    const size_t nw = (size_t)p->hidden * p->dim * 2;
    const struct { void* t; size_t n; } all[6] = {{d->dw_gate, nw}, {d->dw_up, nw}, {d->dw_down, nw},
                                                  {d->db_gate, (size_t)p->hidden * 2}, {d->db_up, (size_t)p->hidden * 2},
                                                  {d->db_down, (size_t)p->dim * 2}};
    for (int i = 0; i < 6; ++i)
        for (int j = 0; j < i; ++j)
            if (bytes_overlap(all[i].t, all[i].n, all[j].t, all[j].n)) return fail(PRISM_E_ARG, "%s: two gradients overlap", who);
    DeviceGuard g(ctx->device);
    cudaStream_t s = as_stream(stream);
    if (p->rows == 0) {  // no rows: the sums are zero
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
