// gated_fused.cu - the gated feed-forward block for dim <= 256 as one kernel a direction.
//
// A CTA pair (tcgen05 cta_group::2) keeps 256 rows of x (backward: and dy) in shared memory and walks the
// hidden layer in steps (128 columns forward, 64 backward, what TMEM and shared memory hold); the
// hidden values never leave the SM forward.  Per step:
//   forward   [g | u] = x [Wg | Wu]^T -> TMEM;  epilogue: h = act(g + bg) (u + bu) -> smem;  y += h Wd^T
//   backward  [g | u] and dh = dy Wd -> TMEM;  epilogue: dg, du, h -> smem, from where TMA also stores
//             them for the weight gradients' products;  dx += dg Wg + du Wu
// The products of step c + 1 are issued before those that need the epilogue of step c, so the tensor pipe
// works through the epilogue.  Only weights stream: 96 KB a step and SM forward (3070 cycles of the
// tensor pipe), 80 KB backward (2560), at that pace some 30 bytes a clock; the streaming kernels of
// gated_ffn.cu load every operand for every product and are held at the 37 to 40 that L2 gives an SM.
// Measured: forward 522,240 x 256, hidden 1024, fp16 with residual 627 us, 1311 TFLOP/s (589 us without: the
// 1400 that the power limit leaves a long library product); backward with dx alone, bf16, 55 us for a row
// tile of every pair.  Steps and tensor pipe: 27 row tiles a pair forward, run for seconds, 4720 cycles a step at
// the sampled 1410 MHz (4640 a step more for a tile more), three tiles 4800 with the pipe 64 % busy; backward
// 6210 at 1590 MHz over 14 tiles (6170), three tiles 5810 with the pipe 44 % busy.  The rest is waits: for the ring's
// stages, the commits between, and the epilogue that the next products' operands come from.
#include <type_traits>

#include "gated_fused.cuh"

namespace prism {
namespace {

constexpr int kEpiWarps = 16;  // warp w: TMEM lanes 32 (w % 4) .., part (w - 2) / 4 of the columns
constexpr int kTile = 16384;   // 128 rows x 64 columns

template <bool BWD>
struct Cfg {
    // Producer, MMA issuer, epilogue warps; then, backward, one that stores p; forward, four that write the
    // output while the epilogue warps, bound by their exponentials and reciprocals, go on with the next tile.
    static constexpr int kThreads = 32 * (2 + kEpiWarps + (BWD ? 1 : 4));
    static constexpr int kStep = BWD ? 64 : 128;  // hidden columns a step
    static constexpr int kCols = kStep / 4;       // of an epilogue warp
    // Large stages: the commit that gives one back costs the tensor pipe some 100 cycles (backward with six of
    // 8 KB: 4600 cycles a step).
    static constexpr int kRing = 3, kStage = BWD ? 16384 : 32768;
    static constexpr int kXBytes = (BWD ? 8 : 4) * kTile;  // x, dy: four K-blocks each
    static constexpr int kPBytes = (BWD ? 3 : 2) * kTile;  // dg, du, h of 64 columns, or h of 128
    static constexpr int kOut = BWD ? 0 : 4 * 3 * 2048;  // forward: three 32 x 32 boxes an output warp (backward: in p)
    static constexpr int kDown = BWD ? 0 : 1024;         // the output's bias
    static constexpr int kBias = 2 * kCols * 4;          // bytes an epilogue warp
    // the dynamic shared memory of a kernel without static shared memory starts 1024-byte aligned
    static constexpr int kSmem = kXBytes + kPBytes + kRing * kStage + kOut + kDown + kEpiWarps * kBias + 512;
    static_assert(kSmem <= 232448, "227 KB");
    static constexpr int kAcc = 256;  // first TMEM column of [g | u (| dh)], behind the output accumulator
};
struct Bars {
    uint64_t full[3], empty[3], x_full, y_full, x_empty, acc_full, acc_empty, p_full, p_empty, o_full, o_empty;
    uint64_t p_quad[4], p_read;  // backward: a quad's rows of p are written; p's stores have read it
    uint64_t dy_read;            // backward: dy's columns are summed
    uint64_t res_full[4][3];     // forward: a box of the residual has landed
    uint32_t tmem_base;
    int abort;
};

template <typename T, int ACT>
PRISM_DEV void gate32(const uint32_t (&g)[32], const uint32_t (&u)[32], const float* bg, const float* bu, uint32_t (&h)[16]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const ulonglong2 b0 = reinterpret_cast<const ulonglong2*>(bg)[j], b1 = reinterpret_cast<const ulonglong2*>(bu)[j];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int i = 2 * j + e;
            float h0, h1;
            f2_unpack(gate2<ACT>(f2_pack(__uint_as_float(g[2 * i]), __uint_as_float(g[2 * i + 1])),
                                 f2_pack(__uint_as_float(u[2 * i]), __uint_as_float(u[2 * i + 1])), e ? b0.y : b0.x, e ? b1.y : b1.x),
                      h0, h1);
            h[i] = pack2<T>(h0, h1);
        }
    }
}

template <typename T, bool BWD>
__global__ void __launch_bounds__(Cfg<BWD>::kThreads, 1) __cluster_dims__(2, 1, 1)
    gated_fused_kernel(const FusedArgs a, const __grid_constant__ FusedMaps maps) {
    using C = Cfg<BWD>;
    extern __shared__ unsigned char smem[];
    unsigned char* s_x = smem;
    unsigned char* s_p = s_x + C::kXBytes;
    unsigned char* s_ring = s_p + C::kPBytes;
    unsigned char* s_out = s_ring + C::kRing * C::kStage;
    float* s_down = reinterpret_cast<float*>(s_out + C::kOut);
    unsigned char* s_bias = s_out + C::kOut + C::kDown;
    Bars* bars = reinterpret_cast<Bars*>(s_bias + kEpiWarps * C::kBias);
    volatile int* abort = &bars->abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)cluster_rank(), pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    constexpr bool bf16 = !std::is_same<T, __half>::value;
    const int kd = (a.dim + 63) / 64, steps = (a.hidden + C::kStep - 1) / C::kStep;
    const int bh = a.bn / 2;  // this CTA's share of N over dim

    if (threadIdx.x == 0) {
        for (int s = 0; s < C::kRing; ++s) {
            mbar_init(&bars->full[s], 1);
            mbar_init(&bars->empty[s], 1);
        }
        mbar_init(&bars->x_full, 1);
        mbar_init(&bars->y_full, 1);
        mbar_init(&bars->x_empty, 1);
        mbar_init(&bars->acc_full, 1);
        mbar_init(&bars->acc_empty, 2 * kEpiWarps);  // those that epilogue warps arrive on: the leader's, both CTAs' warps
        mbar_init(&bars->p_full, 2 * kEpiWarps);
        mbar_init(&bars->p_empty, 1);
        mbar_init(&bars->o_full, 1);
        mbar_init(&bars->o_empty, 2 * (BWD ? kEpiWarps : 4));
        for (int q = 0; q < 12; ++q) mbar_init(&bars->res_full[0][q], 1);
        for (int q = 0; q < 4; ++q) mbar_init(&bars->p_quad[q], 4);
        mbar_init(&bars->p_read, 1);
        mbar_init(&bars->dy_read, 1);
        bars->abort = (smem_u32(smem) & 1023u) != 0;
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
        // ---- producer (both CTAs)
        int stage = 0;
        uint32_t phase = 0;
        bool ok = !*abort;
        // one ring stage of `bytes` a CTA: waits for room; true if this lane is to issue the loads
        auto next = [&](uint32_t bytes, uint32_t& dst, uint32_t& bar) {
            ok = ok && mbar_wait_w(&bars->empty[stage], phase ^ 1, abort);
            dst = smem_u32(s_ring + stage * C::kStage);
            bar = peer_addr(smem_u32(&bars->full[stage]), 0);
            if (ok && lane == 0 && rank == 0) mbar_expect_tx(&bars->full[stage], 2 * bytes);
            if (++stage == C::kRing) {
                stage = 0;
                phase ^= 1;
            }
            return ok && lane == 0;
        };
        uint32_t it = 0;
        for (int tile = pair; tile < a.tiles && ok; tile += pairs, ++it) {
            const int row = tile * 256 + rank * 128;
            ok = mbar_wait_w(&bars->x_empty, (it & 1) ^ 1, abort);
            if (BWD && ok) ok = mbar_wait_w(&bars->dy_read, (it & 1) ^ 1, abort);
            if (!ok) break;
            if (lane == 0) {
                const uint32_t bx = peer_addr(smem_u32(&bars->x_full), 0), by = peer_addr(smem_u32(&bars->y_full), 0);
                if (rank == 0) {
                    mbar_expect_tx(&bars->x_full, 2 * kd * kTile);
                    if (BWD) mbar_expect_tx(&bars->y_full, 2 * kd * kTile);
                }
                for (int k = 0; k < kd; ++k) tma_load_2d_pair(smem_u32(s_x + k * kTile), &maps.x, bx, k * 64, row);
                if (BWD)
                    for (int k = 0; k < kd; ++k) tma_load_2d_pair(smem_u32(s_x + (4 + k) * kTile), &maps.dy, by, k * 64, row);
            }
            __syncwarp();
            uint32_t dst, bar;
            for (int c = 0; c <= steps && ok; ++c) {
                if (c < steps) {
                    // [g | u]: the leader brings Wg's rows, its peer Wu's
                    for (int k = 0; k < kd; k += 2) {
                        const int n = min(2, kd - k);
                        if (next(n * C::kStep * 128, dst, bar))
                            for (int i = 0; i < n; ++i)
                                tma_load_2d_pair(dst + i * C::kStep * 128, rank ? &maps.wu : &maps.wg, bar, (k + i) * 64, c * C::kStep);
                    }
                    // dh: 128 rows of Wd (k) at a time, this CTA's 32 hidden columns (n)
                    if (BWD && next((kd + 1) / 2 * 8192, dst, bar))
                        for (int k = 0; k < kd; k += 2) tma_load_2d_pair(dst + k * 4096, &maps.wd, bar, c * 64 + rank * 32, k * 64);
                }
                if (c > 0 && !BWD) {  // y: this CTA's rows of Wd, both K-blocks of the step
                    if (next(2 * bh * 128, dst, bar))
                        for (int i = 0; i < 2; ++i) tma_load_2d_pair(dst + i * bh * 128, &maps.wd, bar, (c - 1) * 128 + i * 64, rank * bh);
                }
                if (c > 0 && BWD) {  // dx: the step's 64 hidden rows (k) of Wg, then Wu; this CTA's columns of dim (n)
                    for (int s = 0; s < 2; ++s)
                        if (next(bh * 128, dst, bar))
                            for (int n = 0; n < bh; n += 64)
                                tma_load_2d_pair(dst + n * 128, s ? &maps.wu_mn : &maps.wg_mn, bar, rank * bh + n, (c - 1) * 64);
                }
            }
            __syncwarp();
        }
    } else if (warp == 1) {
        // ---- MMA issuer: the leader's, for both CTAs.  (The ring has one consumer: two that pass over each
        // other's stages can be two phases of a barrier apart, which its parity cannot tell from none.)
        if (rank == 0) {
            int stage = 0;
            uint32_t phase = 0, it = 0, i = 0;  // i: steps so far
            bool ok = !*abort;
            auto take = [&] {
                mbar_wait_step(&bars->full[stage], phase, abort);
                tc_fence_after();
                return smem_u32(s_ring + stage * C::kStage);
            };
            auto give = [&] {
                mma_commit_pair_w(&bars->empty[stage]);
                if (++stage == C::kRing) {
                    stage = 0;
                    phase ^= 1;
                }
            };
            const uint32_t id_gu = idesc_pair(256, 2 * C::kStep, bf16, 0, 0), id_dh = idesc_pair(256, 64, bf16, 0, 1);
            const uint32_t id_y = idesc_pair(256, a.bn, bf16, 0, 0), id_dx = idesc_pair(256, a.bn, bf16, 0, 1);
            const uint32_t x_lo = desc_lo(smem_u32(s_x)), p_lo = desc_lo(smem_u32(s_p)), acc = tmem + C::kAcc;
            constexpr uint32_t kBlk = kTile >> 4;
            for (int tile = pair; tile < a.tiles && ok; tile += pairs, ++it) {
                mbar_wait_step(&bars->x_full, it & 1, abort);
                for (int c = 0; c <= steps; ++c) {
                    ok = __all_sync(0xffffffffu, !*abort);
                    if (!ok) break;
                    if (c < steps) {
                        // the epilogue has read the step before
                        mbar_wait_step(&bars->acc_empty, ((i + c) & 1) ^ 1, abort);
                        for (int k = 0; k < kd; k += 2) {
                            const uint32_t b_lo = desc_lo(take());
                            mma_pair_x4<2, 2>(acc, x_lo + k * kBlk, kDescHi128, b_lo, kDescHi128, id_gu, k);
                            if (k + 1 < kd)
                                mma_pair_x4<2, 2>(acc, x_lo + (k + 1) * kBlk, kDescHi128, b_lo + C::kStep * 8, kDescHi128, id_gu, 1);
                            give();
                        }
                        if (BWD) {
                            if (c == 0) mbar_wait_step(&bars->y_full, it & 1, abort);
                            const uint32_t b_lo = desc_lo(take());
                            for (int k = 0; k < kd; ++k)
                                mma_pair_x4<2, 64>(acc + 128, x_lo + (4 + k) * kBlk, kDescHi128, b_lo + k * 256, kDescHi64, id_dh, k);
                            give();
                        }
                        mma_commit_pair_w(&bars->acc_full);
                        if (c == steps - 1) mma_commit_pair_w(&bars->x_empty);
                    }
                    if (c > 0) {
                        if (c == 1) mbar_wait_step(&bars->o_empty, (it & 1) ^ 1, abort);  // the last tile's output has been read
                        mbar_wait_step(&bars->p_full, (i + c - 1) & 1, abort);
                        if (!BWD) {
                            const uint32_t b_lo = desc_lo(take());
                            mma_pair_x4<2, 2>(tmem, p_lo, kDescHi128, b_lo, kDescHi128, id_y, c - 1);
                            mma_pair_x4<2, 2>(tmem, p_lo + kBlk, kDescHi128, b_lo + bh * 8, kDescHi128, id_y, 1);
                            give();
                        } else {
                            for (int s = 0; s < 2; ++s) {
                                mma_pair_x4<2, 128>(tmem, p_lo + s * kBlk, kDescHi128, desc_lo(take(), 8192), kDescHi128, id_dx, (c - 1) | s);
                                give();
                            }
                        }
                        mma_commit_pair_w(&bars->p_empty);
                        if (c == steps) mma_commit_pair_w(&bars->o_full);
                    }
                }
                i += steps;
            }
        }
    } else if (BWD && warp == 2 + kEpiWarps) {
        // ---- stores of p: 32 rows as soon as their four warps have written them; between them, dy's column sums
        // (db_down) from its tile in shared memory: 32 rows of 64 columns a unit, 8 columns a lane, shared out
        // over the tile's steps
        float* sums = a.sums_dy + (int64_t)blockIdx.x * a.dim;
        if (a.first)
            for (int c = lane; c < a.dim; c += 32) sums[c] = 0.0f;
        __syncwarp();
        const int per_step = (4 * kd + steps - 1) / steps;
        uint32_t i = 0;
        for (int tile = pair; tile < a.tiles; tile += pairs) {
            int unit = 0;
            float s8[8];
            for (int c = 0; c < steps; ++c, ++i) {
                for (int q = 0; q < 4; ++q) {
                    mbar_wait_step(&bars->p_quad[q], i & 1, abort);  // (so dy has landed: p needs its products)
                    const int row = tile * 256 + rank * 128 + q * 32;
                    if (lane == 0 && row < a.rows) {
                        const uint32_t src = smem_u32(s_p + q * 4096);
#pragma unroll
                        for (int s = 0; s < 3; ++s) tma_store_3d(&maps.p, src + s * kTile, c * 64, row, s);
                    }
                }
                if (lane == 0) {
                    tma_store_commit();
                    tma_store_wait_read<0>();
                    mbar_arrive(&bars->p_read);
                }
                __syncwarp();
                for (int n = 0; n < per_step && unit < 4 * kd; ++n, ++unit) {
                    const unsigned char* dy = s_x + (4 + (unit >> 2)) * kTile;
                    if ((unit & 3) == 0) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) s8[j] = 0.0f;
                    }
#pragma unroll
                    for (int r = 0; r < 32; r += 4) {
                        const uint4 v = *reinterpret_cast<const uint4*>(dy + sw128_off((unit & 3) * 32 + r + (lane >> 3), lane & 7));
                        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            float f0, f1;
                            unpack2<T>(w[j], f0, f1);
                            s8[2 * j] += f0;
                            s8[2 * j + 1] += f1;
                        }
                    }
                    if ((unit & 3) == 3) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            s8[j] += __shfl_xor_sync(0xffffffffu, s8[j], 8);
                            s8[j] += __shfl_xor_sync(0xffffffffu, s8[j], 16);
                            const int col = (unit >> 2) * 64 + 8 * lane + j;
                            if (lane < 8 && col < a.dim) sums[col] += s8[j];
                        }
                    }
                }
            }
            if (lane == 0) mbar_arrive(&bars->dy_read);
        }
        if (lane == 0) tma_store_wait0();
    } else if (!BWD && warp >= 2 + kEpiWarps) {
        // ---- output (forward): 32 rows a warp, 32 columns at a time.  The residual's boxes come by TMA two ahead
        // into the staging buffers that the output leaves from (a thread that reads a row of its own from
        // global memory touches 32 lines an instruction: 4000 cycles a tile).
        const int quad = warp & 3;
        unsigned char* bufs = s_out + quad * 3 * 2048;
        const uint32_t o_empty = peer_addr(smem_u32(&bars->o_empty), 0);
        for (int j = threadIdx.x - 32 * (2 + kEpiWarps); j < 256; j += 128) s_down[j] = ld_bias<T>(a.b_down, j, a.dim);
        named_bar_sync(6, 128);
        const int boxes = (a.dim + 31) / 32;
        uint32_t it = 0, n = 0;  // n: boxes so far
        for (int tile = pair; tile < a.tiles; tile += pairs, ++it) {
            const int row = tile * 256 + rank * 128 + quad * 32;
            auto load_res = [&](int box) {
                const uint32_t k = (n + box) % 3;
                if (a.residual && box < boxes && lane == 0) {
                    mbar_expect_tx(&bars->res_full[quad][k], 2048);
                    tma_load_2d(smem_u32(bufs + k * 2048), &maps.residual, &bars->res_full[quad][k], box * 32, row);
                }
            };
            if (lane == 0) tma_store_wait_read<0>();
            load_res(0);
            load_res(1);
            mbar_wait_step(&bars->o_full, it & 1, abort);
            tc_fence_after();
            for (int g = 0; g < boxes; ++g) {
                const uint32_t k = (n + g) % 3;
                unsigned char* buf = bufs + k * 2048;
                uint32_t r[32], o[16];
                tmem_ld32(tmem + ((uint32_t)(quad * 32) << 16) + g * 32, r);
                if (a.residual) mbar_wait_step(&bars->res_full[quad][k], ((n + g) / 3) & 1, abort);
                tmem_ld_wait();
                if (g == boxes - 1) {  // all read
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_pair(o_empty);
                }
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const uint4 v = a.residual ? *reinterpret_cast<const uint4*>(buf + sw64_off(lane, q)) : make_uint4(0, 0, 0, 0);
                    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        float f0, f1, y0, y1;
                        unpack2<T>(w[j], f0, f1);
                        const int i = 8 * q + 2 * j;
                        const uint64_t bias = *reinterpret_cast<const uint64_t*>(s_down + g * 32 + i);
                        f2_unpack(f2_add(f2_add(f2_pack(__uint_as_float(r[i]), __uint_as_float(r[i + 1])), bias), f2_pack(f0, f1)), y0, y1);
                        o[4 * q + j] = pack2<T>(y0, y1);
                    }
                }
                if (!a.residual) {  // with one, the loads have waited for the buffer's last store
                    if (lane == 0) tma_store_wait_read<2>();
                    __syncwarp();
                }
                stage_row64(buf, lane, o);
                fence_async_shared();
                __syncwarp();
                if (lane == 0) {
                    if (row < a.rows) tma_store_2d(&maps.out, smem_u32(buf), g * 32, row);
                    tma_store_commit();
                    if (a.residual) tma_store_wait_read<1>();  // the box before: its buffer is the next load's
                }
                load_res(g + 2);
            }
            n += boxes;
        }
        if (lane == 0) tma_store_wait0();
    } else {
        // ---- epilogue
        constexpr int kBiasVals = C::kBias / 128;
        const int quad = warp & 3, part = (warp - 2) >> 2;
        const uint32_t lane_addr = (uint32_t)(quad * 32) << 16;
        unsigned char* buf = s_p + (warp - 2) * 2048;  // backward: store staging, once the tile's steps are done
        float* bias = reinterpret_cast<float*>(s_bias + (warp - 2) * C::kBias);
        const uint32_t acc_empty = peer_addr(smem_u32(&bars->acc_empty), 0), o_empty = peer_addr(smem_u32(&bars->o_empty), 0);
        const uint32_t p_full = peer_addr(smem_u32(&bars->p_full), 0);
        // backward: this warp's rows of the column sums of dg and du; it alone has its columns of them
        float* sums = BWD ? a.sums + ((int64_t)blockIdx.x * 4 + quad) * (2 * a.hidden) : nullptr;
        if (BWD && a.first)
            for (int c = lane; c < a.hidden; c += 32)
                if (((c >> 4) & 3) == part) sums[c] = sums[a.hidden + c] = 0.0f;
        __syncwarp();
        // The biases of this warp's columns of a step, gate's then up's: a value or two a lane, loaded a step
        // ahead and converted when it is their turn (a conversion next to the load waits for it: 1300 cycles).
        T next_bias[kBiasVals];
        auto load_bias = [&](int step) {
#pragma unroll
            for (int j = 0; j < kBiasVals; ++j) {
                const int k = lane + 32 * j, c = step * C::kStep + part * C::kCols + k % C::kCols;
                const void* b = k < C::kCols ? a.b_gate : a.b_up;
                next_bias[j] = from_f32<T>(0.0f);
                if (b && c < a.hidden) next_bias[j] = static_cast<const T*>(b)[c];
            }
        };
        load_bias(0);
        // A wait that gives up does not end the loops: the warps meet at barriers (which are not bounded),
        // so all of them walk on to the end, where every further wait gives up at once.
        uint32_t it = 0, i = 0;
        for (int tile = pair; tile < a.tiles; tile += pairs, ++it) {
            const int row = tile * 256 + rank * 128 + quad * 32;
            for (int c = 0; c < steps; ++c, ++i) {
                const int col = c * C::kStep + part * C::kCols;
                __syncwarp();
#pragma unroll
                for (int j = 0; j < kBiasVals; ++j) bias[lane + 32 * j] = to_f32(next_bias[j]);
                load_bias(c + 1 < steps ? c + 1 : 0);
                __syncwarp();
                mbar_wait_w(&bars->acc_full, i & 1, abort);
                tc_fence_after();
                const uint32_t acc = tmem + lane_addr + C::kAcc + part * C::kCols;
                const int prow = quad * 32 + lane;
                if (!BWD) {
                    uint32_t rg[32], ru[32], h[16];
                    tmem_ld32(acc, rg);
                    tmem_ld32(acc + 128, ru);
                    tmem_ld_wait();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_pair(acc_empty);  // the next step's products may come
                    if (a.act == kActSilu) gate32<T, kActSilu>(rg, ru, bias, bias + 32, h);
                    else if (a.act == kActGelu) gate32<T, kActGelu>(rg, ru, bias, bias + 32, h);
                    else gate32<T, kActRelu>(rg, ru, bias, bias + 32, h);
                    mbar_wait_w(&bars->p_empty, (i & 1) ^ 1, abort);  // y of the step before has read p
                    unsigned char* p = s_p + (part >> 1) * kTile;
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        *reinterpret_cast<uint4*>(p + sw128_off(prow, (part & 1) * 4 + q)) =
                            make_uint4(h[4 * q], h[4 * q + 1], h[4 * q + 2], h[4 * q + 3]);
                    fence_async_shared();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_pair(p_full);
                } else {
                    uint32_t rg[16], ru[16], rd[16], h[8];
                    uint64_t dg[8], du[8];
                    unsigned char* p = s_p;
                    tmem_ld16(acc, rg);
                    tmem_ld16(acc + 64, ru);
                    tmem_ld16(acc + 128, rd);
                    tmem_ld_wait();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_pair(acc_empty);
                    if (a.act == kActSilu) grad_cols<T, kActSilu>(rg, ru, rd, bias, bias + 16, dg, du, h);
                    else if (a.act == kActGelu) grad_cols<T, kActGelu>(rg, ru, rd, bias, bias + 16, dg, du, h);
                    else grad_cols<T, kActRelu>(rg, ru, rd, bias, bias + 16, dg, du, h);
                    // room in p: dx of the step before and the stores have read it; at a tile's start, every
                    // warp's staging of the tile before too
                    mbar_wait_w(&bars->p_empty, (i & 1) ^ 1, abort);
                    mbar_wait_w(&bars->p_read, (i & 1) ^ 1, abort);
                    if (c == 0) {
                        if (lane == 0) tma_store_wait_read<0>();
                        __syncwarp();
                        named_bar_sync(5, 32 * kEpiWarps);
                    }
                    const uint32_t o0 = sw128_off(prow, part * 2), o1 = sw128_off(prow, part * 2 + 1);
                    *reinterpret_cast<uint4*>(p + o0) = pack8<T>(dg);
                    *reinterpret_cast<uint4*>(p + o1) = pack8<T>(dg + 4);
                    *reinterpret_cast<uint4*>(p + kTile + o0) = pack8<T>(du);
                    *reinterpret_cast<uint4*>(p + kTile + o1) = pack8<T>(du + 4);
                    *reinterpret_cast<uint4*>(p + 2 * kTile + o0) = make_uint4(h[0], h[1], h[2], h[3]);
                    *reinterpret_cast<uint4*>(p + 2 * kTile + o1) = make_uint4(h[4], h[5], h[6], h[7]);
                    fence_async_shared();
                    __syncwarp();
                    if (lane == 0) {
                        mbar_arrive_pair(p_full);
                        mbar_arrive(&bars->p_quad[quad]);
                    }
                    // bias gradients from the values before their rounding; one lane adds to an address, in the order of
                    // its steps: the same bits every time
                    const float sg = column_sum(dg, lane), su = column_sum(du, lane);
                    const int cs = col + (lane >> 1);
                    if (cs < a.hidden) atomicAdd(sums + (lane & 1 ? a.hidden : 0) + cs, lane & 1 ? su : sg);
                }
            }
            if (!BWD) continue;
            // ---- the tile's dx: 64 columns a warp (32 where bn is 128)
            const int cols = a.bn / 4, col0 = part * cols;
            mbar_wait_w(&bars->o_full, it & 1, abort);
            mbar_wait_w(&bars->p_read, (i & 1) ^ 1, abort);  // p becomes staging: its last stores have read it
            tc_fence_after();
#pragma unroll
            for (int g = 0; g < 64; g += 32) {
                if (g >= cols) break;
                uint32_t r[32], o[16];
                tmem_ld32(tmem + lane_addr + col0 + g, r);
                tmem_ld_wait();
                if (g + 32 >= cols) {  // all read
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_pair(o_empty);
                }
#pragma unroll
                for (int j = 0; j < 16; ++j) o[j] = pack2<T>(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1]));
                if (lane == 0) tma_store_wait_read<0>();
                __syncwarp();
                stage_row64(buf, lane, o);
                fence_async_shared();
                __syncwarp();
                if (lane == 0 && col0 + g < a.dim && row < a.rows) {
                    tma_store_2d(&maps.out, smem_u32(buf), col0 + g, row);
                    tma_store_commit();
                }
            }
        }
        if (lane == 0) tma_store_wait0();
    }
    if (*abort && lane == 0) atomicOr(a.err, ERR_TIMEOUT);
    __syncwarp();
    tc_fence_before();
    cluster_sync();
    if (warp == 1) tmem_dealloc_pair(tmem, 512);
}

template <typename T, bool BWD>
cudaError_t launch(const FusedArgs& a, const FusedMaps& m, const prism_ctx* ctx, cudaStream_t s) {
    static std::atomic<uint64_t> done{0};
    auto k = gated_fused_kernel<T, BWD>;
    cudaError_t e = allow_smem(k, Cfg<BWD>::kSmem, ctx->device, done);
    if (e != cudaSuccess) return e;
    return launch_pdl(k, dim3(2 * fused_pairs(a.tiles, ctx->sm_count)), dim3(Cfg<BWD>::kThreads), Cfg<BWD>::kSmem, s, a, m);
}

}  // namespace

cudaError_t launch_gated_fused(bool bf16, bool backward, const FusedArgs& a, const FusedMaps& m, const prism_ctx* ctx, cudaStream_t s) {
    if (bf16) return backward ? launch<__nv_bfloat16, true>(a, m, ctx, s) : launch<__nv_bfloat16, false>(a, m, ctx, s);
    return backward ? launch<__half, true>(a, m, ctx, s) : launch<__half, false>(a, m, ctx, s);
}

}  // namespace prism
