// gated_tc.cuh - CTA-pair (cta_group::2) building blocks of the gated feed-forward kernels: TMA loads
// that complete on the leader's barrier, 256-row tcgen05 MMAs over both CTAs' shared memory and TMEM,
// operand descriptors for both majors, and the gate's activations.
#pragma once
#include <type_traits>

#include "train_util.cuh"

namespace prism {

enum GateAct : int { kActGelu = PRISM_ACT_GELU, kActSilu = PRISM_ACT_SILU, kActRelu = PRISM_ACT_RELU };

// ---- pair TMA / MMA ------------------------------------------------------------------------
// Loads into this CTA's shared memory; the bytes complete on an mbarrier of the pair's leader
// (`bar` is a shared::cluster address).  No multicast.
PRISM_DEV void tma_load_2d_pair(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
        "l"(map), "r"(bar), "r"(c0), "r"(c1)
        : "memory");
}
PRISM_DEV void tma_load_3d_pair(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
        "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2)
        : "memory");
}
PRISM_DEV void tma_store_2d(const CUtensorMap* map, uint32_t src, int c0, int c1) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%2, %3}], [%1];" ::"l"(map), "r"(src),
                 "r"(c0), "r"(c1)
                 : "memory");
}
// fp32 box added to global memory in L2
PRISM_DEV void tma_add_3d(const CUtensorMap* map, uint32_t src, int c0, int c1, int c2) {
    asm volatile("cp.reduce.async.bulk.tensor.3d.global.shared::cta.add.tile.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(map),
                 "r"(src), "r"(c0), "r"(c1), "r"(c2)
                 : "memory");
}
PRISM_DEV void tmem_alloc_pair(uint32_t* dst_smem, uint32_t ncols) {  // one warp of each CTA
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(dst_smem)), "r"(ncols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
PRISM_DEV void tmem_dealloc_pair(uint32_t taddr, uint32_t ncols) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
// Matrix descriptors as (low, high) words: the low word holds the address, so the operands of one MMA
// after another differ by an addition there.  K-major tiles are rows of 128 bytes (64 k; 16 k further is
// 2 units of 16 bytes on); MN-major ones groups of 64 MN values, each [k][64] with 128 bytes a k row, 8
// rows = 1024 bytes (the stride field), `group_bytes` from one group to the next (16 k further: 128 units).
PRISM_DEV uint32_t desc_lo(uint32_t saddr, uint32_t group_bytes = 16) { return (saddr >> 4) | (group_bytes >> 4) << 16; }
constexpr uint32_t kDescHi128 = (1024u >> 4) | (1u << 14) | ((uint32_t)SW128 << 29);
constexpr uint32_t kDescHi64 = (512u >> 4) | (1u << 14) | ((uint32_t)SW64 << 29);
// D (+)= A x B^T over the pair: rows 0..127 of A and of D in the leader, 128..255 in its peer; the
// first half of B's N rows from the leader's shared memory, the second from the peer's.  Issued by one
// elected lane of the leader's converged MMA warp.
// Four MMAs (64 deep) whose descriptors advance by ASTEP, BSTEP 16-byte units, the first one adding to D
// if `accumulate`.  One block, one elect: issued one by one, with their descriptors worked out each
// time, 16 MMAs of N = 128 took 2000 cycles to issue for 1072 cycles of work.
template <int ASTEP, int BSTEP>
PRISM_DEV void mma_pair_x4(uint32_t d_tmem, uint32_t alo, uint32_t ahi, uint32_t blo, uint32_t bhi, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, e, t;\n\t.reg .b32 r, a1, a2, a3, b1, b2, b3;\n\t.reg .b64 x0, x1, x2, x3, y0, y1, y2, y3;\n\t"
        "add.u32 a1, %1, %7;\n\tadd.u32 a2, %1, %8;\n\tadd.u32 a3, %1, %9;\n\t"
        "add.u32 b1, %3, %10;\n\tadd.u32 b2, %3, %11;\n\tadd.u32 b3, %3, %12;\n\t"
        "mov.b64 x0, {%1, %2};\n\tmov.b64 x1, {a1, %2};\n\tmov.b64 x2, {a2, %2};\n\tmov.b64 x3, {a3, %2};\n\t"
        "mov.b64 y0, {%3, %4};\n\tmov.b64 y1, {b1, %4};\n\tmov.b64 y2, {b2, %4};\n\tmov.b64 y3, {b3, %4};\n\t"
        "setp.ne.b32 p, %6, 0;\n\tsetp.eq.u32 t, 0, 0;\n\t"
        "elect.sync r|e, 0xffffffff;\n\t"
        "@e tcgen05.mma.cta_group::2.kind::f16 [%0], x0, y0, %5, p;\n\t"
        "@e tcgen05.mma.cta_group::2.kind::f16 [%0], x1, y1, %5, t;\n\t"
        "@e tcgen05.mma.cta_group::2.kind::f16 [%0], x2, y2, %5, t;\n\t"
        "@e tcgen05.mma.cta_group::2.kind::f16 [%0], x3, y3, %5, t;\n\t}" ::"r"(d_tmem),
        "r"(alo), "r"(ahi), "r"(blo), "r"(bhi), "r"(idesc), "r"(accumulate), "n"(ASTEP), "n"(2 * ASTEP), "n"(3 * ASTEP),
        "n"(BSTEP), "n"(2 * BSTEP), "n"(3 * BSTEP)
        : "memory");
}
// A wait of a whole converged warp without the vote on its outcome: a wait that gives up raises *abort,
// which the role looks at once a step (MMAs issued meanwhile compute on stale but valid memory).
PRISM_DEV void mbar_wait_step(uint64_t* bar, uint32_t parity, volatile int* abort) {
    if (!mbar_try_wait(bar, parity)) mbar_wait_spin(bar, parity, abort);
    __syncwarp();
}
// Arrives on an mbarrier of this CTA or its peer (a shared::cluster address), without a cluster-scope
// release, which costs a full memory barrier: 40 -> 33 us for 8160 rows forward.  What is handed over is
// this CTA's own shared memory, written before a fence.proxy.async and read by the tensor core alone, or
// its TMEM, read before a tcgen05.fence.  The written memory model orders that against the other CTA's
// waiter only by a cluster-scope release.  That the fence and this arrival are enough is practice relied on (the
// memory that the tensor core reads is the one that the fence completed the writes to), not its guarantee.
PRISM_DEV void mbar_arrive_pair(uint32_t bar_cluster) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar_cluster) : "memory");
}
// arrives on the barrier at this offset in both CTAs once every MMA issued before has completed
PRISM_DEV void mma_commit_pair_w(uint64_t* bar) {
    asm volatile(
        "{\n\t.reg .pred e;\n\t.reg .b32 r;\n\t.reg .b16 m;\n\t"
        "mov.b16 m, 3;\n\t"
        "elect.sync r|e, 0xffffffff;\n\t"
        "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], m;\n\t}" ::"r"(
            smem_u32(bar))
        : "memory");
}

// Instruction descriptor, kind::f16, D fp32: formats (0 = fp16, 1 = bf16), majors (1 = MN), N, M.
PRISM_DEV uint32_t idesc_pair(int M, int N, int bf16, int a_mn, int b_mn) {
    return (1u << 4) | ((uint32_t)bf16 << 7) | ((uint32_t)bf16 << 10) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) |
           ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
// ---- epilogues ------------------------------------------------------------------------------
template <typename T>
PRISM_DEV float ld_bias(const void* b, int i, int n) {
    return b && i < n ? to_f32(static_cast<const T*>(b)[i]) : 0.0f;
}

// A 32 x 32 box of a warp's rows: this lane's row as 16 packed pairs into 64-byte swizzled rows.
PRISM_DEV void stage_row64(unsigned char* buf, int lane, const uint32_t (&v)[16]) {
#pragma unroll
    for (int q = 0; q < 4; ++q)
        *reinterpret_cast<uint4*>(buf + sw64_off(lane, q)) = make_uint4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
}
// ---- the gate ----------------------------------------------------------------------------------
// 1 / (1 + 2^-t): both hardware approximations are good to about 2^-22, far under the 16-bit rounding
// that follows (tanh.approx's 2^-11 would double the error of an fp16 result).
PRISM_DEV float sigmoid_exp2(float t) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + ex2_approx(-t)));
    return r;
}
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kGelu2c = 1.5957691216057308f;  // 2 sqrt(2 / pi)
constexpr float kGeluA = 0.044715f;
// act(g); gelu as the framework's tanh form, written g sigmoid(2 sqrt(2/pi) (g + 0.044715 g^3))
template <int ACT>
PRISM_DEV float gate(float g) {
    if (ACT == kActRelu) return g <= 0.0f ? 0.0f : g;  // NaN stays
    if (ACT == kActSilu) return g * sigmoid_exp2(kLog2e * g);
    const float z = g * fmaf(kGelu2c * kGeluA * kLog2e, g * g, kGelu2c * kLog2e);
    return g * sigmoid_exp2(z);
}
PRISM_DEV uint64_t f2_same(float v) { return f2_pack(v, v); }
// act(g + bg) (u + bu) of two columns
template <int ACT>
PRISM_DEV uint64_t gate2(uint64_t g, uint64_t u, uint64_t bg, uint64_t bu) {
    g = f2_add(g, bg);
    u = f2_add(u, bu);
    float g0, g1;
    f2_unpack(g, g0, g1);
    if (ACT == kActRelu) return f2_mul(f2_pack(g0 <= 0.0f ? 0.0f : g0, g1 <= 0.0f ? 0.0f : g1), u);  // NaN stays
    const uint64_t z = ACT == kActSilu ? f2_mul(g, f2_same(-kLog2e))
                                       : f2_mul(g, f2_fma(f2_same(-kGelu2c * kGeluA * kLog2e), f2_mul(g, g), f2_same(-kGelu2c * kLog2e)));
    float z0, z1, e0, e1, s0, s1;
    f2_unpack(z, z0, z1);
    f2_unpack(f2_add(f2_pack(ex2_approx(z0), ex2_approx(z1)), f2_same(1.0f)), e0, e1);
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s0) : "f"(e0));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s1) : "f"(e1));
    return f2_mul(f2_mul(g, f2_pack(s0, s1)), u);
}
// The gradient of two columns: from g, u (before their biases) and dh to dg, du and h, all in fp32
// pairs (f32x2: the epilogue that runs this is bound by its instructions).
template <int ACT>
PRISM_DEV void gate_grad2(uint64_t g, uint64_t u, uint64_t dh, uint64_t bg, uint64_t bu, uint64_t& dg, uint64_t& du, uint64_t& h) {
    g = f2_add(g, bg);
    u = f2_add(u, bu);
    uint64_t a, d;  // act(g), act'(g)
    if (ACT == kActRelu) {
        float g0, g1;
        f2_unpack(g, g0, g1);
        a = f2_pack(g0 <= 0.0f ? 0.0f : g0, g1 <= 0.0f ? 0.0f : g1);  // NaN stays
        d = f2_pack(g0 > 0.0f ? 1.0f : 0.0f, g1 > 0.0f ? 1.0f : 0.0f);
    } else {
        const uint64_t g2 = f2_mul(g, g);
        const uint64_t z = ACT == kActSilu ? f2_mul(g, f2_same(-kLog2e))
                                           : f2_mul(g, f2_fma(f2_same(-kGelu2c * kGeluA * kLog2e), g2, f2_same(-kGelu2c * kLog2e)));
        float z0, z1, e0, e1, s0, s1;
        f2_unpack(z, z0, z1);
        f2_unpack(f2_add(f2_pack(ex2_approx(z0), ex2_approx(z1)), f2_same(1.0f)), e0, e1);
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s0) : "f"(e0));
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s1) : "f"(e1));
        const uint64_t s = f2_pack(s0, s1), r = f2_fma(s, f2_same(-1.0f), f2_same(1.0f));  // 1 - s
        a = f2_mul(g, s);
        d = ACT == kActSilu ? f2_fma(a, r, s) : f2_fma(f2_mul(a, r), f2_fma(f2_same(3.0f * kGelu2c * kGeluA), g2, f2_same(kGelu2c)), s);
    }
    dg = f2_mul(f2_mul(dh, u), d);
    du = f2_mul(dh, a);
    h = f2_mul(a, u);
}

// 16 columns of one row: dg, du as fp32 pairs for the column sums, and all three packed
template <typename T, int ACT>
PRISM_DEV void grad_cols(const uint32_t (&g)[16], const uint32_t (&u)[16], const uint32_t (&dh)[16], const float* bg,
                         const float* bu, uint64_t (&dg)[8], uint64_t (&du)[8], uint32_t* h) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const ulonglong2 b0 = reinterpret_cast<const ulonglong2*>(bg)[j], b1 = reinterpret_cast<const ulonglong2*>(bu)[j];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int i = 2 * j + e;
            uint64_t hv;
            gate_grad2<ACT>(f2_pack(__uint_as_float(g[2 * i]), __uint_as_float(g[2 * i + 1])),
                            f2_pack(__uint_as_float(u[2 * i]), __uint_as_float(u[2 * i + 1])),
                            f2_pack(__uint_as_float(dh[2 * i]), __uint_as_float(dh[2 * i + 1])), e ? b0.y : b0.x, e ? b1.y : b1.x,
                            dg[i], du[i], hv);
            float h0, h1;
            f2_unpack(hv, h0, h1);
            h[i] = pack2<T>(h0, h1);
        }
    }
}
template <typename T>
PRISM_DEV uint4 pack8(const uint64_t* v) {
    uint32_t o[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        float a, b;
        f2_unpack(v[j], a, b);
        o[j] = pack2<T>(a, b);
    }
    return make_uint4(o[0], o[1], o[2], o[3]);
}
// Sums of 16 columns (as 8 pairs) over the warp's 32 rows: each step halves the columns that a lane still
// holds (16 shuffles for 16 columns).  Lanes l and l + 1 end with column l / 2 (bits of l, high first).
PRISM_DEV float column_sum(uint64_t (&v)[8], int lane) {
#pragma unroll
    for (int o = 4, bit = 16; o > 0; o >>= 1, bit >>= 1) {
        const bool up = lane & bit;
#pragma unroll
        for (int i = 0; i < o; ++i) {
            const uint64_t send = up ? v[i] : v[i + o], keep = up ? v[i + o] : v[i];
            v[i] = f2_add(keep, __shfl_xor_sync(0xffffffffu, send, bit));
        }
    }
    float a, b;
    f2_unpack(v[0], a, b);
    const bool up = lane & 2;
    a = (up ? b : a) + __shfl_xor_sync(0xffffffffu, up ? a : b, 2);
    return a + __shfl_xor_sync(0xffffffffu, a, 1);
}

}  // namespace prism
