"""Plain 64-bit forms of the trainable sub-block's operators, written from their formulas, with the
tolerances of their fp32 arithmetic.

A tolerance is counted in roundings.  U32 = 2^-24 is one fp32 rounding; u(dtype) = eps / 2 is the one
rounding of an output to its type.  A sum of n terms in fp32 is off by at most (its longest chain of
additions) * U32 * (the sum of the terms' magnitudes)."""
from __future__ import annotations

import math

import torch

U32 = 2.0 ** -24
M32 = 0xFFFFFFFF
# the smallest spacing of each type below its normal range (subnormal results are off by half of it)
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}


def u(dtype):
    return torch.finfo(dtype).eps / 2


def check(got, want, tol, what):
    """|got - want| <= u |want| + tol, element by element; infinities and NaN in the same places."""
    got64, want = got.double().cpu(), want.cpu()
    tol = tol.cpu() if torch.is_tensor(tol) else torch.full_like(want, tol)
    fin = torch.isfinite(want)
    assert torch.equal(torch.isnan(want), torch.isnan(got64)), f"{what}: NaN in other places"
    same_inf = want[torch.isinf(want)] == got64[torch.isinf(want)]
    assert same_inf.all(), f"{what}: infinities in other places"
    # the value before its rounding is off by tol, so its own rounding is half a step of |want| + tol
    bound = tol + u(got.dtype) * (want.abs() + tol) + TINY[got.dtype]
    off = (got64 - want).abs()
    bad = fin & ~(off <= bound)
    if bad.any():
        i = (off / bound).masked_fill(~bad, 0).argmax()
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off; worst at {int(i)}: got "
                             f"{got64.reshape(-1)[i]:.9g}, want {want.reshape(-1)[i]:.9g}, bound {bound.reshape(-1)[i]:.3g}")


# ---- layer norm -----------------------------------------------------------------------------
# A thread adds at most 64 of its own values, then at most 5 lanes and 8 warps: 77 additions, and a
# few roundings on each value: 96 in all.
K_ROW = 96


def norm(x, w, b, eps):
    """(y, mean, rstd) and their tolerances."""
    x, D = x.double(), x.shape[-1]
    w = torch.ones(D, dtype=torch.float64, device=x.device) if w is None else w.double()
    b = torch.zeros(D, dtype=torch.float64, device=x.device) if b is None else b.double()
    mean = x.mean(-1)
    c = x - mean[:, None]
    var = (c * c).mean(-1)
    rstd = 1 / torch.sqrt(var + eps)
    y = c * rstd[:, None] * w + b
    t_mean = K_ROW * U32 * x.abs().mean(-1)
    t_c = t_mean[:, None] + U32 * c.abs()  # x - mean
    # the second moment: its own additions and twice the error of the centred values
    t_var = (K_ROW * U32 * (c * c) + 2 * c.abs() * t_c + t_c * t_c).mean(-1)
    t_rstd = rstd * (0.5 * t_var / (var + eps) + 4 * U32)
    t_y = w.abs() * (t_c * rstd[:, None] + c.abs() * t_rstd[:, None]) + 4 * U32 * ((c * rstd[:, None] * w).abs() + b.abs())
    return (y, mean, rstd), (t_y, t_mean, t_rstd)


def norm_back(x, w, mean, rstd, dy, add):
    """(dx, dweight, dbias) and their tolerances, from the given statistics."""
    x, dy, R, D = x.double(), dy.double(), x.shape[0], x.shape[-1]
    w = torch.ones(D, dtype=torch.float64, device=x.device) if w is None else w.double()
    m, r = mean.double()[:, None], rstd.double()[:, None]
    xh, g = (x - m) * r, dy * w
    t_xh = 3 * U32 * (x.abs() + m.abs()) * r.abs()
    m0, m1 = g.mean(-1, keepdim=True), (g * xh).mean(-1, keepdim=True)
    t_m0 = K_ROW * U32 * g.abs().mean(-1, keepdim=True)
    t_m1 = (K_ROW * U32 * (g * xh).abs() + g.abs() * t_xh).mean(-1, keepdim=True)
    dx = r * (g - m0 - xh * m1)
    t_dx = r.abs() * (t_m0 + t_xh * m1.abs() + xh.abs() * t_m1 + 6 * U32 * (g.abs() + m0.abs() + (xh * m1).abs()))
    if add is not None:
        dx = dx + add.double()
        t_dx = t_dx + 2 * U32 * (add.double().abs() + dx.abs())
    # rows one after the other in a thread (at least 148 threads a column, one on each SM, once there are
    # that many rows), then the teams of a warp, the warps (13 together) and the CTAs' partial sums (10 + 32)
    k = R / 148 + 1 + 64
    dw, db = (dy * xh).sum(0), dy.sum(0)
    t_dw = k * U32 * (dy * xh).abs().sum(0) + (dy.abs() * t_xh).sum(0)
    t_db = k * U32 * dy.abs().sum(0)
    return (dx, dw, db), (t_dx, t_dw, t_db)


# ---- dropout ----------------------------------------------------------------------------------


def philox_block(counter, key):
    """One Philox4x32-10 block in Python integers (Salmon, Moraes, Dror, Shaw, 2011)."""
    c, k = list(counter), list(key)
    for _ in range(10):
        a, b = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [(b >> 32) ^ c[1] ^ k[0], b & M32, (a >> 32) ^ c[3] ^ k[1], a & M32]
        k = [(k[0] + 0x9E3779B9) & M32, (k[1] + 0xBB67AE85) & M32]
    return c


def draws(rng, n):
    """The 16-bit draws of elements 0 .. n - 1."""
    seed, off = int(rng[0]), int(rng[1])
    out = []
    for i in range((n + 7) // 8):
        for word in philox_block([i & M32, i >> 32, off & M32, (off >> 32) & M32], [seed & M32, (seed >> 32) & M32]):
            out += [word & 0xFFFF, word >> 16]
    return torch.tensor(out[:n], dtype=torch.int64)


def dropout(x, residual, threshold, rng):
    x = x.double().cpu()
    keep = (draws(rng, x.numel()) >= threshold).reshape(x.shape)
    v = torch.where(keep, x * (65536 / (65536 - threshold)), torch.zeros_like(x))
    y = v if residual is None else v + residual.double().cpu()
    return y, 4 * U32 * (v.abs() + y.abs()), keep


# ---- the gated feed-forward block ------------------------------------------------------------


def act(g, kind):
    """act(g), its first derivative, and bounds of the first and second derivatives' magnitudes."""
    if kind == "relu":
        return g.clamp(min=0), (g > 0).double()
    if kind == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    c, a = math.sqrt(2 / math.pi), 0.044715
    s = torch.sigmoid(2 * c * (g + a * g ** 3))
    return g * s, s + g * s * (1 - s) * 2 * c * (1 + 3 * a * g * g)


# The kernels' sigmoid comes from two hardware approximations of about 2^-22 each; 2^-18 of the values
# involved covers them and the roundings between.
APPROX = 2.0 ** -18


def _rounded(v, t, dtype):
    """Error of v after one more rounding to `dtype`."""
    return t + u(dtype) * (v.abs() + t) + TINY[dtype]


def _hidden(x, wg, wu, bg, bu, kind):
    """g, u, their error, act(g), act'(g) and the latter's error.  A product of n terms in the tensor cores'
    fp32 accumulators, which need not round to nearest, is off by at most 2 n U32 of the magnitudes' sum."""
    n = 2 * (x.shape[1] + 2) * U32
    g, v = x @ wg.T + bg, x @ wu.T + bu
    t_g, t_u = n * (x.abs() @ wg.abs().T + bg.abs()), n * (x.abs() @ wu.abs().T + bu.abs())
    a, d = act(g, kind)
    t_a = 1.2 * t_g + APPROX * a.abs()  # |act'| <= 1.13
    # |act''| <= 0.8 (gelu), 0.5 (silu); relu's derivative jumps at 0, where g's error decides it
    t_d = (g.abs() <= t_g).double() if kind == "relu" else t_g + APPROX * (1 + a.abs())
    return g, v, t_u, a, t_a, d, t_d


def gated(x, w, b, residual, kind, dtype):
    """(y, tolerance).  w = (gate, up, down), b = (gate, up, down), None = zeros."""
    x, (wg, wu, wd) = x.double(), (v.double() for v in w)
    bg, bu, bd = (torch.zeros(n, dtype=torch.float64, device=x.device) if v is None else v.double()
                  for v, n in zip(b, (wg.shape[0], wg.shape[0], wd.shape[0])))
    g, v, t_u, a, t_a, _, _ = _hidden(x, wg, wu, bg, bu, kind)
    h = a * v
    t_h = _rounded(h, t_a * (v.abs() + t_u) + a.abs() * t_u + 2 * U32 * h.abs(), dtype)
    y = h @ wd.T + bd
    t = t_h @ wd.abs().T + 2 * (h.shape[1] + 2) * U32 * ((h.abs() + t_h) @ wd.abs().T + bd.abs())
    if residual is not None:
        y = y + residual.double()
        t = t + 2 * U32 * (residual.double().abs() + y.abs())
    return y, t


def gated_back(x, w, b, dy, kind, dtype):
    """{name: (gradient, tolerance)}"""
    x, dy, (wg, wu, wd) = x.double(), dy.double(), (v.double() for v in w)
    R, H = x.shape[0], wg.shape[0]
    bg, bu = (torch.zeros(H, dtype=torch.float64, device=x.device) if v is None else v.double() for v in b[:2])
    g, v, t_u, a, t_a, d, t_d = _hidden(x, wg, wu, bg, bu, kind)
    dh = dy @ wd
    t_dh = 2 * (dy.shape[1] + 2) * U32 * (dy.abs() @ wd.abs())
    h, du, dg = a * v, dh * a, dh * v * d
    dha, va, aa, da = dh.abs() + t_dh, v.abs() + t_u, a.abs() + t_a, d.abs() + t_d
    t_h = _rounded(h, t_a * va + a.abs() * t_u + 2 * U32 * h.abs(), dtype)
    t_du = _rounded(du, t_dh * aa + dh.abs() * t_a + 2 * U32 * du.abs(), dtype)
    t_dg = _rounded(dg, t_dh * va * da + dha * t_u * da + dha * va * t_d + 4 * U32 * dg.abs(), dtype)
    kx, kr = 2 * (2 * H + 2) * U32, 2 * (R + 2) * U32

    def rows(p, t_p, q):  # p^T q over the rows
        return p.T @ q, t_p.T @ q.abs() + kr * ((p.abs() + t_p).T @ q.abs())
    one = torch.ones((R, 1), dtype=torch.float64, device=x.device)
    dwd, t_dwd = rows(h, t_h, dy)
    out = {"dx": (dg @ wg + du @ wu, t_dg @ wg.abs() + t_du @ wu.abs() + kx * ((dg.abs() + t_dg) @ wg.abs() + (du.abs() + t_du) @ wu.abs())),
           "dw_gate": rows(dg, t_dg, x), "dw_up": rows(du, t_du, x), "dw_down": (dwd.T, t_dwd.T)}
    for n, p, t in (("db_gate", dg, t_dg), ("db_up", du, t_du), ("db_down", dy, torch.zeros_like(dy))):
        s, ts = rows(p, t, one)
        out[n] = (s[:, 0], ts[:, 0])
    return out


# ---- whole numbers: sums that have to be exact ------------------------------------------------


def whole_numbers(R, D, H, seed, device="cpu"):
    """(x, w, b, dy) of a ReLU-gated block, as fp64 tensors, whose intermediate values are all small whole
    numbers: x, dy and biases of -1, 0, 1; four entries of +-1 a row of w_gate and w_up, three a column of w_down
    (fewer where places fall together).  So |g|, |u| <= 5, |dh| <= 3, |h| <= 25, |dg|, |du| <= 15, which fp16
    and bf16 hold, and every sum stays below 25 max(R, H) < 2^24, which fp32 adds without error in any order:
    the outputs are the exact sums, rounded once.  Signs are even-handed, so sums stay near sqrt(R) and one
    row too many or too few shows behind that rounding."""
    assert 25 * max(R, H) < 2 ** 24
    g = torch.Generator(device=device).manual_seed(seed)

    def small(*shape):
        return torch.randint(-1, 2, shape, generator=g, device=device).double()

    def few(rows, cols, n):
        at = torch.randint(cols, (rows, n), generator=g, device=device)
        sign = torch.randint(0, 2, (rows, n), generator=g, device=device).double() * 2 - 1
        return torch.zeros((rows, cols), dtype=torch.float64, device=device).scatter_(1, at, sign)
    return small(R, D), (few(H, D, 4), few(H, D, 4), few(H, D, 3).T.contiguous()), (small(H), small(H), small(D)), small(R, D)


def relu_gated(x, w, b, residual):
    return (x @ w[0].T + b[0]).clamp(min=0) * (x @ w[1].T + b[1]) @ w[2].T + b[2] + residual


def relu_gated_back(x, w, b, dy):
    """{name: gradient} in 64 bits."""
    g, u, dh = x @ w[0].T + b[0], x @ w[1].T + b[1], dy @ w[2]
    a, du, dg = g.clamp(min=0), dh * g.clamp(min=0), dh * u * (g > 0)
    return {"dx": dg @ w[0] + du @ w[1], "dw_gate": dg.T @ x, "dw_up": du.T @ x, "dw_down": dy.T @ (a * u),
            "db_gate": dg.sum(0), "db_up": du.sum(0), "db_down": dy.sum(0)}


def bias_grads(x, w, b, dy, kind):
    """{name: (bias gradient, tolerance)} where the rows' values are summed in fp32 before any rounding to 16
    bits: 32 rows by butterfly, then a chain of the blocks of at most R / 16 additions, then 32 + 32 partial sums."""
    x, dy, (wg, wu, wd) = x.double(), dy.double(), (v.double() for v in w)
    g, v, t_u, a, t_a, d, t_d = _hidden(x, wg, wu, b[0].double(), b[1].double(), kind)
    dh = dy @ wd
    t_dh = 2 * (dy.shape[1] + 2) * U32 * (dy.abs() @ wd.abs())
    du, dg = dh * a, dh * v * d
    dha, va, da = dh.abs() + t_dh, v.abs() + t_u, d.abs() + t_d
    t_du = t_dh * (a.abs() + t_a) + dh.abs() * t_a + 2 * U32 * du.abs()
    t_dg = t_dh * va * da + dha * t_u * da + dha * va * t_d + 4 * U32 * dg.abs()
    k = (x.shape[0] / 16 + 5 + 64) * U32
    return {n: (p.sum(0), (t + k * (p.abs() + t)).sum(0))
            for n, p, t in (("db_gate", dg, t_dg), ("db_up", du, t_du), ("db_down", dy, torch.zeros_like(dy)))}


# ---- the generator on whole tensors ------------------------------------------------------------


def kept(rng, first, n, threshold, device="cpu"):
    """Which of the elements first .. first + n - 1 dropout keeps (first: a multiple of 8), as one tensor
    computation: products of 32-bit words in int64, split at 16 bits."""
    blocks = first // 8 + torch.arange((n + 7) // 8, device=device)
    c = [blocks & M32, blocks >> 32, torch.full_like(blocks, int(rng[1]) & M32), torch.full_like(blocks, int(rng[1]) >> 32 & M32)]
    k = [int(rng[0]) & M32, int(rng[0]) >> 32 & M32]

    def wide(m, v):  # (high, low) words of m v
        low, high = m * (v & 0xFFFF), m * (v >> 16)
        high = high + (low >> 16)
        return high >> 16, (high & 0xFFFF) << 16 | (low & 0xFFFF)
    for _ in range(10):
        (h0, l0), (h1, l1) = wide(0xD2511F53, c[0]), wide(0xCD9E8D57, c[2])
        c = [h1 ^ c[1] ^ k[0], l1, h0 ^ c[3] ^ k[1], l0]
        k = [(k[0] + 0x9E3779B9) & M32, (k[1] + 0xBB67AE85) & M32]
    return (torch.stack([w >> s & 0xFFFF for w in c for s in (0, 16)], 1).reshape(-1)[:n] >= threshold)
