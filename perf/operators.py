"""The trainable pre-norm gated feed-forward sub-block: layer norm, dropout with the residual add, and the gated
feed-forward block, each in both directions.

    n = LN(x);  h = W_d (act(W_g n + b_g) * (W_u n + b_u)) + b_d;  y = x + dropout(h)

Sizes are those of the bottleneck: 64-token windows, 68 x 120 = 8160 tokens a frame, dim 128 or 256, hidden 512 or 1024, 1 to 64
frames; and generic ones beside them.
"""
import functools
import math

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
BYTES = {"fp16": 2, "bf16": 2, "fp32": 4}
FRAME = 68 * 120
EPS = 1e-5
GELU_C, GELU_A = math.sqrt(2.0 / math.pi), 0.044715


def listed():
    return [
        # one window of tokens before its block: the smallest call, where latency counts
        dict(name="norm window", op="norm", rows=64, dim=256, dtype="fp16", params="fp16", pad=0),
        # the norm of a full batch of 64 frames
        dict(name="norm 64 frames", op="norm", rows=64 * FRAME, dim=256, dtype="fp16", params="fp16", pad=0),
        # a training step's norm on 16 frames: the gradient joins the one that came past the block
        dict(name="norm back 16 frames", op="norm_back", rows=16 * FRAME, dim=256, dtype="bf16", params="fp32", pad=0, add=True),
        # a wide model's rows, odd counts, in 32 bits, rows of a wider buffer
        dict(name="norm back odd fp32", op="norm_back", rows=4099, dim=1001, dtype="fp32", params="fp32", pad=23, add=False),
        # the gradient of one frame through the mask (no residual)
        dict(name="dropout frame", op="dropout", rows=FRAME, dim=128, dtype="fp16", p=0.1, residual=False, pad=0),
        # 64 frames' block output dropped and added to the residual stream
        dict(name="dropout add 64 frames", op="dropout", rows=64 * FRAME, dim=256, dtype="bf16", p=0.2, residual=True, pad=0),
        # serving: one token
        dict(name="ffn token", op="ffn", rows=1, dim=256, hidden=1024, dtype="fp16", act="gelu", residual=True, pad=0),
        # serving: one frame
        dict(name="ffn frame", op="ffn", rows=FRAME, dim=256, hidden=1024, dtype="fp16", act="gelu", residual=True, pad=0),
        # throughput: 64 frames
        dict(name="ffn 64 frames", op="ffn", rows=64 * FRAME, dim=256, hidden=1024, dtype="fp16", act="silu", residual=True, pad=0),
        # a training step of the narrow model on one frame
        dict(name="ffn back frame", op="ffn_back", rows=FRAME, dim=128, hidden=512, dtype="bf16", act="gelu", pad=0),
        # a training step on 16 frames
        dict(name="ffn back 16 frames", op="ffn_back", rows=16 * FRAME, dim=256, hidden=1024, dtype="bf16", act="silu", pad=0),
        # a generic wide block on a ragged batch whose rows lie in a wider buffer
        dict(name="ffn back ragged wide", op="ffn_back", rows=2051, dim=1000, hidden=2744, dtype="bf16", act="silu", pad=24),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "norm_back", "dropout", "ffn", "ffn_back"])
    if op in ("ffn", "ffn_back"):
        dim, hidden = 8 * _log(rng, 2, 128), 8 * _log(rng, 2, 512)
        most = (64 if op == "ffn" else 16) * FRAME * 256 * 1024
        rows = _log(rng, 1, max(1, min(64 * FRAME, most // (dim * hidden))))
        c = dict(op=op, rows=rows, dim=dim, hidden=hidden, dtype=rng.choice(["fp16", "bf16"]), act=rng.choice(["gelu", "silu", "relu"]), pad=rng.choice([0, 0, 8, 40]))
        return dict(c, residual=rng.random() < 0.5) if op == "ffn" else c
    dim = _log(rng, 8, 4096)
    rows = _log(rng, 1, 64 * FRAME * 256 // max(256, dim) // (1 if op != "norm_back" else 2))
    dtype = rng.choice(["fp16", "bf16", "fp32"])
    c = dict(op=op, rows=rows, dim=dim, dtype=dtype, pad=rng.choice([0, 0, 8, 13]))
    if op == "dropout":
        return dict(c, p=round(rng.uniform(0.0, 0.7), 3), residual=rng.random() < 0.5)
    c["params"] = rng.choice([dtype, "fp32"])
    return dict(c, add=rng.random() < 0.5) if op == "norm_back" else c


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, R, D = DTYPES[case["dtype"]], case["rows"], case["dim"]

    def normal(*shape, std=1.0):
        return torch.randn(shape, generator=g, device="cuda") * std

    def rows(t):
        """`t` as the first columns of a buffer whose rows are `pad` values longer."""
        if not case["pad"]:
            return t.to(dt)
        wide = torch.zeros((t.shape[0], t.shape[1] + case["pad"]), dtype=dt, device="cuda")
        wide[:, : t.shape[1]] = t
        return wide[:, : t.shape[1]]

    op = case["op"]
    s = dict(case=case)
    if op in ("norm", "norm_back"):
        pt = DTYPES[case["params"]]
        # a residual stream: channels of unlike scale around an offset
        s["x"] = rows(normal(R, D) * (0.5 + torch.rand(D, generator=g, device="cuda")) + normal(D, std=0.3))
        s["weight"], s["bias"] = (1 + normal(D, std=0.2)).to(pt), normal(D, std=0.2).to(pt)
        if op == "norm_back":
            s["dy"] = rows(normal(R, D))
            s["add"] = rows(normal(R, D)) if case["add"] else None
            x = s["x"].float()  # the statistics that the forward pass kept
            s["mean"] = x.mean(1)
            s["rstd"] = torch.rsqrt((x - s["mean"][:, None]).square().mean(1) + EPS)
    elif op == "dropout":
        s["x"] = rows(normal(R, D))
        s["residual"] = rows(normal(R, D)) if case["residual"] else None
        # the generator's state (seed, offset), 64 bits each
        s["rng"] = torch.randint(-(2**63), 2**63 - 1, (2,), generator=g, device="cuda", dtype=torch.int64)
    else:
        H = case["hidden"]
        s["x"] = rows(normal(R, D))
        s["w_gate"], s["w_up"] = normal(H, D, std=D**-0.5).to(dt), normal(H, D, std=D**-0.5).to(dt)
        s["w_down"] = normal(D, H, std=H**-0.5).to(dt)
        s["b_gate"], s["b_up"] = normal(H, std=0.1).to(dt), normal(H, std=0.1).to(dt)
        if op == "ffn":
            s["b_down"] = normal(D, std=0.1).to(dt)
            s["residual"] = rows(normal(R, D)) if case["residual"] else None
        else:
            s["dy"] = rows(normal(R, D))
    return s


# ---- the plain forms -------------------------------------------------------------------------


def _norm(s):
    dt, x = s["x"].dtype, s["x"].float()
    mean = x.mean(1)
    c = x - mean[:, None]
    rstd = torch.rsqrt(c.square().mean(1) + EPS)
    y = c * rstd[:, None] * s["weight"].float() + s["bias"].float()
    return {"y": y.to(dt), "mean": mean, "rstd": rstd}


def _norm_back(s):
    dt, pt = s["x"].dtype, s["weight"].dtype
    dy = s["dy"].float()
    xh = (s["x"].float() - s["mean"][:, None]) * s["rstd"][:, None]
    g = dy * s["weight"].float()
    dx = s["rstd"][:, None] * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    if s["add"] is not None:
        dx = dx + s["add"].float()
    return {"dx": dx.to(dt), "dweight": (dy * xh).sum(0, dtype=torch.float64).to(pt), "dbias": dy.sum(0, dtype=torch.float64).to(pt)}


M32 = 0xFFFFFFFF


def _mulhilo(a, b):
    """(high, low) 32 bits of the product of a 32-bit constant and 32-bit words that int64 holds."""
    lo = (a & 0xFFFF) * b
    hi = (a >> 16) * b + (lo >> 16)
    return hi >> 16, ((hi & 0xFFFF) << 16) | (lo & 0xFFFF)


def _keep(rng, rows, dim, threshold):
    """The mask of a rows x dim tensor: element i takes 16 bits of the Philox4x32-10 block i / 8 (Salmon et al., 2011)."""
    n = rows * dim
    block = torch.arange((n + 7) // 8, device=rng.device, dtype=torch.int64)
    k0, k1, o0, o1 = rng[0] & M32, (rng[0] >> 32) & M32, rng[1] & M32, (rng[1] >> 32) & M32
    c0, c1, c2, c3 = block & M32, block >> 32, o0.expand_as(block), o1.expand_as(block)
    for _ in range(10):
        h0, l0 = _mulhilo(0xD2511F53, c0)
        h1, l1 = _mulhilo(0xCD9E8D57, c2)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & M32, (k1 + 0xBB67AE85) & M32
    bits = torch.stack([c0 & 0xFFFF, c0 >> 16, c1 & 0xFFFF, c1 >> 16, c2 & 0xFFFF, c2 >> 16, c3 & 0xFFFF, c3 >> 16], 1)
    return (bits.reshape(-1)[:n] >= threshold).reshape(rows, dim)


def _dropout(s):
    x, t = s["x"].float(), int(round(65536 * s["case"]["p"]))
    y = torch.where(_keep(s["rng"], x.shape[0], x.shape[1], t), x * (65536 / (65536 - t)), 0.0)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return {"y": y.to(s["x"].dtype)}


def _gate(g, act):
    """act(g) and its derivative."""
    if act == "relu":
        return torch.relu(g), (g > 0).to(g.dtype)
    if act == "silu":
        z = torch.sigmoid(g)
        return g * z, z * (1 + g * (1 - z))
    t = torch.tanh(GELU_C * (g + GELU_A * g * g * g))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * GELU_C * (1 + 3 * GELU_A * g * g)


def _ffn(s):
    dt, x = s["x"].dtype, s["x"].float()
    a, _ = _gate(x @ s["w_gate"].float().T + s["b_gate"].float(), s["case"]["act"])
    y = (a * (x @ s["w_up"].float().T + s["b_up"].float())) @ s["w_down"].float().T + s["b_down"].float()
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return {"y": y.to(dt)}


def _ffn_back(s):
    dt, x, dy = s["x"].dtype, s["x"].float(), s["dy"].float()
    wg, wu = s["w_gate"].float(), s["w_up"].float()
    a, da = _gate(x @ wg.T + s["b_gate"].float(), s["case"]["act"])
    u = x @ wu.T + s["b_up"].float()
    dh = dy @ s["w_down"].float()
    dg, du = dh * u * da, dh * a
    out = {"dx": dg @ wg + du @ wu, "dw_gate": dg.T @ x, "dw_up": du.T @ x, "dw_down": dy.T @ (a * u),
           "db_gate": dg.sum(0, dtype=torch.float64), "db_up": du.sum(0, dtype=torch.float64), "db_down": dy.sum(0, dtype=torch.float64)}
    return {k: v.to(dt) for k, v in out.items()}


# ---- the framework's calls -------------------------------------------------------------------


@functools.lru_cache(None)
def _ctx(device):
    from prism_inference_b200 import Prism
    return Prism(device)


def _own(s):
    c, x = s["case"], s["x"]
    ctx, op = _ctx(x.device.index), c["op"]
    if op == "norm":
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        mean, rstd = torch.empty((2, x.shape[0]), dtype=torch.float32, device=x.device)
        ctx.layer_norm(x, s["weight"], s["bias"], y, eps=EPS, mean=mean, rstd=rstd)
        return {"y": y, "mean": mean, "rstd": rstd}
    if op == "norm_back":
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        dw, db = torch.empty_like(s["weight"]), torch.empty_like(s["weight"])
        ctx.layer_norm_backward(x, s["weight"], s["mean"], s["rstd"], s["dy"], dx, dweight=dw, dbias=db, add=s["add"])
        return {"dx": dx, "dweight": dw, "dbias": db}
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if op == "dropout":
        ctx.dropout_add(x, s["residual"], y, c["p"], s["rng"])
        return {"y": y}
    weights = (s["w_gate"], s["w_up"], s["w_down"])
    if op == "ffn":
        ctx.gated_ffn(x, *weights, y, b_gate=s["b_gate"], b_up=s["b_up"], b_down=s["b_down"], residual=s["residual"], activation=c["act"])
        return {"y": y}
    dwg, dwu, dwd = (torch.empty_like(w) for w in weights)
    dbg, dbu, dbd = torch.empty_like(s["b_gate"]), torch.empty_like(s["b_up"]), torch.empty(x.shape[1], dtype=x.dtype, device=x.device)
    ctx.gated_ffn_backward(x, *weights, s["dy"], y, dwg, dwu, dwd, b_gate=s["b_gate"], b_up=s["b_up"], db_gate=dbg, db_up=dbu, db_down=dbd, activation=c["act"])
    return {"dx": y, "dw_gate": dwg, "dw_up": dwu, "dw_down": dwd, "db_gate": dbg, "db_up": dbu, "db_down": dbd}


def run(state):
    if own:
        return _own(state)
    return {"norm": _norm, "norm_back": _norm_back, "dropout": _dropout, "ffn": _ffn, "ffn_back": _ffn_back}[state["case"]["op"]](state)


def work(case):
    R, D, s, op = case["rows"], case["dim"], BYTES[case["dtype"]], case["op"]
    t = R * D * s
    if op == "norm":
        return {"bytes": 2 * t + 8 * R + 2 * D * BYTES[case["params"]], "flops": 8 * R * D}
    if op == "norm_back":
        return {"bytes": (3 + case["add"]) * t + 8 * R + 3 * D * BYTES[case["params"]], "flops": 14 * R * D}
    if op == "dropout":
        return {"bytes": (2 + case["residual"]) * t + 16, "flops": 2 * R * D}
    H = case["hidden"]
    if op == "ffn":
        return {"bytes": (2 + case["residual"]) * t + s * (3 * D * H + 2 * H + D), "flops": 6 * R * D * H}
    # the gate's and the up projection's products are part of what a backward pass from x has to compute
    return {"bytes": 3 * t + 2 * s * (3 * D * H + 2 * H) + s * D, "flops": 16 * R * D * H}


# ---- the definition in 64 bits -----------------------------------------------------------------


def _exact_act(v, act):
    if act == "relu":
        return v.clamp(min=0), torch.where(v > 0, 1.0, 0.0).to(v.dtype)
    if act == "silu":
        e = torch.exp(-v)
        return v / (1 + e), (1 + e + v * e) / (1 + e).square()
    inner, slope = 2 * GELU_C * (v + GELU_A * v**3), 2 * GELU_C * (1 + 3 * GELU_A * v**2)
    z = 1 / (1 + torch.exp(-inner))
    return v * z, z + v * z * (1 - z) * slope


def _exact_bits(seed, offset, first, count, device):
    """16-bit draws first .. first + 8 count - 1, the generator written with products split at 16 bits."""
    i = torch.arange(first, first + count, device=device, dtype=torch.int64)
    ctr = [i & M32, i >> 32, torch.full_like(i, offset & M32), torch.full_like(i, (offset >> 32) & M32)]
    key = [seed & M32, (seed >> 32) & M32]

    def high(a, b):
        ah, al, bh, bl = a >> 16, a & 0xFFFF, b >> 16, b & 0xFFFF
        mid = ah * bl + ((al * bl) >> 16)
        return ah * bh + (mid >> 16) + (((mid & 0xFFFF) + al * bh) >> 16)

    for r in range(10):
        p, q = ctr[0], ctr[2]
        a, b = 0xD2511F53, 0xCD9E8D57
        ctr = [high(b, q) ^ ctr[1] ^ ((key[0] + r * 0x9E3779B9) & M32), (b * q) & M32, high(a, p) ^ ctr[3] ^ ((key[1] + r * 0xBB67AE85) & M32), (a * p) & M32]
    return torch.stack([(w >> k) & 0xFFFF for w in ctr for k in (0, 16)], 1).reshape(-1)


def exact(case, seed):
    s = prepare(case, seed)
    op, R, D = case["op"], case["rows"], case["dim"]
    step = max(1, 2**25 // max(D, case.get("hidden", 0)))  # rows at a time
    parts = [slice(a, min(R, a + step)) for a in range(0, R, step)]
    w = {k: v.double() for k, v in s.items() if k.startswith(("w", "b_", "bias"))}
    if op == "norm":
        y, stats = [], []
        for p in parts:
            x = s["x"][p].double()
            var, mean = torch.var_mean(x, 1, unbiased=False)
            y.append((x - mean[:, None]) / torch.sqrt(var + EPS)[:, None] * w["weight"] + w["bias"])
            stats.append((mean, 1 / torch.sqrt(var + EPS)))
        return {"y": torch.cat(y), "mean": torch.cat([a for a, _ in stats]), "rstd": torch.cat([b for _, b in stats])}
    if op == "norm_back":
        dx, dw, db = [], 0, 0
        for p in parts:
            dy, m, r = s["dy"][p].double(), s["mean"][p].double()[:, None], s["rstd"][p].double()[:, None]
            n = (s["x"][p].double() - m) * r
            g = dy * w["weight"]
            d = (g - g.sum(1, keepdim=True) / D - n * ((g * n).sum(1, keepdim=True) / D)) * r
            dx.append(d + s["add"][p].double() if s["add"] is not None else d)
            dw, db = dw + (dy * n).sum(0), db + dy.sum(0)
        return {"dx": torch.cat(dx), "dweight": dw, "dbias": db}
    if op == "dropout":
        t = int(round(65536 * case["p"]))
        sd, off = s["rng"].tolist()
        n, y = R * D, []
        for a in range(0, n, 2**26):
            m = min(n, a + 2**26) - a
            keep = _exact_bits(sd, off, a // 8, (m + 7) // 8, "cuda")[:m] >= t
            y.append(keep)
        keep = torch.cat(y).reshape(R, D)
        out = s["x"].double() * keep / (1 - t / 65536)
        return {"y": out + s["residual"].double() if s["residual"] is not None else out}
    if op == "ffn":
        y = []
        for p in parts:
            x = s["x"][p].double()
            a, _ = _exact_act(torch.addmm(w["b_gate"], x, w["w_gate"].T), case["act"])
            o = torch.addmm(w["b_down"], a * torch.addmm(w["b_up"], x, w["w_up"].T), w["w_down"].T)
            y.append(o + s["residual"][p].double() if s["residual"] is not None else o)
        return {"y": torch.cat(y)}
    dx, sums = [], None
    for p in parts:
        x, dy = s["x"][p].double(), s["dy"][p].double()
        a, slope = _exact_act(torch.addmm(w["b_gate"], x, w["w_gate"].T), case["act"])
        u = torch.addmm(w["b_up"], x, w["w_up"].T)
        dh = dy @ w["w_down"]
        du, dg = dh * a, dh * u * slope
        dx.append(torch.addmm(du @ w["w_up"], dg, w["w_gate"]))
        new = [dg.T @ x, du.T @ x, dy.T @ (a * u), dg.sum(0), du.sum(0), dy.sum(0)]
        sums = new if sums is None else [i + j for i, j in zip(sums, new)]
    return dict(zip(("dx", "dw_gate", "dw_up", "dw_down", "db_gate", "db_up", "db_down"), [torch.cat(dx)] + sums))
