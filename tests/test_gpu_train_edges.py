"""Calls of the trainable sub-block that its documentation allows at the edges: tensors at any address their type allows,
between guard bytes; a workspace of exactly the size asked for; single tokens in graphs, weights written just
before; long chains without a wait; the widest layers."""
import ctypes as C

import pytest
import torch

import train_ref as ref
from prism_inference_b200.abi import GatedParams, NormParams

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
GRADS = ("dw_gate", "dw_up", "dw_down", "db_gate", "db_up", "db_down")


class Guarded:
    """Tensors cut out of buffers of a byte that nothing here writes; intact() says whether it is still all around them."""
    def __init__(self):
        self.all = []

    def __call__(self, shape, dtype, offset, like=None):
        """A contiguous tensor `offset` elements (of its type) behind a 256-byte boundary."""
        es, n = torch.empty(0, dtype=dtype).element_size(), 1
        for v in shape:
            n *= v
        first = 4096 + offset * es
        buf = torch.full((first + n * es + 4096,), 0xA5, dtype=torch.uint8, device="cuda")
        t = buf[first:first + n * es].view(dtype).view(shape)
        if like is not None:
            t.copy_(like)
        self.all.append((buf, first, first + n * es))
        return t

    def intact(self):
        return all(bool((b[:i] == 0xA5).all()) and bool((b[j:] == 0xA5).all()) for b, i, j in self.all)


def randn(shape, dtype, seed, std=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype).cuda()


def layer(D, H, dtype):
    w = [randn(s, dtype, i, s[1] ** -0.5) for i, s in enumerate(((H, D), (H, D), (D, H)))]
    return w, [randn((n,), dtype, 5 + i, 0.1) for i, n in enumerate((H, H, D))]


def asked(ctx, backward, **kw):
    n = C.c_size_t()
    assert ctx.lib.prism_gated_ffn_workspace(ctx.h, C.byref(GatedParams(**kw)), backward, C.byref(n)) == 0
    return n.value


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("shape", [(1, 64, 72), (5, 264, 136), (300, 72, 328), (700, 256, 512), (515, 520, 200), (300, 1000, 136)])
def test_gated_addresses_and_guards(prism_ctx, dtype, shape):
    """Row tensors and weights on 16-byte boundaries, biases and gradients on any 2-byte one, the workspace on a 16-byte
    one: the bits of the ordinary call, and nothing written around the outputs and the workspace."""
    R, D, H = shape
    w, b = layer(D, H, dtype)
    x, dy = randn((R, D), dtype, 11), randn((R, D), dtype, 12)
    y, dx = torch.empty_like(x), torch.empty_like(x)
    g = {n: torch.empty_like(t) for n, t in zip(GRADS, (*w, *b))}
    prism_ctx.gated_ffn(x, *w, y, b_gate=b[0], b_up=b[1], b_down=b[2], residual=dy)
    prism_ctx.gated_ffn_backward(x, *w, dy, dx, b_gate=b[0], b_up=b[1], **g)
    at = Guarded()
    w1, b1 = [at(t.shape, dtype, 8 * (2 * i + 1), t) for i, t in enumerate(w)], [at(t.shape, dtype, 1 + 2 * i, t) for i, t in enumerate(b)]
    x1, dy1, y1, dx1 = (at(x.shape, dtype, 8 * o, t) for o, t in ((1, x), (3, dy), (5, None), (7, None)))
    g1 = {n: at(t.shape, dtype, 1 + i) for i, (n, t) in enumerate(g.items())}
    sizes = dict(rows=R, dim=D, hidden=H, dtype=0 if dtype is F16 else 1, x_stride=D, y_stride=D, dy_stride=D, dx_stride=D)
    ws = [at((asked(prism_ctx, k, **sizes),), torch.uint8, 16 + 32 * k) for k in (0, 1)]
    prism_ctx.gated_ffn(x1, *w1, y1, b_gate=b1[0], b_up=b1[1], b_down=b1[2], residual=dy1, workspace=ws[0])
    prism_ctx.gated_ffn_backward(x1, *w1, dy1, dx1, b_gate=b1[0], b_up=b1[1], workspace=ws[1], **g1)
    prism_ctx.status()
    assert torch.equal(y, y1) and torch.equal(dx, dx1) and all(torch.equal(g[n], g1[n]) for n in GRADS) and at.intact()
    prism_ctx.gated_ffn(x1, *w1, dy1, b_gate=b1[0], b_up=b1[1], b_down=b1[2], residual=dy1, workspace=ws[0])  # on the residual itself
    assert torch.equal(y, dy1) and at.intact()


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("shape", [(1, 1), (3, 17), (700, 64), (2000, 101), (300, 1000), (37, 4100)])
def test_row_op_addresses_and_guards(prism_ctx, dtype, shape):
    R, D = shape
    x, dy, add = (randn(shape, dtype, i) for i in range(3))
    w, b = randn((D,), F32, 3), randn((D,), F32, 4)
    rng = torch.tensor([77, -9], device="cuda")

    def run(x, dy, add, w, b, out, ws):
        y, dx, z, mean, rstd, dw, db = out
        prism_ctx.layer_norm(x, w, b, y, mean=mean, rstd=rstd)
        prism_ctx.layer_norm_backward(x, w, mean, rstd, dy, dx, dweight=dw, dbias=db, add=add, workspace=ws)
        prism_ctx.dropout_add(x, dy, z, 0.3, rng)
        return out
    like = (x, x, x, x.new_empty(R, dtype=F32), x.new_empty(R, dtype=F32), w, b)
    want = run(x, dy, add, w, b, [torch.empty_like(t) for t in like], None)
    n = C.c_size_t()
    p = NormParams(rows=R, dim=D, dtype=(F16, BF16, F32).index(dtype), param_dtype=2)
    assert prism_ctx.lib.prism_layer_norm_backward_workspace(prism_ctx.h, C.byref(p), C.byref(n)) == 0
    for k in (1, 3, 5):
        at = Guarded()
        ins = [at(t.shape, t.dtype, o, t) for t, o in ((x, k), (dy, k + 1), (add, 2 * k), (w, k), (b, k + 2))]
        out = [at(t.shape, t.dtype, k + i) for i, t in enumerate(like)]
        got = run(*ins, out, at((n.value,), torch.uint8, 16 * k))
        # another kernel by the rows' alignment, so within the tolerances; dropout is element by element, the same bits
        r, tol = ref.norm(x, w, b, 1e-5)
        for i, v, t, name in zip((0, 3, 4), r, tol, ("y", "mean", "rstd")):
            ref.check(got[i], v, t, name)
        r, tol = ref.norm_back(x, w, got[3], got[4], dy, add)
        for i, v, t, name in zip((1, 5, 6), r, tol, ("dx", "dweight", "dbias")):
            ref.check(got[i], v, t, name)
        assert torch.equal(want[2], got[2])
        assert at.intact()


@pytest.mark.parametrize("rows", [1, 2, 5, 8, 9])
def test_tokens_in_a_graph_with_changing_weights(prism_ctx, rows):
    """A graph that writes weights and tokens and runs the block at once: each replay sees what it wrote."""
    D, H = 256, 512
    w, b = layer(D, H, F16)
    new = [[randn(t.shape, F16, 100 * k + i, t.shape[1] ** -0.5) for i, t in enumerate(w)] for k in range(4)]
    xs = [randn((rows, D), F16, 50 + k) for k in range(4)]
    want = [prism_ctx.gated_ffn(x, *n, torch.empty_like(x), b_gate=b[0], b_up=b[1], b_down=b[2], residual=x) for x, n in zip(xs, new)]
    torch.cuda.synchronize()
    src, x, y = [t.clone() for t in w], torch.empty_like(xs[0]), torch.empty_like(xs[0])
    xin = torch.empty_like(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for t, s in zip(w, src):
            t.copy_(s)
        torch.add(xin, 0, out=x)  # a kernel right before the block
        prism_ctx.gated_ffn(x, *w, y, b_gate=b[0], b_up=b[1], b_down=b[2], residual=x)
    got = []
    for k in range(16):
        for s, n in zip(src, new[k % 4]):
            s.copy_(n)
        xin.copy_(xs[k % 4])
        graph.replay()
        got.append(y.clone())
    for k in range(16):  # and without a graph, w_down written by the kernel right before
        for t, n in zip(w, new[k % 4]):
            torch.add(n, 0, out=t)
        got.append(prism_ctx.gated_ffn(xs[k % 4], *w, torch.empty_like(x), b_gate=b[0], b_up=b[1], b_down=b[2], residual=xs[k % 4]))
    assert all(torch.equal(g, want[k % 4]) for k, g in enumerate(got))


@pytest.mark.parametrize("shape", [(1, 256, 512), (8, 256, 1024), (300, 256, 512), (9000, 128, 256), (300, 264, 512)])
def test_long_chains_without_a_wait(prism_ctx, shape):
    """Forty layers one after the other in place, and their backward calls, queued at once: the bits of the same calls
    with a wait after each."""
    R, D, H = shape
    w, b = layer(D, H, BF16)
    gamma, beta = torch.ones(D, device="cuda"), torch.zeros(D, device="cuda")

    def chain(wait):
        x, n, g = randn((R, D), BF16, 1), torch.empty(R, D, dtype=BF16, device="cuda"), randn((R, D), BF16, 2)
        mean, rstd, dn, dh = torch.empty(R, device="cuda"), torch.empty(R, device="cuda"), torch.empty_like(n), torch.empty_like(n)
        dw, rng = [torch.empty_like(t) for t in (*w, *b)], torch.tensor([1, 0], device="cuda")
        sums = [torch.zeros_like(t, dtype=F32) for t in dw]
        for k in range(40):
            prism_ctx.layer_norm(x, gamma, beta, n, mean=mean, rstd=rstd)
            prism_ctx.gated_ffn(n, *w, dh, b_gate=b[0], b_up=b[1], b_down=b[2])
            prism_ctx.dropout_add(dh, x, x, 0.1, rng)
            prism_ctx.dropout_add(g, None, dh, 0.1, rng)
            prism_ctx.gated_ffn_backward(n, *w, dh, dn, b_gate=b[0], b_up=b[1], **dict(zip(GRADS, dw)))
            prism_ctx.layer_norm_backward(n, gamma, mean, rstd, dn, g, add=g)
            for s, t in zip(sums, dw):
                s += t
            rng[1] += 1
            if wait:
                torch.cuda.synchronize()
        return [x, g, *sums]
    slow = chain(True)
    for _ in range(2):
        assert all(torch.equal(p.nan_to_num(), q.nan_to_num()) for p, q in zip(slow, chain(False)))
    assert torch.isfinite(slow[0]).all()
    prism_ctx.status()


@pytest.mark.parametrize("shape", [(1, 16384, 2048), (300, 16384, 2048), (1, 256, 65536), (300, 256, 65536), (300, 264, 65536), (9, 16384, 8)])
def test_the_widest_layers(prism_ctx, shape):
    R, D, H = shape
    x, w, b, dy = ref.whole_numbers(R, D, H, 9, "cuda")
    wl, bl = [t.to(F16) for t in w], [t.to(F16) for t in b]
    xs, dys = x.to(F16), dy.to(F16)
    y, dx = torch.empty_like(xs), torch.empty_like(xs)
    prism_ctx.gated_ffn(xs, *wl, y, b_gate=bl[0], b_up=bl[1], b_down=bl[2], residual=dys, activation="relu")
    assert torch.equal(y, ref.relu_gated(x, w, b, dy).float().to(F16))
    want = ref.relu_gated_back(x, w, b, dy)
    g = {n: torch.empty(want[n].shape, dtype=F16, device="cuda") for n in GRADS}
    prism_ctx.gated_ffn_backward(xs, *wl, dys, dx, b_gate=bl[0], b_up=bl[1], activation="relu", **g)
    prism_ctx.status()
    assert torch.equal(dx, want["dx"].float().to(F16))
    for n in GRADS:
        assert torch.equal(g[n], want[n].float().to(F16)), n


def test_the_default_streams_handle(prism_ctx):
    """torch.cuda.current_stream().cuda_stream is 0 on the default stream: as good as the stream object, scratch included."""
    D, H = 128, 256
    w, b = layer(D, H, F16)
    x = randn((300, D), F16, 1)
    m, r, out = torch.zeros(300, device="cuda"), torch.ones(300, device="cuda"), []
    for s in (None, torch.cuda.current_stream(), torch.cuda.current_stream().cuda_stream, torch.cuda.Stream(), torch.cuda.Stream().cuda_stream):
        torch.cuda.synchronize()
        y, dx, dn, dw, dg = torch.empty_like(x), torch.empty_like(x), torch.empty_like(x), torch.empty_like(w[0]), torch.empty(D, device="cuda")
        tok = torch.empty_like(x[:3])
        torch.cuda.synchronize()
        prism_ctx.gated_ffn(x, *w, y, stream=s)
        prism_ctx.gated_ffn(x[:3], *w, tok, stream=s)
        prism_ctx.gated_ffn_backward(x, *w, y, dx, dw_gate=dw, stream=s)
        prism_ctx.layer_norm_backward(x, None, m, r, y, dn, dweight=dg, stream=s)
        torch.cuda.synchronize()
        out.append((y, tok, dx, dw, dn, dg))
    assert all(torch.equal(p, q) for o in out[1:] for p, q in zip(out[0], o))
