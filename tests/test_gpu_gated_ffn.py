"""The gated feed-forward block, forward and backward, on the GPU through the public calls, against plain
64-bit forms; and the sub-block it belongs to as a training step runs it."""
import pytest
import torch

import train_ref as ref
from prism_inference_b200.abi import PrismError

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16
GRADS = ("dw_gate", "dw_up", "dw_down", "db_gate", "db_up", "db_down")


def rand(shape, dtype, seed, pad=0, std=1.0):
    g = torch.Generator().manual_seed(seed)
    t = torch.full((shape[0], shape[1] + pad), 7.0, dtype=dtype)
    t[:, :shape[1]] = (torch.randn(shape, generator=g) * std).to(dtype)
    return t.cuda()[:, :shape[1]]


def empty(shape, dtype, pad=0):
    return torch.full((shape[0], shape[1] + pad), 7.0, dtype=dtype, device="cuda")[:, :shape[1]]


def pad_untouched(t):
    base = t._base if t._base is not None else t
    return bool((base[:, t.shape[1]:] == 7.0).all())


def weights(D, H, dtype, seed=50, bias=True):
    w = (rand((H, D), dtype, seed, std=D ** -0.5), rand((H, D), dtype, seed + 1, std=D ** -0.5),
         rand((D, H), dtype, seed + 2, std=H ** -0.5))
    w = tuple(t.contiguous() for t in w)
    b = tuple(rand((1, n), dtype, seed + 3 + i, std=0.1)[0].contiguous() for i, n in enumerate((H, H, D))) if bias else (None,) * 3
    return w, b


def forward(ctx, x, w, b, y, **kw):
    return ctx.gated_ffn(x, *w, y, b_gate=b[0], b_up=b[1], b_down=b[2], **kw)


def grads_like(w, H, D):
    f = lambda *s: torch.full(s, 7.0, dtype=w[0].dtype, device="cuda")  # noqa: E731
    return {"dw_gate": f(H, D), "dw_up": f(H, D), "dw_down": f(D, H), "db_gate": f(H), "db_up": f(H), "db_down": f(D)}


def backward(ctx, x, w, b, dy, dx, grads, **kw):
    return ctx.gated_ffn_backward(x, *w, dy, dx, b_gate=b[0], b_up=b[1], **grads, **kw)


SHAPES = [(1, 8, 8), (2, 264, 40), (4, 256, 1024), (8, 1000, 2744), (9, 256, 512), (1, 256, 1024), (3, 64, 64), (16, 256, 512), (17, 128, 136), (64, 256, 1024), (129, 128, 512), (130, 72, 200),
          (257, 256, 256), (300, 264, 328), (1000, 128, 512), (77, 1000, 2744), (515, 520, 72), (5, 1024, 4096), (19000, 64, 128),
          (19000, 16, 9600)]  # the last one's backward pass goes through in two chunks of rows


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("kind,pad,res", [("gelu", 0, True), ("silu", 8, False), ("relu", 40, True)])
def test_forward(prism_ctx, dtype, shape, kind, pad, res):
    R, D, H = shape
    x = rand((R, D), dtype, R + D, pad)
    w, b = weights(D, H, dtype, bias=kind != "silu" or R % 2 == 1)
    r = rand((R, D), dtype, 3, pad) if res else None
    y = empty((R, D), dtype, pad)
    forward(prism_ctx, x, w, b, y, residual=r, activation=kind)
    prism_ctx.status()
    want, tol = ref.gated(x, w, b, r, kind, dtype)
    ref.check(y, want, tol, "y")
    assert pad_untouched(y)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("kind,pad", [("gelu", 0), ("silu", 8), ("relu", 40)])
def test_backward(prism_ctx, dtype, shape, kind, pad):
    R, D, H = shape
    x, dy = rand((R, D), dtype, R + D, pad), rand((R, D), dtype, R + D + 1, pad)
    w, b = weights(D, H, dtype, bias=kind != "silu" or R % 2 == 1)
    dx, grads = empty((R, D), dtype, pad), grads_like(w, H, D)
    backward(prism_ctx, x, w, b, dy, dx, grads, activation=kind)
    prism_ctx.status()
    want = ref.gated_back(x, w, b, dy, kind, dtype)
    ref.check(dx, *want["dx"], "dx")
    for n in GRADS:
        ref.check(grads[n], *want[n], n)
    assert pad_untouched(dx)


def test_forward_in_chunks(prism_ctx):
    """dim > 256 and a hidden layer so wide that the rows go through in two chunks."""
    R, D, H = 19000, 264, 14344
    x, (w, b) = rand((R, D), F16, 1), weights(D, H, F16)
    y = empty((R, D), F16)
    forward(prism_ctx, x, w, b, y, residual=x)
    for part in (slice(0, 300), slice(18800, R)):
        want, tol = ref.gated(x[part], w, b, x[part], "gelu", F16)
        ref.check(y[part], want, tol, "y")


@pytest.mark.parametrize("shape", [(200, 128, 256), (200, 264, 72)])
def test_backward_gradients_are_optional(prism_ctx, shape):
    R, D, H = shape
    x, dy = rand((R, D), BF16, 1), rand((R, D), BF16, 2)
    w, b = weights(D, H, BF16)
    dx, grads = empty((R, D), BF16), grads_like(w, H, D)
    backward(prism_ctx, x, w, b, dy, dx, grads)
    for n in GRADS + (None,):
        one = {n: torch.full_like(grads[n], 7.0)} if n else {}
        dx1 = empty((R, D), BF16)
        backward(prism_ctx, x, w, b, dy, dx1, one)
        assert torch.equal(dx, dx1) and all(torch.equal(one[k], grads[k]) for k in one), n


def test_three_dimensions_and_residual_in_place(prism_ctx):
    D, H = 256, 512
    x = rand((120, D), F16, 1).reshape(2, 60, D)
    w, b = weights(D, H, F16)
    r = rand((120, D), F16, 2).reshape(2, 60, D)
    y = torch.empty_like(x)
    forward(prism_ctx, x, w, b, y, residual=r)
    forward(prism_ctx, x, w, b, r, residual=r)
    assert torch.equal(y, r)


@pytest.mark.parametrize("dim", [256, 264])
def test_residual_in_place_and_column_slices_over_many_tiles(prism_ctx, dim):
    """y as the residual itself, and x, residual and y as column slices of one buffer, with more row tiles than
    CTA pairs: a tile's output must not reach what another still reads."""
    R, H = 20000, 128
    w, b = weights(dim, H, F16)
    wide = rand((R, 3 * dim), F16, 4)
    x, r, y = wide[:, :dim], wide[:, dim:2 * dim], wide[:, 2 * dim:]
    want = torch.empty((R, dim), dtype=F16, device="cuda")
    forward(prism_ctx, x.contiguous(), w, b, want, residual=r.contiguous())
    forward(prism_ctx, x, w, b, y, residual=r)
    assert torch.equal(y, want)
    forward(prism_ctx, x, w, b, r, residual=r)
    assert torch.equal(r, want)


def test_two_graphs_at_once(prism_ctx):
    """Two captured steps replayed on two streams at the same time share no workspace."""
    R, D, H = 3000, 256, 512
    w, b = weights(D, H, BF16)
    made = []
    for seed in (1, 2):
        x = rand((R, D), BF16, seed)
        y, dx, g = torch.empty_like(x), torch.empty_like(x), grads_like(w, H, D)
        want = (torch.empty_like(x), torch.empty_like(x), grads_like(w, H, D))
        forward(prism_ctx, x, w, b, want[0])
        backward(prism_ctx, x, w, b, x, want[1], want[2])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            forward(prism_ctx, x, w, b, y)
            backward(prism_ctx, x, w, b, x, dx, g)
        made.append((graph, torch.cuda.Stream(), (y, dx, g), want, x))
    torch.cuda.synchronize()
    for _ in range(3):
        for graph, s, *_ in made:
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for _, _, (y, dx, g), want, _ in made:
        assert torch.equal(y, want[0]) and torch.equal(dx, want[1]) and all(torch.equal(g[k], want[2][k]) for k in g)
    prism_ctx.status()


def test_nonfinite_rows_stay_in_their_row(prism_ctx):
    """An infinity or a NaN in one row reaches that row's output only, also across a chunk's border."""
    for R, D, H in ((300, 64, 128), (19000, 16, 9600)):
        x = rand((R, D), F16, 1)
        w, b = weights(D, H, F16)
        y, y2 = torch.empty_like(x), torch.empty_like(x)
        forward(prism_ctx, x, w, b, y)
        bad = x.clone()
        rows = [0, 130, R - 1, min(R - 2, 18944)]
        bad[rows[0], 3], bad[rows[1], 5], bad[rows[2]], bad[rows[3], 0] = float("inf"), float("nan"), float("-inf"), float("nan")
        forward(prism_ctx, bad, w, b, y2)
        ok = torch.ones(R, dtype=torch.bool, device="cuda")
        ok[rows] = False
        assert torch.equal(y[ok], y2[ok]) and not torch.isfinite(y2[rows]).all(1).any()
        dx, dx2 = torch.empty_like(x), torch.empty_like(x)
        backward(prism_ctx, x, w, b, x, dx, {})
        backward(prism_ctx, bad, w, b, x, dx2, {})
        assert torch.equal(dx[ok], dx2[ok])


def test_no_rows(prism_ctx):
    w, b = weights(64, 128, F16)
    x = torch.empty((0, 64), dtype=F16, device="cuda")
    grads = grads_like(w, 128, 64)
    forward(prism_ctx, x, w, b, x)
    backward(prism_ctx, x, w, b, x, x, grads)
    assert not any(g.any() for g in grads.values())


def test_gradient_against_differences(prism_ctx):
    """Against central differences of the plain 64-bit forward with step 2^-8: their cut-off error is below
    h^2 / 6 times a third derivative of order 1, 2^-18; the bf16 gradients' own tolerance is far above."""
    R, D, H, h = 3, 16, 24, 2.0 ** -8
    x, dy = rand((R, D), BF16, 1), rand((R, D), BF16, 2)
    w, b = weights(D, H, BF16)
    dx, grads = empty((R, D), BF16), grads_like(w, H, D)
    backward(prism_ctx, x, w, b, dy, dx, grads, activation="gelu")
    want = ref.gated_back(x, w, b, dy, "gelu", BF16)
    base = [t.double() for t in (x, *w, *b)]
    loss = lambda p: float((ref.gated(p[0], p[1:4], p[4:], None, "gelu", BF16)[0] * dy.double()).sum())  # noqa: E731
    names = ("dx", "dw_gate", "dw_up", "dw_down", "db_gate", "db_up", "db_down")
    for k, n in enumerate(names):
        got = dx if n == "dx" else grads[n]
        for i in range(0, got.numel(), 7):
            v = []
            for s in (1, -1):
                p = list(base)
                p[k] = p[k].clone()
                p[k].view(-1)[i] += s * h
                v.append(loss(p))
            d, tol = (v[0] - v[1]) / (2 * h), float(want[n][1].reshape(-1)[i])
            assert abs(float(got.view(-1)[i]) - d) <= tol + ref.u(BF16) * (abs(d) + tol) + 2.0 ** -14, (n, i)


def test_bits_streams_and_graph(prism_ctx):
    """The same bits on every run, on another stream, and from a replayed graph with new inputs."""
    R, D, H = 700, 256, 512
    w, b = weights(D, H, BF16)

    def step(x, dy, stream=None):
        y, dx, grads = torch.empty_like(x), torch.empty_like(x), grads_like(w, H, D)
        forward(prism_ctx, x, w, b, y, residual=x, stream=stream)
        backward(prism_ctx, x, w, b, dy, dx, grads, stream=stream)
        return [y, dx, *grads.values()]
    x, dy = rand((R, D), BF16, 1), rand((R, D), BF16, 2)
    first = step(x, dy)
    assert all(torch.equal(p, q) for p, q in zip(first, step(x, dy)))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    for stream in (s, s.cuda_stream):
        with torch.cuda.stream(s):
            got = step(x, dy, stream)
        s.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(first, got))
    xs, dys = x.clone(), dy.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(xs, dys)
    for seed in (3, 5):
        xs.copy_(rand((R, D), BF16, seed))
        dys.copy_(rand((R, D), BF16, seed + 1))
        graph.replay()
        assert all(torch.equal(p, q) for p, q in zip(out, step(xs, dys)))
    prism_ctx.status()


def test_two_streams_at_once(prism_ctx):
    """Calls in flight on two streams share nothing."""
    D, H = 256, 1024
    w, b = weights(D, H, F16)
    xs = [rand((4000, D), F16, i) for i in (1, 2)]
    want = [(forward(prism_ctx, x, w, b, torch.empty_like(x)), grads_like(w, H, D), torch.empty_like(x)) for x in xs]
    for x, (y, g, dx) in zip(xs, want):
        backward(prism_ctx, x, w, b, x, dx, g)
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        got = []
        for s, x in zip(streams, xs):
            with torch.cuda.stream(s):
                y, g, dx = torch.empty_like(x), grads_like(w, H, D), torch.empty_like(x)
                forward(prism_ctx, x, w, b, y)
                backward(prism_ctx, x, w, b, x, dx, g)
                got.append((y, g, dx))
    torch.cuda.synchronize()
    for (y, g, dx), (y1, g1, dx1) in zip(want, got):
        assert torch.equal(y, y1) and torch.equal(dx, dx1) and all(torch.equal(g[k], g1[k]) for k in g)
    prism_ctx.status()


def test_refusals(prism_ctx):
    D, H = 64, 128
    x = rand((4, D), F16, 1)
    y = torch.empty_like(x)
    w, b = weights(D, H, F16)
    with pytest.raises(PrismError, match="multiples of 8"):
        forward(prism_ctx, torch.empty((4, 60), dtype=F16, device="cuda"), [torch.empty(s, dtype=F16, device="cuda") for s in
                ((H, 60), (H, 60), (60, H))], (None,) * 3, torch.empty((4, 60), dtype=F16, device="cuda"))
    with pytest.raises(PrismError, match="UNSUPPORTED"):
        forward(prism_ctx, x.float(), [t.float() for t in w], (None,) * 3, y.float())
    wide = torch.zeros((4, 2 * D + 8), dtype=F16, device="cuda")
    with pytest.raises(PrismError, match="overlaps"):
        forward(prism_ctx, x, w, b, x)
    with pytest.raises(PrismError, match="overlaps"):
        forward(prism_ctx, wide[:, :D], w, b, wide[:, 32:32 + D])
    with pytest.raises(PrismError, match="ALIGN"):
        forward(prism_ctx, wide[:, 1:1 + D], w, b, y)
    small = torch.empty(16, dtype=torch.uint8, device="cuda")
    with pytest.raises(PrismError, match="workspace"):
        backward(prism_ctx, x, w, b, y, torch.empty_like(x), {}, workspace=small)
    with pytest.raises(PrismError, match="workspace"):  # the forward pass needs one above dim 256
        x2, (w2, b2) = rand((4, 264), F16, 1), weights(264, H, F16)
        forward(prism_ctx, x2, w2, b2, torch.empty_like(x2), workspace=small)
    with pytest.raises(PrismError, match="overlaps"):
        backward(prism_ctx, x, w, b, y, y, {})
    for bad in (lambda: forward(prism_ctx, x, w, b, y, activation="tanh"), lambda: forward(prism_ctx, x, w, b, y.bfloat16()),
                lambda: forward(prism_ctx, x, (w[0], w[1], w[2].t()), b, y), lambda: forward(prism_ctx, x.cpu(), w, b, y),
                lambda: forward(prism_ctx, x, (w[0], w[1][:-8], w[2]), b, y),
                lambda: backward(prism_ctx, x, w, b, y, torch.empty_like(x), {"dw_gate": torch.empty_like(w[2])})):
        with pytest.raises(ValueError):
            bad()


def test_training_step_of_the_sub_block(prism_ctx):
    """y = x + dropout(ffn(norm(x))) and its gradients as a training step runs them, each call fed with the
    one before, against the chain in 64 bits on the same intermediate values."""
    R, D, H, p = 1000, 256, 512, 0.2
    dt = BF16
    x, dy = rand((R, D), dt, 1), rand((R, D), dt, 2)
    gamma, beta = (1 + 0.1 * torch.randn(D)).cuda(), (0.1 * torch.randn(D)).cuda()
    w, b = weights(D, H, dt)
    rng = torch.tensor([1234, 5], dtype=torch.int64, device="cuda")
    n, h, y = (torch.empty_like(x) for _ in range(3))
    mean, rstd = torch.empty(R, device="cuda"), torch.empty(R, device="cuda")
    prism_ctx.layer_norm(x, gamma, beta, n, mean=mean, rstd=rstd)
    forward(prism_ctx, n, w, b, h)
    prism_ctx.dropout_add(h, x, y, p, rng)
    want, tol, keep = ref.dropout(h, x, int(round(65536 * p)), rng.tolist())
    ref.check(y, want, tol, "y")
    dh, dn, dx = (torch.empty_like(x) for _ in range(3))
    grads = grads_like(w, H, D)
    dgamma, dbeta = torch.empty_like(gamma), torch.empty_like(beta)
    prism_ctx.dropout_add(dy, None, dh, p, rng)
    backward(prism_ctx, n, w, b, dh, dn, grads)
    prism_ctx.layer_norm_backward(x, gamma, mean, rstd, dn, dx, dweight=dgamma, dbias=dbeta, add=dy)
    want, tol, _ = ref.dropout(dy, None, int(round(65536 * p)), rng.tolist())
    ref.check(dh, want, tol, "dh")
    g64 = ref.gated_back(n, w, b, dh, "gelu", dt)
    ref.check(dn, *g64["dx"], "dn")
    for k in GRADS:
        ref.check(grads[k], *g64[k], k)
    want, tol = ref.norm_back(x, gamma, mean, rstd, dn, dy)
    for got, v, t, k in zip((dx, dgamma, dbeta), want, tol, ("dx", "dgamma", "dbeta")):
        ref.check(got, v, t, k)
    # the whole chain by automatic differentiation in 64 bits: near it, as far as bf16 intermediates allow
    x64 = x.double().requires_grad_()
    c = x64 - x64.mean(1, keepdim=True)
    n64 = c * torch.rsqrt((c * c).mean(1, keepdim=True) + 1e-5) * gamma.double() + beta.double()
    a, v = n64 @ w[0].double().T + b[0].double(), n64 @ w[1].double().T + b[1].double()
    o = (torch.nn.functional.gelu(a, approximate="tanh") * v) @ w[2].double().T + b[2].double()
    y64 = x64 + o * keep.cuda() / (1 - round(65536 * p) / 65536)
    (gx,) = torch.autograd.grad((y64 * dy.double()).sum(), x64)
    for got, v in ((y, y64.detach()), (dx, gx)):
        # some ten bf16 roundings of relative size 2^-8 lie on the way; their root sum is near 2^-7
        assert float((got.double() - v).norm() / v.norm()) < 2.0 ** -6
