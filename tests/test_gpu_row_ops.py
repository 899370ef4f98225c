"""Layer norm and dropout with the residual add (both directions) on the GPU, through the public calls,
against plain 64-bit forms."""
import ctypes as C

import pytest
import torch

import train_ref as ref
from prism_inference_b200.abi import NormParams, PrismError

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def rand(shape, dtype, seed, pad=0, std=1.0, off=0.0):
    """Values in the first columns of a buffer with `pad` more; the pad holds a sentinel."""
    g = torch.Generator().manual_seed(seed)
    t = torch.full((shape[0], shape[1] + pad), 7.0, dtype=dtype)
    t[:, :shape[1]] = (torch.randn(shape, generator=g) * std + off).to(dtype)
    return t.cuda()[:, :shape[1]]


def empty(shape, dtype, pad=0):
    return torch.full((shape[0], shape[1] + pad), 7.0, dtype=dtype, device="cuda")[:, :shape[1]]


def pad_untouched(t):
    base = t._base if t._base is not None else t
    return bool((base.as_strided((base.shape[0], base.shape[1]), base.stride())[:, t.shape[1]:] == 7.0).all())


NORM_SHAPES = [(1, 1), (3, 2), (64, 256), (5, 7), (33, 64), (300, 100), (17, 128), (9, 130), (2, 513), (40, 1000), (7, 1024),
               (5, 1025), (3, 2052), (4, 4097), (2, 8200), (2, 16384), (2500, 96), (70000, 8)]


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("shape", NORM_SHAPES)
@pytest.mark.parametrize("pad", [0, 8, 3])
def test_norm_forward_and_backward(prism_ctx, dtype, shape, pad):
    R, D = shape
    pt = F32 if (R + pad) % 2 else dtype
    x, dy, add = (rand(shape, dtype, 10 * D + i, pad, off=0.5 * (i == 0)) for i in range(3))
    w, b = rand((1, D), pt, 4, off=1.0)[0].contiguous(), rand((1, D), pt, 5)[0].contiguous()
    y, dx = empty(shape, dtype, pad), empty(shape, dtype, pad)
    mean, rstd = torch.empty(R, device="cuda"), torch.empty(R, device="cuda")
    prism_ctx.layer_norm(x, w, b, y, eps=1e-5, mean=mean, rstd=rstd)
    want, tol = ref.norm(x, w, b, 1e-5)
    for g, v, t, n in zip((y, mean, rstd), want, tol, ("y", "mean", "rstd")):
        ref.check(g, v, t, n)
    assert pad_untouched(y)
    dw, db = torch.empty_like(w), torch.empty_like(b)
    a = add if pad != 8 else None
    prism_ctx.layer_norm_backward(x, w, mean, rstd, dy, dx, dweight=dw, dbias=db, add=a)
    want, tol = ref.norm_back(x, w, mean, rstd, dy, a)
    for g, v, t, n in zip((dx, dw, db), want, tol, ("dx", "dweight", "dbias")):
        ref.check(g, v, t, n)
    assert pad_untouched(dx)


def test_norm_optional_tensors(prism_ctx):
    x, dy = rand((37, 200), F16, 1), rand((37, 200), F16, 2)
    y = empty((37, 200), F16)
    prism_ctx.layer_norm(x, None, None, y, eps=1e-3)
    (want, mean, rstd), (tol, _, _) = ref.norm(x, None, None, 1e-3)
    ref.check(y, want, tol, "y")
    mean, rstd = mean.float(), rstd.float()
    want, tol = ref.norm_back(x, None, mean, rstd, dy, None)
    dx = empty((37, 200), F16)
    prism_ctx.layer_norm_backward(x, None, mean, rstd, dy, dx)  # no sums, no workspace
    ref.check(dx, want[0], tol[0], "dx")
    for i, kw in ((1, "dweight"), (2, "dbias")):
        out = torch.empty(200, device="cuda")
        prism_ctx.layer_norm_backward(x, None, mean, rstd, dy, dx, **{kw: out})
        ref.check(out, want[i], tol[i], kw)


def test_norm_three_dimensions_and_in_place(prism_ctx):
    x = rand((60, 256), BF16, 3).reshape(3, 20, 256)
    w, b = rand((1, 256), F32, 4)[0].contiguous(), rand((1, 256), F32, 5)[0].contiguous()
    y, mean, rstd = torch.empty_like(x), torch.empty(60, device="cuda"), torch.empty(60, device="cuda")
    prism_ctx.layer_norm(x, w, b, y, mean=mean, rstd=rstd)
    z = x.clone()
    prism_ctx.layer_norm(z, w, b, z)
    assert torch.equal(y, z)
    dy = torch.randn_like(x)
    out = [torch.empty_like(x), dy.clone()]
    prism_ctx.layer_norm_backward(x, w, mean, rstd, dy, out[0])
    prism_ctx.layer_norm_backward(x, w, mean, rstd, out[1], out[1])
    assert torch.equal(out[0], out[1])


@pytest.mark.parametrize("dtype", [F16, F32])
def test_odd_rows_in_place_and_as_column_slices(prism_ctx, dtype):
    """Rows off 16-byte boundaries: in place, and as neighbouring column slices of one buffer, whose 16-byte
    chunks the rows share."""
    R, D = 3001, 101
    x, dy = rand((R, D), dtype, 1), rand((R, D), dtype, 2)
    w, b = rand((1, D), F32, 3)[0].contiguous(), rand((1, D), F32, 4)[0].contiguous()
    mean, rstd = torch.empty(R, device="cuda"), torch.empty(R, device="cuda")
    y, dx, z = torch.empty_like(x), torch.empty_like(x), torch.empty_like(x)
    prism_ctx.layer_norm(x, w, b, y, mean=mean, rstd=rstd)
    prism_ctx.layer_norm_backward(x, w, mean, rstd, dy, dx, add=y)
    prism_ctx.dropout_add(x, dy, z, 0.4, rng_of(*RNG))
    wide = torch.full((R, 3 * D + 2), 7.0, dtype=dtype, device="cuda")
    for src, call, want in ((x, lambda s, o: prism_ctx.layer_norm(s, w, b, o), y),
                            (dy, lambda s, o: prism_ctx.layer_norm_backward(x, w, mean, rstd, s, o, add=y), dx),
                            (x, lambda s, o: prism_ctx.dropout_add(s, dy, o, 0.4, rng_of(*RNG)), z)):
        t = src.clone()
        call(t, t)
        assert torch.equal(t, want)
        wide.fill_(7.0)
        wide[:, :D] = src
        call(wide[:, :D], wide[:, D:2 * D])
        assert torch.equal(wide[:, D:2 * D], want) and torch.equal(wide[:, :D], src) and (wide[:, 2 * D:] == 7.0).all()


def test_norm_constant_and_nonfinite_rows(prism_ctx):
    """A constant row has variance 0; an infinity or a NaN stays in its own row."""
    x = rand((6, 96), F32, 6)
    x[1], x[3, 5], x[4, 95] = 2.5, float("inf"), float("nan")
    w, b = torch.ones(96, device="cuda"), torch.full((96,), 0.25, device="cuda")
    y, mean, rstd = torch.empty_like(x), torch.empty(6, device="cuda"), torch.empty(6, device="cuda")
    prism_ctx.layer_norm(x, w, b, y, mean=mean, rstd=rstd)
    assert torch.allclose(y[1], b, atol=1e-3) and torch.isnan(y[3:5]).all()
    ok = [0, 1, 2, 5]
    want, tol = ref.norm(x[ok], w, b, 1e-5)
    ref.check(y[ok], want[0], tol[0], "finite rows")


def test_norm_no_rows(prism_ctx):
    x = torch.empty((0, 64), dtype=F16, device="cuda")
    e = torch.empty(0, device="cuda")
    dw, db = torch.full((64,), 3.0, device="cuda"), torch.full((64,), 3.0, device="cuda")
    prism_ctx.layer_norm(x, None, None, x)
    prism_ctx.layer_norm_backward(x, None, e, e, x, x, dweight=dw, dbias=db)
    assert not dw.any() and not db.any()


def test_norm_gradient_against_differences(prism_ctx):
    """dx, dweight, dbias against central differences of the plain 64-bit forward (step 2^-12: the cut-off
    error is below 2^-20 of the third derivative, far under the tolerance)."""
    R, D, h = 3, 24, 2.0 ** -12
    x, dy = rand((R, D), F32, 7), rand((R, D), F32, 8)
    w, b = rand((1, D), F32, 9)[0].contiguous(), rand((1, D), F32, 10)[0].contiguous()
    mean, rstd, y, dx = torch.empty(R, device="cuda"), torch.empty(R, device="cuda"), torch.empty_like(x), torch.empty_like(x)
    dw, db = torch.empty(D, device="cuda"), torch.empty(D, device="cuda")
    prism_ctx.layer_norm(x, w, b, y, mean=mean, rstd=rstd)
    prism_ctx.layer_norm_backward(x, w, mean, rstd, dy, dx, dweight=dw, dbias=db)
    loss = lambda x, w, b: float((ref.norm(x, w, b, 1e-5)[0][0] * dy.double()).sum())  # noqa: E731
    for got, k in ((dx, 0), (dw, 1), (db, 2)):
        for i in range(0, got.numel(), 5):
            args = [[x.double(), w.double(), b.double()] for _ in range(2)]
            for s, a in zip((1, -1), args):
                a[k] = a[k].clone()
                a[k].view(-1)[i] += s * h
            d = (loss(*args[0]) - loss(*args[1])) / (2 * h)
            assert abs(float(got.view(-1)[i]) - d) < 1e-4 * max(1.0, abs(d))


def test_norm_bits_streams_and_graph(prism_ctx):
    """The same bits on every run, on another stream, and from a replayed graph with new inputs."""
    R, D = 5000, 256
    x, dy = rand((R, D), BF16, 11), rand((R, D), BF16, 12)
    w, b = torch.randn(D, device="cuda"), torch.randn(D, device="cuda")

    def step(x, dy, stream=None):
        o = [torch.empty_like(x), torch.empty(R, device="cuda"), torch.empty(R, device="cuda"), torch.empty_like(x),
             torch.empty(D, device="cuda"), torch.empty(D, device="cuda")]
        prism_ctx.layer_norm(x, w, b, o[0], mean=o[1], rstd=o[2], stream=stream)
        prism_ctx.layer_norm_backward(x, w, o[1], o[2], dy, o[3], dweight=o[4], dbias=o[5], stream=stream)
        return o
    first = step(x, dy)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    for stream in (s, s.cuda_stream):
        with torch.cuda.stream(s):  # the outputs belong to s
            got = step(x, dy, stream)
        s.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(first, got))
    xs, dys = x.clone(), dy.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(xs, dys)
    for seed in (13, 14):
        xs.copy_(rand((R, D), BF16, seed))
        dys.copy_(rand((R, D), BF16, seed + 2))
        graph.replay()
        assert all(torch.equal(a, c) for a, c in zip(out, step(xs, dys)))


def test_norm_refusals(prism_ctx):
    x = rand((4, 64), F16, 1)
    y = torch.empty_like(x)
    w = torch.ones(64, device="cuda")
    m = torch.empty(4, device="cuda")
    wide = torch.empty((4, 128), dtype=F16, device="cuda")
    with pytest.raises(PrismError, match="UNSUPPORTED"):
        big = torch.empty((1, 16385), dtype=F16, device="cuda")
        prism_ctx.layer_norm(big, None, None, torch.empty_like(big))
    with pytest.raises(PrismError, match="overlaps"):
        prism_ctx.layer_norm(wide[:, :64], None, None, wide[:, 32:96])
    prism_ctx.layer_norm(wide.zero_()[:, :64], None, None, wide[:, 64:])  # column slices do not overlap
    with pytest.raises(PrismError, match="workspace"):
        prism_ctx.layer_norm_backward(x, w, m, m, x, y, dweight=torch.empty_like(w),
                                      workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))
    with pytest.raises(PrismError, match="NULL"):
        prism_ctx.layer_norm_backward(x, w, None, m, x, y)
    for bad in (lambda: prism_ctx.layer_norm(x.cpu(), None, None, y), lambda: prism_ctx.layer_norm(x, None, None, y.float()),
                lambda: prism_ctx.layer_norm(x, w[:63], None, y), lambda: prism_ctx.layer_norm(x, w.half(), w, y),
                lambda: prism_ctx.layer_norm(x.t(), None, None, y), lambda: prism_ctx.layer_norm(x, None, None, y, mean=m[:3]),
                lambda: prism_ctx.layer_norm(x.double(), None, None, y.double()),
                lambda: prism_ctx.layer_norm(x, None, None, y[:3])):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(PrismError, match="ARG"):
        prism_ctx.layer_norm(x, w.bfloat16(), None, y)  # parameters: the rows' type or fp32
    p = NormParams(rows=4, x_stride=63, y_stride=64, dim=64, dtype=0, param_dtype=0, eps=1e-5)
    assert prism_ctx.lib.prism_layer_norm(prism_ctx.h, C.byref(p), x.data_ptr(), None, None, y.data_ptr(), None, None, None) == 1
    p.x_stride = 64
    assert prism_ctx.lib.prism_layer_norm(prism_ctx.h, C.byref(p), x.data_ptr() + 1, None, None, y.data_ptr(), None, None, None) == 2


# ---- dropout ----------------------------------------------------------------------------------


def rng_of(seed, offset):
    to64 = lambda v: v - (1 << 64) if v >= 1 << 63 else v  # noqa: E731
    return torch.tensor([to64(seed), to64(offset)], dtype=torch.int64, device="cuda")


RNG = (0xDEADBEEF12345678, 0xF00000000000000A)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("shape", [(1, 1), (1, 7), (1, 8), (3, 5), (64, 128), (33, 24), (7, 1001), (130, 256)])
@pytest.mark.parametrize("pad", [0, 8, 5])
@pytest.mark.parametrize("with_residual", [False, True])
def test_dropout(prism_ctx, dtype, shape, pad, with_residual):
    x = rand(shape, dtype, 20, pad)
    res = rand(shape, dtype, 21, pad) if with_residual else None
    y = empty(shape, dtype, pad)
    rng = rng_of(*RNG)
    prism_ctx.dropout_add(x, res, y, 0.3, rng)
    want, tol, keep = ref.dropout(x, res, int(round(65536 * 0.3)), rng.tolist())
    ref.check(y, want, tol, "y")
    assert pad_untouched(y)
    if not with_residual:
        assert not y.cpu()[~keep].any()


def test_dropout_mask_is_a_function_of_the_index(prism_ctx):
    """The same mask for every type, stride and launch, another for another seed or offset; rate as asked."""
    shape, p = (997, 264), 0.25
    masks = []
    for dtype, pad in ((F16, 0), (F32, 0), (BF16, 8), (F32, 3)):
        x, y = torch.ones(shape, dtype=dtype, device="cuda"), empty(shape, dtype, pad)
        prism_ctx.dropout_add(x, None, y, p, rng_of(*RNG))
        masks.append(y != 0)
    assert all(torch.equal(masks[0], m) for m in masks)
    for other in ((RNG[0] + 1, RNG[1]), (RNG[0], RNG[1] + 1), (RNG[0] ^ 1 << 40, RNG[1]), (RNG[0], RNG[1] ^ 1 << 40)):
        y = torch.empty(shape, device="cuda")
        prism_ctx.dropout_add(torch.ones(shape, device="cuda"), None, y, p, rng_of(*other))
        same = float(((y != 0) == masks[0]).float().mean())
        assert abs(same - (p * p + (1 - p) ** 2)) < 5 * (0.25 / y.numel()) ** 0.5  # independent masks agree this often
    rate = float(masks[0].float().mean())
    assert abs(rate - (1 - p)) < 5 * (p * (1 - p) / masks[0].numel()) ** 0.5


def test_dropout_edges(prism_ctx):
    x, res = rand((9, 40), F16, 22), rand((9, 40), F16, 23)
    y = torch.empty_like(x)
    prism_ctx.dropout_add(x, None, y, 0.0, rng_of(1, 2))
    assert torch.equal(y, x)
    # what a dropped element holds does not matter: infinities and NaN leave the residual
    bad = x.clone()
    t = int(round(65536 * 0.5))
    keep = ref.dropout(x, None, t, (1, 2))[2].cuda()
    bad[~keep] = float("nan")
    prism_ctx.dropout_add(bad, res, y, 0.5, rng_of(1, 2))
    assert torch.equal(y[~keep], res[~keep]) and torch.isfinite(y).all()
    # in place, on the residual and on the input
    z = res.clone()
    prism_ctx.dropout_add(bad, z, z, 0.5, rng_of(1, 2))
    assert torch.equal(z, y)
    z = bad.clone()
    prism_ctx.dropout_add(z, res, z, 0.5, rng_of(1, 2))
    assert torch.equal(z, y)
    none = torch.empty((0, 40), dtype=F16, device="cuda")
    prism_ctx.dropout_add(none, None, none, 0.5, rng_of(1, 2))


def test_dropout_graph_reads_the_generator_when_it_runs(prism_ctx):
    x, y, rng = torch.ones((64, 256), device="cuda"), torch.empty((64, 256), device="cuda"), rng_of(5, 0)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        prism_ctx.dropout_add(x, None, y, 0.5, rng)
        rng[1] += 1
    seen = []
    for k in range(3):
        g.replay()
        seen.append(y.clone())
        z = torch.empty_like(y)
        prism_ctx.dropout_add(x, None, z, 0.5, rng_of(5, k))
        assert torch.equal(y, z)
    assert not torch.equal(seen[0], seen[1]) and not torch.equal(seen[1], seen[2])


def test_dropout_refusals(prism_ctx):
    x = rand((4, 64), F16, 1)
    y, rng = torch.empty_like(x), rng_of(1, 2)
    for p in (1.0, -0.1, 2.0):
        with pytest.raises(PrismError, match="threshold"):
            prism_ctx.dropout_add(x, None, y, p, rng)
    wide = torch.empty((4, 128), dtype=F16, device="cuda")
    with pytest.raises(PrismError, match="overlaps"):
        prism_ctx.dropout_add(wide[:, :64], None, wide[:, 1:65], 0.1, rng)
    for bad in (lambda: prism_ctx.dropout_add(x, y[:3], y, 0.1, rng), lambda: prism_ctx.dropout_add(x, None, y, 0.1, rng.int()),
                lambda: prism_ctx.dropout_add(x, None, y, 0.1, rng.cpu()), lambda: prism_ctx.dropout_add(x, None, y.t(), 0.1, rng)):
        with pytest.raises(ValueError):
            bad()
