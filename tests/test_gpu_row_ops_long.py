"""Layer norm and dropout where a team of threads walks several rows and a thread several blocks, against plain
64-bit forms; and tensors of more than 2^31 elements."""
import pytest
import torch

import train_ref as ref

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def rand(shape, dtype, seed, pad=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = torch.full((shape[0], shape[1] + pad), 7.0, dtype=dtype, device="cuda")
    t[:, :shape[1]] = torch.randn(shape, generator=g, device="cuda") + 0.25
    return t[:, :shape[1]]


def pad_untouched(t):
    return t._base is None or bool((t._base[:, t.shape[1]:] == 7.0).all())


# A team has 4 to 256 threads by dim (64, 128, .. 4096 and above) and a CTA 256, with up to 3 CTAs on each of 148
# SMs: every team of these walks two rows at least, most of them three.  Odd dims and pads take rows off 16-byte boundaries.
ROWS = {64: 60000, 128: 31000, 256: 16000, 512: 8000, 1024: 4000, 2048: 2000, 4096: 1100, 8192: 1050, 16384: 1010}
SHAPES = [(R, D - d, p) for D, R in ROWS.items() for d, p in ((0, 0), (27, 0), (27, 3))] + [(8000, 512, 5), (16000, 256, 8)]


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("shape", SHAPES)
def test_norm_teams_of_several_rows(prism_ctx, dtype, shape):
    R, D, pad = shape
    x, dy, add = (rand((R, D), dtype, D + i, pad) for i in range(3))
    w, b = rand((1, D), F32, 4)[0].contiguous(), rand((1, D), F32, 5)[0].contiguous()
    y, dx = rand((R, D), dtype, 6, pad), rand((R, D), dtype, 6, pad)
    mean, rstd = torch.empty(R, device="cuda"), torch.empty(R, device="cuda")
    prism_ctx.layer_norm(x, w, b, y, mean=mean, rstd=rstd)
    want, tol = ref.norm(x, w, b, 1e-5)
    for g, v, t, n in zip((y, mean, rstd), want, tol, ("y", "mean", "rstd")):
        ref.check(g, v, t, n)
    del want, tol
    dw, db = torch.empty_like(w), torch.empty_like(b)
    prism_ctx.layer_norm_backward(x, w, mean, rstd, dy, dx, dweight=dw, dbias=db, add=add)
    want, tol = ref.norm_back(x, w, mean, rstd, dy, add)
    for g, v, t, n in zip((dx, dw, db), want, tol, ("dx", "dweight", "dbias")):
        ref.check(g, v, t, n)
    assert pad_untouched(y) and pad_untouched(dx)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("shape", [(40000, 101), (3000, 1001), (40000, 128), (3000, 1000), (70000, 3)])
def test_long_rows_in_place_and_as_column_slices(prism_ctx, dtype, shape):
    """A team's next row is being loaded while it writes this one: in place, and beside the input in one buffer,
    whose 16-byte chunks the rows share."""
    R, D = shape
    x, dy = rand((R, D), dtype, 1), rand((R, D), dtype, 2)
    w, b = rand((1, D), F32, 3)[0].contiguous(), rand((1, D), F32, 4)[0].contiguous()
    rng = torch.tensor([11, -3], device="cuda")
    mean, rstd = torch.empty(R, device="cuda"), torch.empty(R, device="cuda")
    y, dx, z = torch.empty_like(x), torch.empty_like(x), torch.empty_like(x)
    prism_ctx.layer_norm(x, w, b, y, mean=mean, rstd=rstd)
    prism_ctx.layer_norm_backward(x, w, mean, rstd, dy, dx, add=y)
    prism_ctx.dropout_add(x, dy, z, 0.4, rng)
    wide = torch.empty((R, 3 * D + 2), dtype=dtype, device="cuda")
    for src, call, want in ((x, lambda s, o: prism_ctx.layer_norm(s, w, b, o), y),
                            (dy, lambda s, o: prism_ctx.layer_norm_backward(x, w, mean, rstd, s, o, add=y), dx),
                            (x, lambda s, o: prism_ctx.dropout_add(s, dy, o, 0.4, rng), z)):
        t = src.clone()
        call(t, t)
        assert torch.equal(t, want)
        wide.fill_(7.0)
        wide[:, :D] = src
        call(wide[:, :D], wide[:, D:2 * D])
        assert torch.equal(wide[:, D:2 * D], want) and torch.equal(wide[:, :D], src) and (wide[:, 2 * D:] == 7.0).all()


RNG = (0xDEADBEEF12345678, 0x0123456789ABCDEF)


def rng_of(seed, offset):
    return torch.tensor([v - (1 << 64) if v >= 1 << 63 else v for v in (seed, offset)], device="cuda")


def check_dropout(x, res, y, p, first, what):
    """y against the plain form, whose generator works on whole tensors; elements `first` and on of the call."""
    t = int(round(65536 * p))
    keep = ref.kept(RNG, first, x.numel(), t, "cuda").reshape(x.shape)
    v = torch.where(keep, x.double() * (65536 / (65536 - t)), 0.0)
    want = v if res is None else v + res.double()
    # the scale's rounding, the product's and the sum's: 4 roundings in fp32 of the terms
    ref.check(y, want, 4 * ref.U32 * (v.abs() + want.abs()), what)


# 5.3 M elements: with 8 elements a block and 148 x 8 CTAs of 256 threads, a thread's third block
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("shape,pad", [((4100, 1280), 0), ((4100, 1280), 8), ((5301, 1001), 0), ((5301, 1001), 5), ((663001, 8), 3),
                                       ((1, 5300003), 0)])
@pytest.mark.parametrize("with_residual", [False, True])
def test_dropout_of_many_blocks_a_thread(prism_ctx, dtype, shape, pad, with_residual):
    x = rand(shape, dtype, 20, pad)
    res = rand(shape, dtype, 21, pad) if with_residual else None
    y = rand(shape, dtype, 22, pad)
    prism_ctx.dropout_add(x, res, y, 0.3, rng_of(*RNG))
    check_dropout(x, res, y, 0.3, 0, "y")
    assert pad_untouched(y)


@pytest.mark.parametrize("D", [256, 101])
def test_element_offsets_past_32_bits(prism_ctx, D):
    R = -(-(2 ** 31 + 100000) // D)
    g = torch.Generator(device="cuda").manual_seed(7)
    x = torch.randn((R, D), generator=g, device="cuda", dtype=F16)
    y = torch.full_like(x, 7.0)
    parts = [slice(a // 8 * 8, n) for a, n in ((0, 400), (2 ** 30 // D - 200, 2 ** 30 // D + 200), (2 ** 31 // D - 200, R))]
    prism_ctx.dropout_add(x, x, y, 0.25, rng_of(*RNG))
    for p in parts:
        check_dropout(x[p], x[p], y[p], 0.25, p.start * D, f"dropout {p}")
    w, b = rand((1, D), F32, 3)[0].contiguous(), rand((1, D), F32, 4)[0].contiguous()
    mean, rstd = torch.empty(R, device="cuda"), torch.empty(R, device="cuda")
    y.fill_(7.0)
    prism_ctx.layer_norm(x, w, b, y, mean=mean, rstd=rstd)
    for p in parts:
        want, tol = ref.norm(x[p], w, b, 1e-5)
        for got, v, t, n in zip((y[p], mean[p], rstd[p]), want, tol, ("y", "mean", "rstd")):
            ref.check(got, v, t, f"{n} {p}")
    y.fill_(7.0)
    prism_ctx.layer_norm_backward(x, w, mean, rstd, x, y)
    for p in parts:
        want, tol = ref.norm_back(x[p], w, mean[p], rstd[p], x[p], None)
        ref.check(y[p], want[0], tol[0], f"dx {p}")


@pytest.mark.parametrize("shape", [(4099, 1001), (4099, 1000), (20000, 256)])
def test_parameter_gradients_lose_little_to_their_sums(prism_ctx, shape):
    """The root mean square of the sums' error over the columns.  An fp32 rounding is off by at most 2^-24 of its value,
    evenly spread, so by 2^-24 / sqrt(3) in the mean square; independent ones add up in squares, each weighted with its partial sum's
    share of the rows: c = rows a thread adds up (c^2 / 2 + c / 2 for each of the R / c threads of a column),
    then p threads of a CTA (a running sum each, c p (p + 1) / 2 for each of the R / (c p) CTAs).  Then a
    rounding to fp32, and three on each term (x - mean, the product with rstd, the fused product with dy).
    What joins the CTAs' partial sums has no share: it adds in 64 bits."""
    R, D = shape
    x, dy = rand(shape, F32, 31) - 0.25, rand(shape, F32, 32) - 0.25
    mean, rstd = torch.zeros(R, device="cuda"), torch.ones(R, device="cuda")
    dw, db = torch.empty(D, device="cuda"), torch.empty(D, device="cuda")
    prism_ctx.layer_norm_backward(x, None, mean, rstd, dy, torch.empty_like(x), dweight=dw, dbias=db)
    # a team has D / 16 threads, rounded up to a power of two; one CTA of 256 threads on each of 148 SMs.  Teams of
    # less than a warp: 32 / team of them come together by butterfly, in place of running sums
    p = 256 // (64 if D > 512 else 16)
    c = -(-R // (148 * p))
    squares = ((c + 1) / 2 + (p + 1) / 2 + 1 + 3)
    for got, want in ((dw, (dy.double() * x.double()).sum(0)), (db, dy.double().sum(0))):
        off = float((got.double() - want).norm() / want.norm())
        assert off < (squares / 3) ** 0.5 * ref.U32, (off, (squares / 3) ** 0.5 * ref.U32)
