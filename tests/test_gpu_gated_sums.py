"""The gated feed-forward block where rows go through in several chunks and a CTA pair takes several units: whole-number
inputs, whose outputs are exact sums rounded once, so nothing hides behind a tolerance."""
import pytest
import torch

import train_ref as ref

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16
NAMES = ("dw_gate", "dw_up", "dw_down", "db_gate", "db_up", "db_down")

# 148 SMs: chunks of 18,944 rows where a row's 3 x hidden 16-bit values leave less than two such chunks in 1 GiB
BACKWARD = [
    (19500, 72, 4736),    # dim <= 256, two chunks
    (38500, 16, 4800),    # three
    (19300, 256, 4736),   # two, full width
    (20000, 128, 72),     # more row tiles than CTA pairs, the last one cut
    (40000, 200, 136),    # three row tiles a pair
    (19300, 264, 4736),   # dim > 256, two chunks
    (38200, 328, 4736),   # three
    (2051, 520, 2744),    # 9 x 22 units of 74 pairs: a third one for some
    (5000, 264, 1032),    # 20 x 9
    (9000, 264, 2056),    # 36 x 17: nine a pair
]
FORWARD = [(40000, 256, 264), (25000, 72, 1032), (2051, 520, 2744), (9000, 264, 2056), (19400, 264, 14344)]


def rows(t, dtype, pad):
    wide = torch.full((t.shape[0], t.shape[1] + pad), 7.0, dtype=dtype, device="cuda")
    wide[:, :t.shape[1]] = t
    return wide, wide[:, :t.shape[1]]


def same(got, want, what):
    """Equal to the exact value rounded to got's type (fp32 holds every one of these whole numbers)."""
    want = want.float().to(got.dtype)
    if not torch.equal(got, want):
        bad = (got != want).nonzero()
        raise AssertionError(f"{what}: {len(bad)} of {got.numel()} differ, first at {bad[0].tolist()}, last at {bad[-1].tolist()}")


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("shape", BACKWARD)
@pytest.mark.parametrize("pad", [0, 24])
def test_backward_is_exact(prism_ctx, dtype, shape, pad):
    R, D, H = shape
    x, w, b, dy = ref.whole_numbers(R, D, H, R + H, "cuda")
    want = ref.relu_gated_back(x, w, b, dy)
    (_, xs), (_, dys), (wide, dx) = rows(x, dtype, pad), rows(dy, dtype, pad), rows(torch.zeros_like(x), dtype, pad)
    wl, bl = [t.to(dtype) for t in w], [t.to(dtype) for t in b]
    grads = {n: torch.full(want[n].shape, 7.0, dtype=dtype, device="cuda") for n in NAMES}
    prism_ctx.gated_ffn_backward(xs, *wl, dys, dx, b_gate=bl[0], b_up=bl[1], activation="relu", **grads)
    prism_ctx.status()
    same(dx, want["dx"], "dx")
    for n in NAMES:
        same(grads[n], want[n], n)
    assert (wide[:, D:] == 7.0).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("shape", FORWARD)
@pytest.mark.parametrize("pad", [0, 24])
def test_forward_is_exact(prism_ctx, dtype, shape, pad):
    R, D, H = shape
    x, w, b, r = ref.whole_numbers(R, D, H, R + H, "cuda")
    (_, xs), (_, rs), (wide, y) = rows(x, dtype, pad), rows(r, dtype, pad), rows(torch.zeros_like(x), dtype, pad)
    wl, bl = [t.to(dtype) for t in w], [t.to(dtype) for t in b]
    prism_ctx.gated_ffn(xs, *wl, y, b_gate=bl[0], b_up=bl[1], b_down=bl[2], residual=rs, activation="relu")
    prism_ctx.status()
    same(y, ref.relu_gated(x, w, b, r), "y")
    assert (wide[:, D:] == 7.0).all()


@pytest.mark.parametrize("shape", [(300, 64, 512), (257, 256, 256), (300, 264, 512), (130, 520, 136)])
@pytest.mark.parametrize("kind", ["gelu", "silu", "relu"])
def test_bias_gradients_are_sums_of_unrounded_rows(prism_ctx, shape, kind):
    R, D, H = shape
    g = torch.Generator().manual_seed(R + D)
    x, dy = (torch.randn(R, D, generator=g).to(BF16).cuda() for _ in range(2))
    w = [(torch.randn(s, generator=g) * s[1] ** -0.5).to(BF16).cuda() for s in ((H, D), (H, D), (D, H))]
    b = [(torch.randn(H, generator=g) * 0.1).to(BF16).cuda() for _ in range(2)]
    want = ref.bias_grads(x, w, b, dy, kind)
    grads = {n: torch.empty(D if n == "db_down" else H, dtype=BF16, device="cuda") for n in want}
    prism_ctx.gated_ffn_backward(x, *w, dy, torch.empty_like(x), b_gate=b[0], b_up=b[1], activation=kind, **grads)
    for n in want:
        ref.check(grads[n], *want[n], n)


@pytest.mark.parametrize("dim", [256, 264])
def test_element_offsets_past_32_bits(prism_ctx, dim):
    """More than 2^31 elements: the last rows, and those around the border, of y and dx.  ReLU on whole numbers."""
    R, H = 2 ** 31 // dim + 3000, 64
    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randint(-1, 2, (R, dim), generator=g, device="cuda", dtype=torch.int8).to(BF16)
    _, w, b, _ = ref.whole_numbers(8, dim, H, 5, "cuda")
    wl, bl = [t.to(BF16) for t in w], [t.to(BF16) for t in b]
    y = torch.full_like(x, 7.0)
    prism_ctx.gated_ffn(x, *wl, y, b_gate=bl[0], b_up=bl[1], b_down=bl[2], residual=x, activation="relu")
    prism_ctx.status()
    parts = (slice(0, 300), slice(2 ** 30 // dim - 200, 2 ** 30 // dim + 200), slice(2 ** 31 // dim - 200, R))
    for p in parts:
        v = x[p].double()
        same(y[p], ref.relu_gated(v, w, b, v), f"y {p}")
    y.fill_(7.0)
    prism_ctx.gated_ffn_backward(x, *wl, x, y, b_gate=bl[0], b_up=bl[1], activation="relu")
    prism_ctx.status()
    for p in parts:
        v = x[p].double()
        same(y[p], ref.relu_gated_back(v, w, b, v)["dx"], f"dx {p}")
