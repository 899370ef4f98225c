"""Do the inputs and tolerances of the long-sum tests show what they are there to show?  The mistakes are made
in the plain forms, on the CPU."""
import pytest
import torch

import train_ref as ref

F16, BF16 = torch.float16, torch.bfloat16
GRADS = ("dw_gate", "dw_up", "dw_down", "db_gate", "db_up", "db_down")


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("lost", [slice(18944, 19500), slice(512, 768)], ids=["last chunk", "one tile"])
def test_lost_rows_show_in_every_gradient(dtype, lost):
    """Rows left out of the sums (a chunk that is not added on, a tile that no unit takes) change every gradient
    of the whole-number inputs in most places, behind its rounding to 16 bits."""
    x, w, b, dy = ref.whole_numbers(19500, 24, 64, 1)
    want = ref.relu_gated_back(x, w, b, dy)
    keep = torch.ones(19500, dtype=torch.bool)
    keep[lost] = False
    less = ref.relu_gated_back(x[keep], w, b, dy[keep])
    for n in GRADS:
        assert float((want[n].to(dtype) != less[n].to(dtype)).float().mean()) > 0.5, n


def test_whole_numbers_are_exact_in_16_bits():
    x, w, b, dy = ref.whole_numbers(300, 40, 72, 2)
    g, u, dh = x @ w[0].T + b[0], x @ w[1].T + b[1], dy @ w[2]
    for t in (x, dy, g.clamp(min=0) * u, dh * u * (g > 0), dh * g.clamp(min=0), *w, *b):
        assert torch.equal(t, t.bfloat16().double()) and torch.equal(t, t.half().double()) and t.any()


@pytest.mark.parametrize("kind", ["gelu", "silu", "relu"])
def test_sums_of_rounded_rows_show(kind):
    """The bias gradients' tolerance has no room for rows rounded to bf16 before their sum, and has some for sums in fp32."""
    g = torch.Generator().manual_seed(3)
    R, D, H = 300, 64, 512
    x, dy = (torch.randn(R, D, generator=g).bfloat16().double() for _ in range(2))
    w = [(torch.randn(s, generator=g) * s[1] ** -0.5).bfloat16().double() for s in ((H, D), (H, D), (D, H))]
    b = [(torch.randn(H, generator=g) * 0.1).bfloat16().double() for _ in range(2)]
    want = ref.bias_grads(x, w, b, dy, kind)
    a, d = ref.act(x @ w[0].T + b[0], kind)
    u, dh = x @ w[1].T + b[1], dy @ w[2]
    for n, rows in (("db_gate", dh * u * d), ("db_up", dh * a)):
        ref.check(rows.float().sum(0).bfloat16(), *want[n], n)
        with pytest.raises(AssertionError):
            ref.check(rows.bfloat16().double().sum(0).bfloat16(), *want[n], n)


def test_vectorised_generator():
    for rng in ((0, 0), (0xDEADBEEF12345678, 0xF00000000000000A), (-5, -1)):
        for t in (1, 20000, 65535):
            assert torch.equal(ref.kept(rng, 0, 1001, t), ref.draws(rng, 1001) >= t)
            assert torch.equal(ref.kept(rng, 800, 201, t), (ref.draws(rng, 1001) >= t)[800:])
    # a counter above 32 bits: the high word
    c = 2 ** 33 + 3
    words = ref.philox_block([c & ref.M32, c >> 32, 7, 0], [9, 0])
    bits = torch.tensor([v for w in words for v in (w & 0xFFFF, w >> 16)])
    assert torch.equal(ref.kept((9, 7), 8 * c, 8, 30000), bits >= 30000)
