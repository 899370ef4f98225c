"""The plain 64-bit forms that the GPU tests compare with, checked by themselves (CPU): the generator
against published answers, gradients against differences."""
import pytest
import torch

import train_ref as ref


def test_philox_known_answers():
    """The known-answer vectors published with the generator (Random123, philox4x32-10)."""
    assert ref.philox_block([0] * 4, [0] * 2) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert ref.philox_block([ref.M32] * 4, [ref.M32] * 2) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]


def test_norm_gradient_formula():
    g = torch.Generator().manual_seed(1)
    x, dy, w, b = (torch.randn(s, generator=g, dtype=torch.float64) for s in ((5, 12), (5, 12), (12,), (12,)))
    x.requires_grad_(), w.requires_grad_(), b.requires_grad_()
    (y, mean, rstd), _ = ref.norm(x, w, b, 1e-5)
    want = torch.autograd.grad((y * dy).sum(), (x, w, b))
    got, _ = ref.norm_back(x.detach(), w.detach(), mean.detach(), rstd.detach(), dy, None)
    for a, c in zip(got, want):
        assert torch.allclose(a, c, rtol=1e-12, atol=1e-12)


@pytest.mark.parametrize("kind", ["gelu", "silu", "relu"])
def test_activation_derivative(kind):
    g = torch.linspace(-6, 6, 401, dtype=torch.float64) + 1e-3
    h = 1e-6
    a, d = ref.act(g, kind)
    num = (ref.act(g + h, kind)[0] - ref.act(g - h, kind)[0]) / (2 * h)
    assert torch.allclose(d, num, atol=1e-8)
