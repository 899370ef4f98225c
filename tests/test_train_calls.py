"""The Python methods of the trainable sub-block without a GPU: tensors without memory and a library that only
notes what it was called with."""
import pytest
import torch

from prism_inference_b200 import Prism

F16 = torch.float16


class Lib:
    """Notes the params of each call and answers 0."""
    def __init__(self):
        self.seen = []

    def __getattr__(self, name):
        if not name.startswith("prism_"):
            raise AttributeError(name)
        return lambda h, p, *a: self.seen.append((name, p._obj)) or 0


@pytest.fixture
def ctx():
    c = Prism.__new__(Prism)  # meta tensors are on "device" -1
    c.lib, c.device, c.h, c._workspaces = Lib(), torch.empty(1, device="meta").get_device(), None, {}
    return c


def meta(*shape, dtype=F16):
    return torch.empty(shape, dtype=dtype, device="meta")


@pytest.mark.parametrize("dim", [2 ** 31, 2 ** 32 + 8])
def test_sizes_beyond_32_bits_are_refused(ctx, dim):
    """The params hold dim and hidden in 32 bits: 2^32 + 8 columns must not become 8."""
    x, rng = meta(1, dim), meta(2, dtype=torch.int64)
    with pytest.raises(ValueError, match="2\\^31"):
        ctx.dropout_add(x, None, x, 0.5, rng, stream=0)
    with pytest.raises(ValueError, match="2\\^31"):
        ctx.dropout_add(meta(dim), None, meta(dim), 0.5, rng, stream=0)
    with pytest.raises(ValueError, match="2\\^31"):
        ctx.layer_norm(x, None, None, x, stream=0)
    with pytest.raises(ValueError, match="2\\^31"):
        ctx.gated_ffn(x, meta(8, dim), meta(8, dim), meta(dim, 8), meta(1, dim), stream=0)
    with pytest.raises(ValueError, match="2\\^31"):
        ctx.gated_ffn(meta(1, 8), meta(dim, 8), meta(dim, 8), meta(8, dim), meta(1, 8), stream=0)
    assert not ctx.lib.seen


def test_sizes_arrive(ctx):
    x, rng = meta(2 ** 33, 24), meta(2, dtype=torch.int64)
    ctx.dropout_add(x, None, x, 0.5, rng, stream=0)
    ctx.layer_norm(x[:, :16], None, None, meta(2 ** 33, 16), stream=0)
    ctx.gated_ffn(x, meta(40, 24), meta(40, 24), meta(24, 40), x, stream=0)
    (_, d), (_, n), (_, _), (_, g) = ctx.lib.seen
    assert (d.rows, d.dim, d.x_stride, d.threshold) == (2 ** 33, 24, 24, 32768)
    assert (n.rows, n.dim, n.x_stride, n.y_stride) == (2 ** 33, 16, 24, 16)
    assert (g.rows, g.dim, g.hidden) == (2 ** 33, 24, 40)
