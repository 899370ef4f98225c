"""Row layouts that the trainable sub-block's C entries take or refuse, beside those of test_train_refusals.py:
without a GPU, where a call that is let through ends with the missing device."""
import pytest

from prism_inference_b200 import abi

from test_train_refusals import at, ctx, drop, gated, gated_back, lib, norm, norm_back  # noqa: F401

RANGE, CUDA = abi.PRISM_E_RANGE, abi.PRISM_E_CUDA


@pytest.mark.parametrize("stride", [0, -8, 1 << 62])
@pytest.mark.parametrize("call,names", [(norm, "x y"), (norm_back, "x dy add dx"), (drop, "x residual y"), (gated, "x residual y"),
                                        (gated_back, "x dy dx")])
def test_the_stride_of_a_single_row_is_ignored(lib, ctx, call, names, stride):  # noqa: F811
    assert call(lib, ctx, rows=1, **{f"{n}_stride": stride for n in names.split()}) == CUDA


@pytest.mark.parametrize("call,names", [(norm, "x y"), (norm_back, "x dy add dx"), (drop, "x residual y"), (gated, "x residual y"),
                                        (gated_back, "x dy dx")])
def test_extents_beyond_64_bits_are_refused(lib, ctx, call, names):  # noqa: F811
    """rows and stride each within its limit, their product beyond what an address or the kernels' offsets hold."""
    for n in names.split():
        for rows, stride in ((1 << 40, 1 << 36), (1 << 30, 1 << 36), (1 << 40, 1 << 23)):
            assert call(lib, ctx, **{"rows": rows, "ws_bytes": 1 << 62, f"{n}_stride": stride}) == RANGE, (n, rows, stride)
