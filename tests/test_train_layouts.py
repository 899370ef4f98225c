"""Row layouts that the trainable sub-block's C entries take or refuse, beside those of test_train_refusals.py:
without a GPU, where a call that is let through ends with the missing device."""
import ctypes as C

import pytest

from prism_inference_b200 import abi
from prism_inference_b200.abi import GatedParams

from test_train_refusals import GATED, at, ctx, drop, gated, gated_back, lib, norm, norm_back  # noqa: F401

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


GRADS = ("dw_gate", "db_gate", "dw_up", "db_up", "dw_down", "db_down")


@pytest.mark.parametrize("rows", [0, 16])
@pytest.mark.parametrize("i,j", [(i, j) for j in range(6) for i in range(j)])
def test_gradients_that_share_memory_are_refused(lib, ctx, rows, i, j):  # noqa: F811
    """One address for two gradients, or the second beginning in the first's last value (dim 64, hidden 128, fp16)."""
    sizes = {"dw_gate": 64 * 128, "db_gate": 128, "dw_up": 64 * 128, "db_up": 128, "dw_down": 64 * 128, "db_down": 64}
    a, b = GRADS[i], GRADS[j]
    for first, second in ((a, b), (b, a)):
        for off in (0, 2 * sizes[first] - 2):
            assert gated_back(lib, ctx, rows=rows, **{first: at(50), second: at(50) + off}) == abi.PRISM_E_ARG
            assert b"overlap" in lib.prism_last_error_string()
        if rows:  # side by side in one buffer
            assert gated_back(lib, ctx, rows=rows, **{first: at(50), second: at(50) + 2 * sizes[first]}) == CUDA


def test_statistics_and_parameter_gradients_that_share_memory_are_refused(lib, ctx):  # noqa: F811
    for off in (0, 60, -60):
        assert norm(lib, ctx, mean=at(50), rstd=at(50) + off) == abi.PRISM_E_ARG and b"overlap" in lib.prism_last_error_string()
    assert norm(lib, ctx, mean=at(50), rstd=at(50) + 64) == CUDA
    for rows in (0, 16):
        for off in (0, 252, -252):  # dim 64, fp32
            assert norm_back(lib, ctx, rows=rows, dweight=at(50), dbias=at(50) + off) == abi.PRISM_E_ARG
            assert b"overlap" in lib.prism_last_error_string()
    assert norm_back(lib, ctx, dweight=at(50), dbias=at(50) + 256) == CUDA
    assert norm_back(lib, ctx, dweight=None, dbias=at(50)) == CUDA


@pytest.mark.parametrize("dim", [64, 256, 264, 4096, 16384])
@pytest.mark.parametrize("hidden", [1024, 9440, 9448, 14336, 28336, 28344, 65536])
def test_workspace_is_what_the_header_says(lib, ctx, dim, hidden):  # noqa: F811
    """A chunk of rows takes the larger of 1 GiB and one wave (128 rows an SM) at most, however many rows there are;
    the gradients' partial sums come on top backward."""
    def size(backward, rows):
        n, p = C.c_size_t(), GatedParams(**dict(GATED, rows=rows, dim=dim, hidden=hidden))
        assert lib.prism_gated_ffn_workspace(C.byref(ctx), C.byref(p), backward, C.byref(n)) == 0
        return n.value
    wave, rows = 128 * 148, 10 ** 8
    chunk = max(1 << 30, wave * 2 * hidden)
    assert (wave * 2 * hidden > 1 << 30) == (hidden > 28336) and (wave * 6 * hidden > 1 << 30) == (hidden > 9440)
    assert size(0, rows) == 0 if dim <= 256 else chunk // 2 < size(0, rows) <= chunk
    chunk = max(1 << 30, wave * 6 * hidden)
    tiles = 3 * -(-hidden // 256) * -(-dim // 256)
    sums = max(1, 74 // tiles) * 12 * hidden * dim + 4 * (8 * 74 * 2 * hidden + (2 * 74 + 16 * 24) * dim)
    assert chunk // 2 < size(1, rows) <= chunk + sums + 2048
