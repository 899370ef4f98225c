"""What the trainable sub-block's entry points refuse, without a GPU: every check comes before any CUDA
work, so a context that was never created (its struct by hand) and made-up addresses do."""
import ctypes as C

import pytest

from prism_inference_b200 import abi
from prism_inference_b200.abi import DropoutParams, GatedGrads, GatedParams, GatedWeights, NormParams

from test_abi import _header_struct_fields, lib  # noqa: F401

ARG, ALIGN, RANGE, UNSUPPORTED = abi.PRISM_E_ARG, abi.PRISM_E_ALIGN, abi.PRISM_E_RANGE, abi.PRISM_E_UNSUPPORTED
BASE = 1 << 40  # addresses far from one another, never touched


class Ctx(C.Structure):
    _fields_ = [("device", C.c_int), ("sm_count", C.c_int), ("err", C.c_void_p), ("codec", C.c_void_p)]


@pytest.fixture(scope="module")
def ctx():
    import torch
    if torch.cuda.is_available():
        pytest.skip("a GPU is present: what is not refused would run")
    return Ctx(0, 148, None, None)


def at(k):
    return BASE + k * (1 << 32)


def norm(lib, ctx, p=None, **kw):  # noqa: F811
    q = dict(rows=16, dim=64, x_stride=64, y_stride=64, dtype=0, param_dtype=0, eps=1e-5)
    a = dict(x=at(0), weight=at(1), bias=at(2), y=at(3), mean=at(4), rstd=at(5))
    q.update({k: v for k, v in kw.items() if k in q})
    a.update({k: v for k, v in kw.items() if k in a})
    return lib.prism_layer_norm(C.byref(ctx), C.byref(NormParams(**q)), *a.values(), None)


def norm_back(lib, ctx, **kw):  # noqa: F811
    q = dict(rows=16, dim=64, x_stride=64, dy_stride=64, add_stride=64, dx_stride=64, dtype=0, param_dtype=2)
    a = dict(x=at(0), weight=at(1), mean=at(2), rstd=at(3), dy=at(4), add=at(5), dx=at(6), dweight=at(7), dbias=at(8),
             ws=at(9), ws_bytes=1 << 30)
    q.update({k: v for k, v in kw.items() if k in q})
    a.update({k: v for k, v in kw.items() if k in a})
    return lib.prism_layer_norm_backward(C.byref(ctx), C.byref(NormParams(**q)), *a.values(), None)


def drop(lib, ctx, **kw):  # noqa: F811
    q = dict(rows=16, dim=64, x_stride=64, residual_stride=64, y_stride=64, dtype=0, threshold=100)
    a = dict(x=at(0), residual=at(1), rng=at(2), y=at(3))
    q.update({k: v for k, v in kw.items() if k in q})
    a.update({k: v for k, v in kw.items() if k in a})
    return lib.prism_dropout_add(C.byref(ctx), C.byref(DropoutParams(**q)), *a.values(), None)


GATED = dict(rows=300, dim=64, hidden=128, x_stride=64, residual_stride=64, y_stride=64, dy_stride=64, dx_stride=64, dtype=0,
             activation=0)
WEIGHTS = {n: at(20 + i) for i, (n, _) in enumerate(GatedWeights._fields_)}


def gated(lib, ctx, **kw):  # noqa: F811
    q, w = dict(GATED), dict(WEIGHTS)
    a = dict(x=at(0), residual=at(1), y=at(2), ws=at(3), ws_bytes=1 << 30)
    for d in (q, w, a):
        d.update({k: v for k, v in kw.items() if k in d})
    return lib.prism_gated_ffn(C.byref(ctx), C.byref(GatedParams(**q)), C.byref(GatedWeights(**w)), *a.values(), None)


def gated_back(lib, ctx, **kw):  # noqa: F811
    q, w = dict(GATED), dict(WEIGHTS)
    g = {n: at(30 + i) for i, (n, _) in enumerate(GatedGrads._fields_)}
    a = dict(x=at(0), dy=at(1), dx=at(2))
    e = dict(ws=at(3), ws_bytes=1 << 34)
    for d in (q, w, g, a, e):
        d.update({k: v for k, v in kw.items() if k in d})
    return lib.prism_gated_ffn_backward(C.byref(ctx), C.byref(GatedParams(**q)), C.byref(GatedWeights(**w)), *a.values(),
                                        C.byref(GatedGrads(**g)), *e.values(), None)


CASES = [
    (norm, dict(dtype=3), ARG), (norm, dict(dtype=-1), ARG), (norm, dict(param_dtype=1), ARG), (norm, dict(rows=-1), ARG),
    (norm, dict(dim=0), ARG), (norm, dict(dim=16385, x_stride=16385, y_stride=16385), UNSUPPORTED), (norm, dict(x=None), ARG),
    (norm, dict(y=None), ARG), (norm, dict(x=at(0) + 1), ALIGN), (norm, dict(weight=at(1) + 1), ALIGN), (norm, dict(mean=at(4) + 2), ALIGN),
    (norm, dict(x_stride=63), ARG), (norm, dict(y_stride=0), ARG), (norm, dict(y_stride=-64), ARG), (norm, dict(x_stride=1 << 41), RANGE),
    (norm, dict(y=at(0) + 2), ARG), (norm, dict(y=at(0) - 64), ARG), (norm, dict(y=at(0), y_stride=128), ARG),
    (norm, dict(rows=(1 << 40) + 1), RANGE),
    (norm_back, dict(mean=None), ARG), (norm_back, dict(rstd=None), ARG), (norm_back, dict(dy=None), ARG), (norm_back, dict(dx=None), ARG),
    (norm_back, dict(ws=None), ARG), (norm_back, dict(ws_bytes=16 * 2 * 64 * 4 - 1), ARG), (norm_back, dict(ws=at(9) + 4), ALIGN),
    (norm_back, dict(dx=at(4) + 16), ARG), (norm_back, dict(dx=at(5) - 2), ARG), (norm_back, dict(add_stride=10), ARG),
    (norm_back, dict(dweight=at(7) + 2), ALIGN), (norm_back, dict(param_dtype=1), ARG),
    (drop, dict(threshold=-1), ARG), (drop, dict(threshold=65536), ARG), (drop, dict(dtype=7), ARG), (drop, dict(rng=None), ARG),
    (drop, dict(rng=at(2) + 4), ALIGN), (drop, dict(x=None), ARG), (drop, dict(y=at(1) + 2), ARG), (drop, dict(residual_stride=5), ARG),
    (drop, dict(dim=-3), ARG),
    (gated, dict(dtype=2), UNSUPPORTED), (gated, dict(dtype=5), ARG), (gated, dict(activation=3), ARG), (gated, dict(activation=-1), ARG),
    (gated, dict(dim=60), UNSUPPORTED), (gated, dict(hidden=100), UNSUPPORTED), (gated, dict(hidden=0), ARG),
    (gated, dict(hidden=65544), UNSUPPORTED), (gated, dict(rows=-5), ARG), (gated, dict(x=None), ARG), (gated, dict(y=None), ARG),
    (gated, dict(w_gate=None), ARG), (gated, dict(w_up=None), ARG), (gated, dict(w_down=None), ARG), (gated, dict(w_up=at(22) + 8), ALIGN),
    (gated, dict(b_gate=at(21) + 1), ALIGN), (gated, dict(x=at(0) + 8), ALIGN), (gated, dict(x_stride=68), ALIGN),
    (gated, dict(y_stride=56), ARG), (gated, dict(residual=at(1) + 2), ALIGN), (gated, dict(y=at(0)), ARG), (gated, dict(y=at(1) + 32), ARG),
    (gated, dict(rows=4, ws=None), ARG), (gated, dict(rows=4, ws_bytes=4 * 128 * 4 - 1), ARG), (gated, dict(rows=4, ws=at(3) + 4), ALIGN),
    (gated, dict(dim=264, x_stride=264, y_stride=264, residual_stride=264, ws_bytes=300 * 128 * 2 - 1), ARG),
    (gated_back, dict(dy=None), ARG), (gated_back, dict(dx=None), ARG), (gated_back, dict(dx=at(0)), ARG), (gated_back, dict(dx=at(1) + 64), ARG),
    (gated_back, dict(dy_stride=72, dy=at(1) + 4), ALIGN), (gated_back, dict(ws_bytes=1000), ARG), (gated_back, dict(ws=None), ARG),
    (gated_back, dict(dw_down=at(34) + 1), ALIGN), (gated_back, dict(w_gate=None), ARG),
]


@pytest.mark.parametrize("call,change,code", CASES, ids=lambda v: getattr(v, "__name__", str(v))[:60])
def test_refused(lib, ctx, call, change, code):  # noqa: F811
    assert call(lib, ctx, **change) == code
    assert lib.prism_last_error_string()


@pytest.mark.parametrize("call", [norm, drop, gated])
def test_no_rows_is_a_no_op(lib, ctx, call):  # noqa: F811
    assert call(lib, ctx, rows=0, x=None, y=None) == abi.PRISM_OK


def test_null_arguments(lib, ctx):  # noqa: F811
    n = C.c_size_t()
    for rc in (lib.prism_layer_norm(None, None, None, None, None, None, None, None, None),
               lib.prism_layer_norm_backward(None, None, *[None] * 10, 0, None),
               lib.prism_layer_norm_backward_workspace(C.byref(ctx), None, C.byref(n)),
               lib.prism_layer_norm_backward_workspace(C.byref(ctx), C.byref(NormParams(rows=1, dim=8)), None),
               lib.prism_dropout_add(None, None, None, None, None, None, None),
               lib.prism_gated_ffn(None, None, None, None, None, None, None, 0, None),
               lib.prism_gated_ffn_backward(None, None, None, None, None, None, None, None, 0, None),
               lib.prism_gated_ffn_workspace(C.byref(ctx), None, 0, C.byref(n))):
        assert rc == ARG


def test_workspaces_stay_bounded(lib, ctx):  # noqa: F811
    def size(backward, **kw):
        n = C.c_size_t()
        assert lib.prism_gated_ffn_workspace(C.byref(ctx), C.byref(GatedParams(**dict(GATED, **kw))), backward, C.byref(n)) == 0
        return n.value
    big = dict(dim=256, hidden=1024)
    assert size(0, rows=10 ** 9, **big) == 0 and size(0, rows=3, **big) == 3 * 1024 * 4
    assert size(0, rows=1000, dim=512, hidden=1024) == 1000 * 1024 * 2
    assert size(0, rows=10 ** 9, dim=512, hidden=1024) <= 1 << 30
    assert size(1, rows=10 ** 9, **big) <= (1 << 30) + (1 << 26)
    assert size(1, rows=0, **big) == 0


@pytest.mark.parametrize("cname,pyt", [("prism_norm_params", NormParams), ("prism_dropout_params", DropoutParams),
                                       ("prism_gated_params", GatedParams), ("prism_gated_weights", GatedWeights),
                                       ("prism_gated_grads", GatedGrads)])
def test_struct_layout_matches_header(cname, pyt):
    assert [f for f, _ in pyt._fields_] == [n.lstrip("* ") for n in _header_struct_fields(cname)]
