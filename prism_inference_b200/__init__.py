"""prism_inference_b200 - B200 (sm_100a) implementation of Prism's bottleneck
transformer / MoE stack behind the C ABI of include/prism_moe.h.

The Python layer is a thin host mirror over libprism_moe.so (ctypes): PyTorch is
used only to own device memory and streams.  Three interfaces:

* the per-pass drop-ins, one call per reference vkCmdDispatch, taking the same
  push-constant blocks (AttnParams, RouterParams, ExpertParams, ProjParams,
  DenseParams) and the three arenas (fp16 weight blob, fp16 feature arena, int32 aux
  arena) - the dispatch contract of prism_moe_bench.cpp:213-505;
* Stack: the whole stack of a StackLayout over a batch of frames (the fast path);
* the trainable pre-norm gated feed-forward sub-block on the caller's own tensors: layer_norm,
  gated_ffn, dropout_add and their backward passes (methods of Prism).

No entry point falls back to the CPU: a missing libprism_moe.so raises.
"""
from __future__ import annotations

import ctypes as C
import functools

from . import abi, configs, layout, synth
from .abi import (AttnParams, DenseParams, DropoutParams, ExpertParams, GatedGrads, GatedParams, GatedWeights, NormParams,
                  PrismError, ProjParams, RouterParams, check)
from .layout import StackLayout, build_stack

__all__ = ["Prism", "Stack", "AttnParams", "RouterParams", "ExpertParams", "ProjParams",
           "DenseParams", "PrismError", "StackLayout", "build_stack", "configs", "layout", "synth"]


def _ptr(t) -> int:
    return t.data_ptr()


def _host_ptr(a) -> int | None:
    """Address of a host array (CPU tensor or numpy array); None passes through."""
    if a is None:
        return None
    if hasattr(a, "data_ptr"):
        if a.is_cuda or not a.is_contiguous():
            raise ValueError("expected a contiguous host tensor")
        return a.data_ptr()
    if not a.flags["C_CONTIGUOUS"]:
        raise ValueError("expected a C-contiguous array")
    return a.ctypes.data


def _stream(stream) -> int | None:
    if stream is None:
        import torch
        return torch.cuda.current_stream().cuda_stream
    return getattr(stream, "cuda_stream", stream)


_DTYPES = {}  # torch dtype -> prism_dtype


def _dtype(t, name: str) -> int:
    code = _DTYPES.get(t.dtype)
    if code is None:
        import torch
        _DTYPES.update({getattr(torch, d): i for i, d in enumerate(abi.DTYPES)})
        if t.dtype not in _DTYPES:
            raise ValueError(f"{name}: dtype {t.dtype} (fp16, bf16 or fp32)")
        code = _DTYPES[t.dtype]
    return code


@functools.lru_cache(None)
def _F32():
    import torch
    return torch.float32


@functools.lru_cache(None)
def _raw_stream():
    """device -> handle of torch's current stream (torch.cuda.current_stream makes an object for it)."""
    import torch
    return getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda d: torch.cuda.current_stream(d).cuda_stream)


@functools.lru_cache(None)
def _I64():
    import torch
    return torch.int64


# These run on every call of the operators below, whose smallest calls take less time than their
# checks: few attribute look-ups (a tensor's shape, device and so on are objects made anew each time).
_MAX32 = 2 ** 31 - 1  # the params' fields for sizes; ctypes drops the bits above without a word


def _rows(t, name: str):
    """(rows, dim, row stride) of a tensor [..., dim] whose last dimension is consecutive in memory."""
    shape = t.shape
    if len(shape) == 2:
        rows, dim = shape
        if dim > _MAX32:
            raise ValueError(f"{name}: {dim} columns, 2^31 - 1 at most (as rows of fewer columns any number of elements)")
        stride, last = t.stride()
        if last != 1 and dim > 1:
            raise ValueError(f"{name}: the last dimension is not consecutive in memory")
        return rows, dim, stride if rows > 1 else dim
    if len(shape) < 1 or (shape[-1] > 1 and t.stride(-1) != 1):
        raise ValueError(f"{name}: the last dimension is not consecutive in memory")
    dim = shape[-1]
    if dim > _MAX32:
        raise ValueError(f"{name}: {dim} columns, 2^31 - 1 at most (as rows of fewer columns any number of elements)")
    rows, stride = t.numel() // max(1, dim), dim
    if not t.is_contiguous():
        try:
            stride = t.view(-1, dim).stride(0)
        except RuntimeError:
            raise ValueError(f"{name}: its rows do not lie at one stride") from None
    return rows, dim, stride if rows > 1 else dim


def _stride(t, name: str, dtype, device: int, rows: int, dim: int) -> int:
    """Row stride of a tensor [..., dim] that has to be of this type, device and size."""
    r, d, stride = _rows(t, name)
    if r != rows or d != dim or t.dtype is not dtype or t.get_device() != device:
        raise ValueError(f"{name}: {t.dtype} {list(t.shape)} on {t.device}, expected {dtype} [{rows}, {dim}] on cuda:{device}")
    return stride


def _flat(t, name: str, shape, dtype, device: int) -> int | None:
    """Address of a contiguous parameter, gradient or statistics tensor; None passes through."""
    if t is None:
        return None
    if t.shape != shape or t.dtype is not dtype or t.get_device() != device or not t.is_contiguous():
        raise ValueError(f"{name}: expected a contiguous {dtype} {list(shape)} on cuda:{device}, got {t.dtype} "
                         f"{list(t.shape)} on {t.device}")
    return t.data_ptr()


def _workspace(workspace, nbytes: int, device: int, stream):
    """(tensor, address, bytes): the caller's workspace, or one from torch's allocator that belongs to
    the call's stream (so it is not handed out again before the call's work has run)."""
    if workspace is not None:
        if workspace.get_device() != device or not workspace.is_contiguous():
            raise ValueError(f"workspace: expected a contiguous tensor on cuda:{device}")
        return workspace, workspace.data_ptr(), workspace.numel() * workspace.element_size()
    if not nbytes:
        return None, None, 0
    import torch
    if stream is None:
        w = torch.empty(nbytes, dtype=torch.uint8, device=device)
    else:
        if not hasattr(stream, "cuda_stream"):
            stream = torch.cuda.ExternalStream(stream, device=device)
        with torch.cuda.stream(stream):
            w = torch.empty(nbytes, dtype=torch.uint8, device=device)
    return w, w.data_ptr(), nbytes


class Prism:
    """One context per CUDA device (prism_create)."""

    def __init__(self, device: int = 0):
        self.lib = abi.load()
        self.device = device
        self._workspaces = {}  # bytes of scratch by call and sizes
        h = C.c_void_p()
        check(self.lib, self.lib.prism_create(device, C.byref(h)))
        self.h = h

    def close(self):
        if self.h:
            self.lib.prism_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    # ---- per-pass drop-ins (tensors are flat CUDA arenas) ------------------------
    def attn_window(self, p: AttnParams, weights, features, stream=None):
        check(self.lib, self.lib.prism_attn_window(self.h, C.byref(p), _ptr(weights), weights.numel(),
                                                   _ptr(features), features.numel(), _stream(stream)))

    def router(self, p: RouterParams, weights, features, aux, stream=None):
        check(self.lib, self.lib.prism_router(self.h, C.byref(p), _ptr(weights), weights.numel(),
                                              _ptr(features), features.numel(), _ptr(aux), aux.numel(),
                                              _stream(stream)))

    def expert(self, p: ExpertParams, weights, features, aux, stream=None):
        check(self.lib, self.lib.prism_expert(self.h, C.byref(p), _ptr(weights), weights.numel(),
                                              _ptr(features), features.numel(), _ptr(aux), aux.numel(),
                                              _stream(stream)))

    def expert_all_static(self, p: ExpertParams, n_experts: int, expert_stride: int, weights, features, aux,
                          stream=None):
        """All experts of one pass in one call without device allocation
        (prism_expert_all_static): scratch lives in a fixed per-device array."""
        check(self.lib, self.lib.prism_expert_all_static(self.h, C.byref(p), n_experts, expert_stride, _ptr(weights),
                                                         weights.numel(), _ptr(features), features.numel(), _ptr(aux),
                                                         aux.numel(), _stream(stream)))

    def proj_up(self, p: ProjParams, weights, features, stream=None):
        check(self.lib, self.lib.prism_proj_up(self.h, C.byref(p), _ptr(weights), weights.numel(),
                                               _ptr(features), features.numel(), _stream(stream)))

    def proj_down(self, p: ProjParams, weights, features, stream=None):
        check(self.lib, self.lib.prism_proj_down(self.h, C.byref(p), _ptr(weights), weights.numel(),
                                                 _ptr(features), features.numel(), _stream(stream)))

    def dense_block(self, p: DenseParams, ffn_hidden: int, ffn_chunk: int, weights, features, stream=None):
        check(self.lib, self.lib.prism_dense_block(self.h, C.byref(p), ffn_hidden, ffn_chunk, _ptr(weights),
                                                   weights.numel(), _ptr(features), features.numel(),
                                                   _stream(stream)))

    def codec_pass(self, shader: str, push, weights, features, rgb=None, stream=None):
        """prism_codec_pass: one dispatch of an encoder / decoder shader (abi.CODEC_KINDS) with
        its push constants, on CUDA fp16 tensors (weights = binding 0, features = binding 1,
        rgb = binding 2 for pixelshuffle_sigmoid)."""
        pc = (C.c_int32 * len(push))(*[int(v) for v in push])
        check(self.lib, self.lib.prism_codec_pass(self.h, abi.CODEC_KINDS.index(shader), pc, len(push),
                                                  _ptr(weights), weights.numel(), _ptr(features), features.numel(),
                                                  _ptr(rgb) if rgb is not None else None,
                                                  rgb.numel() if rgb is not None else 0, _stream(stream)))

    # ---- the trainable pre-norm gated feed-forward sub-block (caller-owned CUDA tensors) ----
    # Tensors are [..., dim] with the last dimension consecutive and the rows at one stride (column
    # slices of wider buffers work); the caller allocates outputs.  stream: None = torch's current
    # stream of the context's device; tensors made on another stream are the caller's to order.
    # workspace: scratch memory of at least the *_workspace() bytes, None = from torch's allocator.
    def _stream(self, stream):
        if stream is None:
            return _raw_stream()(self.device)
        return getattr(stream, "cuda_stream", stream)

    def _scratch(self, query, p, key, *args) -> int:
        """Bytes of workspace that `query` answers for params p: a function of the sizes in `key`, asked once."""
        n = self._workspaces.get(key)
        if n is None:
            need = C.c_size_t()
            check(self.lib, query(self.h, C.byref(p), *args, C.byref(need)))
            if len(self._workspaces) >= 1024:  # ragged batches: sizes that hardly come again
                self._workspaces.clear()
            n = self._workspaces[key] = need.value
        return n

    @staticmethod
    def _param_dtype(x, *params):
        """dtype of the norm's parameters: the first given one's (fp32 or the rows' own), else the rows'."""
        for p in params:
            if p is not None:
                return p.dtype
        return x.dtype

    def layer_norm(self, x, weight, bias, y, eps: float = 1e-5, mean=None, rstd=None, stream=None):
        """prism_layer_norm: y = (x - mean) * rstd * weight + bias over the last dimension.  weight, bias
        ([dim], x's dtype or fp32) and the fp32 statistics mean, rstd ([rows]) are optional."""
        dev, dt, (rows, dim, xs) = self.device, x.dtype, _rows(x, "x")
        if x.get_device() != dev:
            raise ValueError(f"x: on {x.device}, the context is for cuda:{dev}")
        code, pt = _dtype(x, "x"), self._param_dtype(x, weight, bias)
        p = NormParams(rows, xs, _stride(y, "y", dt, dev, rows, dim), 0, 0, 0, dim, code, _DTYPES.get(pt, -1), eps)
        f32 = _F32()
        rc = self.lib.prism_layer_norm(
            self.h, C.byref(p), x.data_ptr(), _flat(weight, "weight", (dim,), pt, dev), _flat(bias, "bias", (dim,), pt, dev),
            y.data_ptr(), _flat(mean, "mean", (rows,), f32, dev), _flat(rstd, "rstd", (rows,), f32, dev), self._stream(stream))
        if rc:
            check(self.lib, rc)
        return y

    def layer_norm_backward(self, x, weight, mean, rstd, dy, dx, dweight=None, dbias=None, add=None, workspace=None,
                            stream=None):
        """prism_layer_norm_backward: dx (+ add, the gradient that came past the norm), and the parameters'
        gradients where dweight, dbias are given (overwritten)."""
        dev, dt, (rows, dim, xs) = self.device, x.dtype, _rows(x, "x")
        if x.get_device() != dev:
            raise ValueError(f"x: on {x.device}, the context is for cuda:{dev}")
        code, pt = _dtype(x, "x"), self._param_dtype(x, weight, dweight, dbias)
        p = NormParams(rows, xs, 0, _stride(dy, "dy", dt, dev, rows, dim),
                       0 if add is None else _stride(add, "add", dt, dev, rows, dim), _stride(dx, "dx", dt, dev, rows, dim), dim,
                       code, _DTYPES.get(pt, -1), 0.0)
        need = 0
        if dweight is not None or dbias is not None:
            need = self._scratch(self.lib.prism_layer_norm_backward_workspace, p, ("norm", rows, dim, code, pt))
        keep, ws, ws_bytes = _workspace(workspace, need, dev, stream)
        f32 = _F32()
        rc = self.lib.prism_layer_norm_backward(
            self.h, C.byref(p), x.data_ptr(), _flat(weight, "weight", (dim,), pt, dev), _flat(mean, "mean", (rows,), f32, dev),
            _flat(rstd, "rstd", (rows,), f32, dev), dy.data_ptr(), None if add is None else add.data_ptr(), dx.data_ptr(),
            _flat(dweight, "dweight", (dim,), pt, dev), _flat(dbias, "dbias", (dim,), pt, dev), ws, ws_bytes,
            self._stream(stream))
        if rc:
            check(self.lib, rc)
        return dx

    def dropout_add(self, x, residual, y, p: float, rng, stream=None):
        """prism_dropout_add: y = residual + dropout(x) (residual None: dropout(x)), dropping with probability
        round(65536 p) / 65536.  rng: CUDA int64 [2] {seed, offset}, read when the call runs.  The gradient:
        the same call on it, with the same p and rng and no residual."""
        dev, dt, (rows, dim, xs) = self.device, x.dtype, _rows(x, "x")
        if x.get_device() != dev:
            raise ValueError(f"x: on {x.device}, the context is for cuda:{dev}")
        rs = 0 if residual is None else _stride(residual, "residual", dt, dev, rows, dim)
        q = DropoutParams(rows, xs, rs, _stride(y, "y", dt, dev, rows, dim), dim, _dtype(x, "x"),
                          max(-1, min(65536, int(round(65536 * p)))))
        rc = self.lib.prism_dropout_add(self.h, C.byref(q), x.data_ptr(), None if residual is None else residual.data_ptr(),
                                        _flat(rng, "rng", (2,), _I64(), dev), y.data_ptr(), self._stream(stream))
        if rc:
            check(self.lib, rc)
        return y

    def _gated(self, x, w_gate, w_up, w_down, b_gate, b_up, b_down, activation):
        """(params, weights, dtype, rows, dim, hidden) of a gated feed-forward call."""
        dev, dt, (rows, dim, xs) = self.device, x.dtype, _rows(x, "x")
        if x.get_device() != dev:
            raise ValueError(f"x: on {x.device}, the context is for cuda:{dev}")
        if activation not in abi.ACTIVATIONS:
            raise ValueError(f"activation {activation!r}: one of {', '.join(abi.ACTIVATIONS)}")
        hidden = w_gate.shape[0]
        if hidden > _MAX32:
            raise ValueError(f"w_gate: {hidden} rows, 2^31 - 1 at most")
        w = GatedWeights(_flat(w_gate, "w_gate", (hidden, dim), dt, dev), _flat(b_gate, "b_gate", (hidden,), dt, dev),
                         _flat(w_up, "w_up", (hidden, dim), dt, dev), _flat(b_up, "b_up", (hidden,), dt, dev),
                         _flat(w_down, "w_down", (dim, hidden), dt, dev), _flat(b_down, "b_down", (dim,), dt, dev))
        p = GatedParams(rows, xs, 0, 0, 0, 0, dim, hidden, _dtype(x, "x"), abi.ACTIVATIONS.index(activation))
        return p, w, dt, rows, dim, hidden

    def gated_ffn(self, x, w_gate, w_up, w_down, y, b_gate=None, b_up=None, b_down=None, residual=None,
                  activation: str = "gelu", workspace=None, stream=None):
        """prism_gated_ffn: y = w_down (act(w_gate x + b_gate) * (w_up x + b_up)) + b_down + residual, fp16 or
        bf16; activation "gelu" (tanh form), "silu" or "relu"."""
        p, w, dt, rows, dim, hidden = self._gated(x, w_gate, w_up, w_down, b_gate, b_up, b_down, activation)
        dev = self.device
        p.y_stride = _stride(y, "y", dt, dev, rows, dim)
        if residual is not None:
            p.residual_stride = _stride(residual, "residual", dt, dev, rows, dim)
        need = self._scratch(self.lib.prism_gated_ffn_workspace, p, ("gated", rows, dim, hidden, p.dtype), 0)
        keep, ws, ws_bytes = _workspace(workspace, need, dev, stream)
        rc = self.lib.prism_gated_ffn(self.h, C.byref(p), C.byref(w), x.data_ptr(),
                                      None if residual is None else residual.data_ptr(), y.data_ptr(), ws, ws_bytes,
                                      self._stream(stream))
        if rc:
            check(self.lib, rc)
        return y

    def gated_ffn_backward(self, x, w_gate, w_up, w_down, dy, dx, dw_gate=None, dw_up=None, dw_down=None, b_gate=None,
                           b_up=None, db_gate=None, db_up=None, db_down=None, activation: str = "gelu", workspace=None,
                           stream=None):
        """prism_gated_ffn_backward: dx and the parameters' gradients that are given (overwritten), from x, the
        weights and dy; the forward pass has nothing to keep.  The residual's gradient is dy itself."""
        p, w, dt, rows, dim, hidden = self._gated(x, w_gate, w_up, w_down, b_gate, b_up, None, activation)
        dev = self.device
        p.dy_stride, p.dx_stride = _stride(dy, "dy", dt, dev, rows, dim), _stride(dx, "dx", dt, dev, rows, dim)
        d = GatedGrads(_flat(dw_gate, "dw_gate", (hidden, dim), dt, dev), _flat(db_gate, "db_gate", (hidden,), dt, dev),
                       _flat(dw_up, "dw_up", (hidden, dim), dt, dev), _flat(db_up, "db_up", (hidden,), dt, dev),
                       _flat(dw_down, "dw_down", (dim, hidden), dt, dev), _flat(db_down, "db_down", (dim,), dt, dev))
        need = self._scratch(self.lib.prism_gated_ffn_workspace, p, ("gated back", rows, dim, hidden, p.dtype), 1)
        keep, ws, ws_bytes = _workspace(workspace, need, dev, stream)
        rc = self.lib.prism_gated_ffn_backward(self.h, C.byref(p), C.byref(w), x.data_ptr(), dy.data_ptr(), dx.data_ptr(),
                                               C.byref(d), ws, ws_bytes, self._stream(stream))
        if rc:
            check(self.lib, rc)
        return dx

    def status(self, stream=None):
        """prism_ctx_status: raises PrismError if a per-pass kernel's bounded wait gave up."""
        check(self.lib, self.lib.prism_ctx_status(self.h, _stream(stream)))


class Stack:
    """The whole stack of a StackLayout (prism_stack_create / prism_stack_forward).

    blob: numpy fp16/uint16 array (host) or a CUDA fp16 tensor (device)."""

    def __init__(self, ctx: Prism, L: StackLayout, blob, max_frames: int):
        self.ctx, self.lib, self.layout, self.max_frames = ctx, ctx.lib, L, max_frames
        self._desc, self._keep = abi.stack_desc(L)
        h = C.c_void_p()
        if hasattr(blob, "data_ptr"):
            ptr, n, on_host = blob.data_ptr(), blob.numel(), 0
        else:
            ptr, n, on_host = blob.ctypes.data, blob.size, 1
        check(self.lib, self.lib.prism_stack_create(ctx.h, C.byref(self._desc), ptr, n, on_host, max_frames,
                                                    C.byref(h)))
        self.h = h

    def forward(self, x, out, assign=None, stream=None):
        """x: CUDA fp16 [F, T, in_dim]; out: CUDA fp16 [F, T, out_dim];
        assign: optional CUDA int32 [n_moe_blocks, F*T]."""
        F = x.shape[0]
        check(self.lib, self.lib.prism_stack_forward(self.h, _ptr(x), _ptr(out), F,
                                                     _ptr(assign) if assign is not None else None,
                                                     _stream(stream)))
        return out

    def moe_block(self, x, out, assign=None, counts=None, stream=None):
        """prism_moe_block (a stack of one MoE block, no adapters): x / out CUDA fp16
        [F, T, dim] (views into a feature arena work), assign CUDA int32 [F*T] and counts
        CUDA int32 [n_experts], both optional."""
        check(self.lib, self.lib.prism_moe_block(self.h, _ptr(x), _ptr(out), x.shape[0],
                                                 _ptr(assign) if assign is not None else None,
                                                 _ptr(counts) if counts is not None else None,
                                                 _stream(stream)))
        return out

    def infer(self, host_in, host_out=None) -> float:
        """prism_stack_infer: host_in [F, T, in_dim] / host_out [F, T, out_dim] fp16 host
        arrays (CPU tensors, page-locked for DMA, or numpy arrays); synchronous.  Returns
        the forward's device time in ms."""
        ms = C.c_float()
        check(self.lib, self.lib.prism_stack_infer(self.h, _host_ptr(host_in), _host_ptr(host_out),
                                                   host_in.shape[0], C.byref(ms)))
        return ms.value

    def infer_gpu(self, in_buf, out_buf, frames: int, in_offset: int = 0, out_offset: int = 0) -> float:
        """prism_stack_infer_gpu (the reference's InferGPU): in_buf / out_buf are CUDA tensors
        (any dtype) holding [frames, T, in_dim] / [frames, T, out_dim] fp16 at the given BYTE
        offsets; synchronous.  Returns the forward's device time in ms."""
        ms = C.c_float()
        check(self.lib, self.lib.prism_stack_infer_gpu(self.h, in_buf.data_ptr(), in_offset, out_buf.data_ptr(),
                                                       out_offset, frames, C.byref(ms)))
        return ms.value

    def submit(self, host_in, host_out=None, stream=None) -> int:
        """prism_stack_submit: enqueue upload, forward and download; returns the ticket."""
        t = C.c_int64()
        check(self.lib, self.lib.prism_stack_submit(self.h, _host_ptr(host_in), _host_ptr(host_out),
                                                    host_in.shape[0], _stream(stream), C.byref(t)))
        return t.value

    def wait(self, ticket: int, stream=None, host: bool = True):
        """prism_stack_wait: block the host (default) or make `stream` wait on the device."""
        check(self.lib, self.lib.prism_stack_wait(self.h, ticket, None if host else _stream(stream)))

    def status(self, stream=None):
        check(self.lib, self.lib.prism_stack_status(self.h, _stream(stream)))

    def inject_stall(self, stream=None):
        """Diagnostic (prism_stack_inject_stall): a device wait that nothing releases; the
        next status() raises PRISM_E_TIMEOUT after the library's wait limit."""
        check(self.lib, self.lib.prism_stack_inject_stall(self.h, _stream(stream)))

    def set_pair_attention(self, enable: bool):
        """PRISM_OPT_PAIR_ATTENTION: few-tile dim-256 attention on CTA pairs (default on)."""
        check(self.lib, self.lib.prism_stack_set_option(self.h, abi.OPT_PAIR_ATTENTION, int(enable)))

    def set_bucket_routing(self, enable: bool):
        """PRISM_OPT_BUCKET_ROUTING: router-filled expert buckets, no route kernel (default on)."""
        check(self.lib, self.lib.prism_stack_set_option(self.h, abi.OPT_BUCKET_ROUTING, int(enable)))

    def profile(self, enable: bool = True):
        check(self.lib, self.lib.prism_stack_profile(self.h, int(enable)))

    def profile_read(self):
        """{kernel kind: (total ms, launches)} since the last read (synchronises)."""
        n = len(abi.KERNEL_KINDS)
        ms, cnt = (C.c_double * n)(), (C.c_int64 * n)()
        check(self.lib, self.lib.prism_stack_profile_read(self.h, ms, cnt, n))
        return {k: (ms[i], cnt[i]) for i, k in enumerate(abi.KERNEL_KINDS) if cnt[i]}

    def launch_count(self, frames: int) -> int:
        return self.lib.prism_stack_launch_count(self.h, frames)

    def close(self):
        if self.h:
            self.lib.prism_stack_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
