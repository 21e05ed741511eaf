"""Host-side mirror of ZigNeuron's ``Backend`` operator API for the GEMM path.

``Backend`` keeps the reference method names, argument order and meaning
(src/backend.zig:169-325, 367-399, 649-671): host ``float32`` arrays play the
role of Zig ``[]f32`` slices and outputs are written in place.  Every method
runs on the MI355X through the C ABI (include/zn_hip.h); errors surface as
``ZnError`` subclasses, the analogue of the reference's Zig error unions.

``Context``/``DeviceBuffer`` expose the device-pointer entry points
(``sgemm``, ``sgemm_strided_batched`` and the Dense helpers) for callers that
keep tensors resident in HBM.
"""
from __future__ import annotations

import ctypes
import weakref
from typing import Optional

import numpy as np

from . import _lib
from ._lib import (ACT_LINEAR, ACT_RELU, ACT_SIGMOID, ACT_TANH, LAYOUT_NN, LAYOUT_NT, LAYOUT_TN,
                   InvalidArgumentError, check)

ACTIVATIONS = {"linear": ACT_LINEAR, "relu": ACT_RELU, "sigmoid": ACT_SIGMOID, "tanh": ACT_TANH}
LAYOUTS = {"nn": LAYOUT_NN, "nt": LAYOUT_NT, "tn": LAYOUT_TN}


def act_id(act) -> int:
    """Map an activation name (src/activation.zig:14-22) to its C-ABI id."""
    if isinstance(act, int):
        return act
    try:
        return ACTIVATIONS[str(act)]
    except KeyError:
        raise InvalidArgumentError(_lib.ZN_ERR_INVALID_ARG, "activation",
                                   f"{act!r} is not on the GEMM path (linear, relu, sigmoid, tanh)") from None


def gate_id(act) -> int:
    """Map a gate activation's name to its C-ABI id (zn_gate)."""
    if isinstance(act, int):
        return act
    try:
        return _lib.GATES[str(act)]
    except KeyError:
        raise InvalidArgumentError(_lib.ZN_ERR_INVALID_ARG, "gate",
                                   f"{act!r} is not a gate ({', '.join(_lib.GATES)})") from None


def layout_id(layout) -> int:
    if isinstance(layout, int):
        return layout
    return LAYOUTS[str(layout).lower()]


def available() -> bool:
    """zn_hip_available(): a HIP device is visible."""
    return bool(_lib.load().zn_hip_available())


def _f32_in(x) -> np.ndarray:
    return np.ascontiguousarray(x, dtype=np.float32)


def _f32_out(x) -> np.ndarray:
    if not (isinstance(x, np.ndarray) and x.dtype == np.float32 and x.flags.c_contiguous and x.flags.writeable):
        raise InvalidArgumentError(_lib.ZN_ERR_INVALID_ARG, "output",
                                   "outputs must be writable contiguous float32 arrays")
    return x


def _ptr(x: np.ndarray) -> int:
    return x.ctypes.data


class Graph:
    """A captured sequence of device calls, replayed with one launch (zn_hip_graph_*)."""

    def __init__(self, ctx: "Context", handle: ctypes.c_void_p):
        self._ctx, self.handle = ctx, handle
        ctx._graphs.add(self)

    def launch(self) -> None:
        if not self.handle or not self._ctx.handle:
            raise InvalidArgumentError(_lib.ZN_ERR_INVALID_ARG, "zn_hip_graph_launch", "graph or context closed")
        check(_lib.load().zn_hip_graph_launch(self._ctx.handle, self.handle), "zn_hip_graph_launch")

    def close(self) -> None:
        """Release the graph (a no-op once it or its context is closed: the
        context's destruction releases its graphs)."""
        if self.handle and self._ctx.handle:
            _lib.load().zn_hip_graph_destroy(self.handle)
        self.handle = None

    def __del__(self):  # pragma: no cover - interpreter shutdown order
        try:
            self.close()
        except Exception:
            pass


class Event:
    def __init__(self, ctx: "Context"):
        self._ctx = ctx
        h = ctypes.c_void_p()
        check(_lib.load().zn_hip_event_create(ctx.handle, ctypes.byref(h)), "zn_hip_event_create")
        self.handle = h

    def record(self) -> None:
        check(_lib.load().zn_hip_event_record(self._ctx.handle, self.handle), "zn_hip_event_record")

    def elapsed_ms(self, end: "Event") -> float:
        ms = ctypes.c_float()
        check(_lib.load().zn_hip_event_elapsed_ms(self.handle, end.handle, ctypes.byref(ms)),
              "zn_hip_event_elapsed_ms")
        return float(ms.value)

    def close(self) -> None:
        if self.handle:
            _lib.load().zn_hip_event_destroy(self.handle)
            self.handle = None

    def __del__(self):  # pragma: no cover - interpreter shutdown order
        try:
            self.close()
        except Exception:
            pass


def _name_id(table, name, what: str) -> int:
    if name in table:
        return table[name]
    if isinstance(name, int):
        return name
    raise InvalidArgumentError(_lib.ZN_ERR_INVALID_ARG, what, f"{name!r} is not one of {', '.join(table)}")


def rotary_frequencies(rot_dim: int, base: float = 10000.0, scaling="plain", factor: float = 1.0, trained_len: int = 0,
                       low: float = 1.0, high: float = 32.0) -> np.ndarray:
    """The frequencies of rot_dim / 2 rotary pairs (host array), scaled for contexts `factor` times trained_len:
    "plain", "linear", "base", "turns" or "pairs" (zn_rotary_scaling)."""
    freq = np.empty(max(int(rot_dim), 0) // 2, np.float32)
    check(_lib.load().zn_hip_rotary_frequencies(_ptr(freq), freq.size, rot_dim, float(base),
                                                _name_id(_lib.ROTARY_SCALINGS, scaling, "rotary scaling"), float(factor),
                                                int(trained_len), float(low), float(high)), "zn_hip_rotary_frequencies")
    return freq


class PagedCache:
    """Pools of key and value pages ([num_pages, kv_heads, page_size, head_dim] at (page, head, position) element
    strides, None: contiguous) with the page table ([batch x max_pages] int32) and lengths ([batch] int32) of the
    sequences in them, all on the device and the caller's; dtype is "f32" or "bf16"."""

    def __init__(self, k, v, page_table, kv_lens, batch, num_pages, page_size, max_pages, kv_heads, head_dim, dtype="f32",
                 strides=None):
        if strides is None:
            strides = (kv_heads * page_size * head_dim, page_size * head_dim, head_dim)
        self.desc = _lib.PagedCacheDesc(_dptr(k), _dptr(v), _dptr(page_table), _dptr(kv_lens), batch, num_pages, page_size, max_pages,
                                        kv_heads, head_dim, *strides, _name_id(_lib.CACHE_TYPES, dtype, "cache type"))
        self.address = ctypes.addressof(self.desc)
        self.buffers = (k, v, page_table, kv_lens)  # held as long as the descriptor


class DeviceBuffer:
    """A caller-owned float32 buffer in HBM (zn_hip_alloc / zn_hip_free)."""

    def __init__(self, ctx: "Context", count: int):
        self.ctx = ctx
        self.count = int(count)
        h = ctypes.c_void_p()
        check(_lib.load().zn_hip_alloc(ctx.handle, max(self.count, 1) * 4, ctypes.byref(h)), "zn_hip_alloc")
        self.ptr = int(h.value)

    def upload(self, host) -> "DeviceBuffer":
        h = _f32_in(host)
        if h.size > self.count:
            raise InvalidArgumentError(_lib.ZN_ERR_INVALID_ARG, "upload", "host array larger than buffer")
        check(_lib.load().zn_hip_h2d(self.ctx.handle, self.ptr, _ptr(h), h.size * 4), "zn_hip_h2d")
        return self

    def download(self, count: Optional[int] = None) -> np.ndarray:
        n = self.count if count is None else int(count)
        out = np.empty(n, np.float32)
        check(_lib.load().zn_hip_d2h(self.ctx.handle, _ptr(out), self.ptr, n * 4), "zn_hip_d2h")
        return out

    def fill(self, value: float) -> "DeviceBuffer":
        check(_lib.load().zn_hip_fill_f32(self.ctx.handle, self.ptr, float(value), self.count), "zn_hip_fill_f32")
        return self

    def offset(self, elements: int) -> int:
        return self.ptr + 4 * int(elements)

    def close(self) -> None:
        """Free the buffer; after its context is closed this only drops the pointer."""
        if self.ptr and self.ctx.handle:
            check(_lib.load().zn_hip_free(self.ctx.handle, self.ptr), "zn_hip_free")
        self.ptr = 0

    def __del__(self):  # pragma: no cover
        try:
            if self.ptr and self.ctx.handle:
                self.close()
        except Exception:
            pass


class Context:
    """One device, one stream, the loaded gfx950 code objects (zn_hip_create)."""

    def __init__(self, device: int = 0, code_object_dir: Optional[str] = None):
        h = ctypes.c_void_p()
        d = code_object_dir.encode() if code_object_dir else None
        check(_lib.load().zn_hip_create(int(device), d, ctypes.byref(h)), "zn_hip_create")
        self.handle = h.value
        self._graphs = weakref.WeakSet()
        info = _lib.DeviceInfo()
        check(_lib.load().zn_hip_device_info(self.handle, ctypes.byref(info)), "zn_hip_device_info")
        self.arch = info.name.decode()
        self.compute_units = int(info.compute_units)
        self.clock_khz = int(info.clock_khz)
        self.total_mem = int(info.total_mem)

    # --- memory / sync
    def alloc(self, count: int) -> DeviceBuffer:
        return DeviceBuffer(self, count)

    def to_device(self, host) -> DeviceBuffer:
        h = _f32_in(host)
        return DeviceBuffer(self, h.size).upload(h)

    def sync(self) -> None:
        check(_lib.load().zn_hip_sync(self.handle), "zn_hip_sync")

    def event(self) -> Event:
        return Event(self)

    def capture(self, fn) -> Graph:
        """Run fn() under stream capture and return the graph of its device calls.
        Run fn() once eagerly first (it sizes the split-K workspace)."""
        L = _lib.load()
        check(L.zn_hip_graph_begin(self.handle), "zn_hip_graph_begin")
        h = ctypes.c_void_p()
        try:
            fn()
        except BaseException:
            if L.zn_hip_graph_end(self.handle, ctypes.byref(h)) == _lib.ZN_OK and h:
                L.zn_hip_graph_destroy(h)
            raise
        check(L.zn_hip_graph_end(self.handle, ctypes.byref(h)), "zn_hip_graph_end")
        return Graph(self, h)

    def hold_stream(self, microseconds: float) -> None:
        """Keep the context stream busy for `microseconds` (a timing aid: launches queued behind it run back
        to back on the device)."""
        check(_lib.load().zn_hip_hold_stream(self.handle, float(microseconds)), "zn_hip_hold_stream")

    def copy(self, dst: int, src: int, count: int) -> None:
        check(_lib.load().zn_hip_copy_f32(self.handle, int(dst), int(src), int(count)), "zn_hip_copy_f32")

    def set_gemm_tile(self, tile="auto") -> None:
        """Force one macro tile ("256x128", "128x128", "128x64", "64x64", "32x32", "128x128k32", "64x64k16",
        "256x256"; split operands on the bf16 matrix cores: "256x256s", "256x128s", "128x128s", "128x64s", "128x128sc" and,
        for convolutions, "conv128x128s", "conv64x128s") or "auto"."""
        check(_lib.load().zn_hip_set_gemm_tile(self.handle, _lib.TILES[tile] if isinstance(tile, str) else tile),
              "zn_hip_set_gemm_tile")

    def set_gemm_splits(self, splits: int = 0) -> None:
        """Force the number of split-K slices (1..256), or 0 for the policy."""
        check(_lib.load().zn_hip_set_gemm_splits(self.handle, int(splits)), "zn_hip_set_gemm_splits")

    def set_gemm_wave_split(self, waves: int = -1) -> None:
        """-1: the policy decides; 0: never; 4 or 8: every eligible GEMM splits K over that many waves of a workgroup."""
        check(_lib.load().zn_hip_set_gemm_wave_split(self.handle, int(waves)), "zn_hip_set_gemm_wave_split")

    def set_gemm_persistent(self, mode: int = -1) -> None:
        """-1: the policy decides; 0: never; 1: every eligible GEMM runs on the persistent kernels;
        2: the same, with deferred stores wherever they apply (bit-identical in every mode)."""
        check(_lib.load().zn_hip_set_gemm_persistent(self.handle, int(mode)), "zn_hip_set_gemm_persistent")

    # --- GEMM on device pointers (asynchronous on the context stream)
    def sgemm(self, layout, m, n, k, a, lda, b, ldb, c, ldc, accumulate=False, bias=None, act="linear") -> None:
        check(_lib.load().zn_hip_sgemm(self.handle, layout_id(layout), m, n, k, _dptr(a), lda, _dptr(b), ldb,
                                       _dptr(c), ldc, int(bool(accumulate)), _dptr(bias), act_id(act)),
              "zn_hip_sgemm")

    def sgemm_strided_batched(self, layout, m, n, k, a, lda, stride_a, b, ldb, stride_b, c, ldc, stride_c,
                              batch, accumulate=False, bias=None, act="linear") -> None:
        check(_lib.load().zn_hip_sgemm_strided_batched(
            self.handle, layout_id(layout), m, n, k, _dptr(a), lda, stride_a, _dptr(b), ldb, stride_b,
            _dptr(c), ldc, stride_c, batch, int(bool(accumulate)), _dptr(bias), act_id(act)),
            "zn_hip_sgemm_strided_batched")

    # --- Dense helpers on device pointers
    def add_bias(self, out, bias, rows, n) -> None:
        check(_lib.load().zn_hip_add_bias(self.handle, _dptr(out), _dptr(bias), rows, n), "zn_hip_add_bias")

    def activation_forward(self, act, inp, out, length) -> None:
        check(_lib.load().zn_hip_activation_forward(self.handle, act_id(act), _dptr(inp), _dptr(out), length),
              "zn_hip_activation_forward")

    def activation_backward(self, act, y, grad_out, grad_in, length) -> None:
        check(_lib.load().zn_hip_activation_backward(self.handle, act_id(act), _dptr(y), _dptr(grad_out),
                                                     _dptr(grad_in), length), "zn_hip_activation_backward")

    def accumulate_bias(self, grad_bias, gaa, rows, n) -> None:
        check(_lib.load().zn_hip_accumulate_bias(self.handle, _dptr(grad_bias), _dptr(gaa), rows, n),
              "zn_hip_accumulate_bias")

    def dense_backward(self, act, inp, weights, activated_output, grad_output, grad_after_act, grad_input,
                       grad_weights, grad_bias, batch, in_size, out_size) -> None:
        """Dense.backward in one call: fused activationBackward + bias-gradient pass, NT, TN
        (grad_input may be None)."""
        check(_lib.load().zn_hip_dense_backward(
            self.handle, act_id(act), _dptr(inp), _dptr(weights), _dptr(activated_output), _dptr(grad_output),
            _dptr(grad_after_act), _dptr(grad_input), _dptr(grad_weights), _dptr(grad_bias), batch, in_size, out_size),
            "zn_hip_dense_backward")

    def dense_backward_chain(self, act, inp, weights, activated_output, grad_output, grad_after_act, grad_input,
                             grad_weights, grad_bias, batch, in_size, out_size, gaa_ready=False, prev_act="linear",
                             prev_activated_output=None, prev_grad_after_act=None) -> None:
        """dense_backward for layers walked top-down: gaa_ready means grad_after_act already holds
        this layer's derivative (written by the layer above's call); prev_grad_after_act (with
        prev_act and prev_activated_output) receives the layer below's derivative from grad_input.
        Bit-identical to dense_backward layer by layer."""
        check(_lib.load().zn_hip_dense_backward_chain(
            self.handle, act_id(act), _dptr(inp), _dptr(weights), _dptr(activated_output), _dptr(grad_output),
            _dptr(grad_after_act), _dptr(grad_input), _dptr(grad_weights), _dptr(grad_bias), batch, in_size, out_size,
            int(bool(gaa_ready)), act_id(prev_act), _dptr(prev_activated_output), _dptr(prev_grad_after_act)),
            "zn_hip_dense_backward_chain")

    def dense_pair_forward(self, act1, x, w1, b1, h, act2, w2, b2, y, batch, in_size, hidden, out_size) -> None:
        """Two stacked Dense forwards, h = act1(x.W1 + b1) then y = act2(h.W2 + b2): one launch
        when the top layer has at most 16 outputs and the lower one is small."""
        check(_lib.load().zn_hip_dense_pair_forward(
            self.handle, act_id(act1), _dptr(x), _dptr(w1), _dptr(b1), _dptr(h), act_id(act2), _dptr(w2), _dptr(b2),
            _dptr(y), batch, in_size, hidden, out_size), "zn_hip_dense_pair_forward")

    def dense_pair_backward(self, act1, x, w1, h, gaa1, grad_x, grad_w1, grad_b1, act2, w2, y, grad_y, gaa2,
                            grad_h, grad_w2, grad_b2, batch, in_size, hidden, out_size) -> None:
        """The backward of the same pair (top layer first), in one launch under the same limits."""
        check(_lib.load().zn_hip_dense_pair_backward(
            self.handle, act_id(act1), _dptr(x), _dptr(w1), _dptr(h), _dptr(gaa1), _dptr(grad_x), _dptr(grad_w1),
            _dptr(grad_b1), act_id(act2), _dptr(w2), _dptr(y), _dptr(grad_y), _dptr(gaa2), _dptr(grad_h),
            _dptr(grad_w2), _dptr(grad_b2), batch, in_size, hidden, out_size), "zn_hip_dense_pair_backward")

    # --- convolution and attention on device pointers
    def im2col(self, inp, col, batch, channels, in_h, in_w, k_h, k_w, out_h, out_w, stride_h=1, stride_w=1,
               pad_h=0, pad_w=0) -> None:
        check(_lib.load().zn_hip_im2col(self.handle, _dptr(inp), _dptr(col), batch, channels, in_h, in_w, k_h, k_w,
                                        out_h, out_w, stride_h, stride_w, pad_h, pad_w), "zn_hip_im2col")

    def conv2d_forward_im2col(self, inp, weights, bias, out, batch, in_channels, out_channels, k_h, k_w, in_h,
                              in_w, out_h, out_w, stride_h=1, stride_w=1, pad_h=0, pad_w=0) -> None:
        check(_lib.load().zn_hip_conv2d_forward_im2col(
            self.handle, _dptr(inp), _dptr(weights), _dptr(bias), _dptr(out), batch, in_channels, out_channels, k_h,
            k_w, in_h, in_w, out_h, out_w, stride_h, stride_w, pad_h, pad_w), "zn_hip_conv2d_forward_im2col")

    def conv2d_forward_direct(self, inp, weights, bias, out, batch, in_channels, out_channels, k_h, k_w, in_h,
                              in_w, out_h, out_w, stride_h=1, stride_w=1, pad_h=0, pad_w=0) -> None:
        """Implicit-GEMM convolution with W as [OC][C][kH][kW] (true NCHW convolution)."""
        check(_lib.load().zn_hip_conv2d_forward_direct(
            self.handle, _dptr(inp), _dptr(weights), _dptr(bias), _dptr(out), batch, in_channels, out_channels, k_h,
            k_w, in_h, in_w, out_h, out_w, stride_h, stride_w, pad_h, pad_w), "zn_hip_conv2d_forward_direct")

    def col2im(self, col, out, batch, channels, in_h, in_w, k_h, k_w, out_h, out_w, stride_h=1, stride_w=1,
               pad_h=0, pad_w=0) -> None:
        """Backend.col2im on device (bit-identical to the reference); `out` is overwritten."""
        check(_lib.load().zn_hip_col2im(self.handle, _dptr(col), _dptr(out), batch, channels, in_h, in_w, k_h, k_w,
                                        out_h, out_w, stride_h, stride_w, pad_h, pad_w), "zn_hip_col2im")

    def conv2d_backward_im2col(self, inp, weights, grad_output, grad_input, grad_weights, grad_bias, batch,
                               in_channels, out_channels, k_h, k_w, in_h, in_w, out_h, out_w, stride_h=1, stride_w=1,
                               pad_h=0, pad_w=0) -> None:
        """cpuConv2dBackwardIm2col on device (grad_output read as [batch*OH*OW][OC] by the GEMMs)."""
        check(_lib.load().zn_hip_conv2d_backward_im2col(
            self.handle, _dptr(inp), _dptr(weights), _dptr(grad_output), _dptr(grad_input), _dptr(grad_weights),
            _dptr(grad_bias), batch, in_channels, out_channels, k_h, k_w, in_h, in_w, out_h, out_w, stride_h, stride_w,
            pad_h, pad_w), "zn_hip_conv2d_backward_im2col")

    def conv2d_backward_direct(self, inp, weights, grad_output, grad_input, grad_weights, grad_bias, batch,
                               in_channels, out_channels, k_h, k_w, in_h, in_w, out_h, out_w, stride_h=1, stride_w=1,
                               pad_h=0, pad_w=0) -> None:
        """The direct branch of cpuConv2dBackward on device (NCHW, OIHW)."""
        check(_lib.load().zn_hip_conv2d_backward_direct(
            self.handle, _dptr(inp), _dptr(weights), _dptr(grad_output), _dptr(grad_input), _dptr(grad_weights),
            _dptr(grad_bias), batch, in_channels, out_channels, k_h, k_w, in_h, in_w, out_h, out_w, stride_h, stride_w,
            pad_h, pad_w), "zn_hip_conv2d_backward_direct")

    def softmax_rows(self, inp, out, rows, n, scale=1.0) -> None:
        check(_lib.load().zn_hip_softmax_rows(self.handle, _dptr(inp), _dptr(out), rows, n, float(scale)),
              "zn_hip_softmax_rows")

    def attention_forward(self, q, k, v, out, batch, seq_len, d_k, scale) -> None:
        check(_lib.load().zn_hip_attention_forward(self.handle, _dptr(q), _dptr(k), _dptr(v), _dptr(out), batch,
                                                   seq_len, d_k, float(scale)), "zn_hip_attention_forward")

    # --- language-model blocks on device pointers
    def mha_forward(self, q, k, v, out, lse, batch, q_heads, kv_heads, q_len, kv_len, head_dim, scale, causal=False,
                    q_lens=None, kv_lens=None, q_strides=None, kv_strides=None, out_strides=None) -> None:
        """Multi-head attention with shared key/value heads, causal and length masks.  Tensors are
        [batch, heads, positions, head_dim] at (batch, head, position) element strides (None: contiguous);
        lse ([batch, q_heads, q_len]) is what the backward reads and may be None; q_lens and kv_lens are
        int32 device arrays of the sequences' lengths."""
        check(_lib.load().zn_hip_mha_forward(
            self.handle, _dptr(q), _dptr(k), _dptr(v), _dptr(out), _dptr(lse), batch, q_heads, kv_heads, q_len, kv_len,
            head_dim, float(scale), int(causal), _dptr(q_lens), _dptr(kv_lens),
            *_mha_strides(q_heads, kv_heads, q_len, kv_len, head_dim, q_strides, kv_strides, out_strides)),
            "zn_hip_mha_forward")

    def mha_backward(self, q, k, v, out, lse, grad_out, grad_q, grad_k, grad_v, batch, q_heads, kv_heads, q_len, kv_len,
                     head_dim, scale, causal=False, q_lens=None, kv_lens=None, q_strides=None, kv_strides=None,
                     out_strides=None) -> None:
        """The gradients of mha_forward from its out and lse; grad_q is laid out like q, grad_k and grad_v like
        k, grad_out like out.  The probabilities are computed again."""
        check(_lib.load().zn_hip_mha_backward(
            self.handle, _dptr(q), _dptr(k), _dptr(v), _dptr(out), _dptr(lse), _dptr(grad_out), _dptr(grad_q),
            _dptr(grad_k), _dptr(grad_v), batch, q_heads, kv_heads, q_len, kv_len, head_dim, float(scale), int(causal),
            _dptr(q_lens), _dptr(kv_lens),
            *_mha_strides(q_heads, kv_heads, q_len, kv_len, head_dim, q_strides, kv_strides, out_strides)),
            "zn_hip_mha_backward")

    def gated_dense_forward(self, act, x, w, bias, z, h, batch, in_size, hidden) -> None:
        """h = act(gate) * up with [gate | up] = x.W + bias, W [in_size x 2 hidden] (bias may be None); z
        ([batch x 2 hidden], the projections) is what the backward reads and may be None."""
        check(_lib.load().zn_hip_gated_dense_forward(self.handle, gate_id(act), _dptr(x), _dptr(w), _dptr(bias), _dptr(z),
                                                     _dptr(h), batch, in_size, hidden), "zn_hip_gated_dense_forward")

    def gated_dense_backward(self, act, x, w, z, grad_h, grad_z, grad_x, grad_w, grad_bias, batch, in_size,
                             hidden) -> None:
        """The gradients of gated_dense_forward; grad_bias accumulates, grad_bias and grad_x may be None."""
        check(_lib.load().zn_hip_gated_dense_backward(
            self.handle, gate_id(act), _dptr(x), _dptr(w), _dptr(z), _dptr(grad_h), _dptr(grad_z), _dptr(grad_x),
            _dptr(grad_w), _dptr(grad_bias), batch, in_size, hidden), "zn_hip_gated_dense_backward")

    def distill_forward(self, logits, ld, top_index, top_logits, loss, lse, rows, vocab, k, temperature=1.0) -> None:
        """Per row, the divergence of the teacher's top logits ([rows x k] int32 indices and float32 logits) from
        the student's distribution over the vocabulary, and the log-sum-exp that the backward reads."""
        check(_lib.load().zn_hip_distill_forward(self.handle, _dptr(logits), ld, _dptr(top_index), _dptr(top_logits),
                                                 _dptr(loss), _dptr(lse), rows, vocab, k, float(temperature)),
              "zn_hip_distill_forward")

    def distill_backward(self, logits, ld, top_index, top_logits, lse, grad_loss, grad_logits, grad_ld, rows, vocab, k,
                         temperature=1.0) -> None:
        """The gradient of distill_forward's losses, weighted by grad_loss ([rows]); grad_logits may be logits."""
        check(_lib.load().zn_hip_distill_backward(
            self.handle, _dptr(logits), ld, _dptr(top_index), _dptr(top_logits), _dptr(lse), _dptr(grad_loss),
            _dptr(grad_logits), grad_ld, rows, vocab, k, float(temperature)), "zn_hip_distill_backward")

    def rotary_forward(self, x, y, freq, batch, heads, length, head_dim, rot_dim, layout="half", positions=None,
                       position_stride=None, scale=1.0, x_strides=None, y_strides=None) -> None:
        """Rotary positions: the first rot_dim dims of each head of x ([batch, heads, length, head_dim] at (batch, head,
        position) element strides, None: contiguous) turned by the token's position times the pair's frequency; y may be
        x.  positions: int32 device array, length of them a sequence, position_stride apart (None: length); None: 0, 1, .."""
        _rotary(_lib.load().zn_hip_rotary_forward, self.handle, x, y, freq, batch, heads, length, head_dim, rot_dim, layout, positions,
                position_stride, scale, x_strides, y_strides)

    def rotary_backward(self, grad_y, grad_x, freq, batch, heads, length, head_dim, rot_dim, layout="half", positions=None,
                        position_stride=None, scale=1.0, y_strides=None, x_strides=None) -> None:
        """The gradient of rotary_forward: grad_y turned back to grad_x, which may be grad_y."""
        _rotary(_lib.load().zn_hip_rotary_backward, self.handle, grad_y, grad_x, freq, batch, heads, length, head_dim, rot_dim, layout,
                positions, position_stride, scale, y_strides, x_strides)

    def paged_append(self, cache: PagedCache, token_starts, tokens, k, v, kv_strides=None, q=None, q_out=None, q_heads=0,
                     q_strides=None, q_out_strides=None, freq=None, rot_dim=0, layout="half", scale=1.0, positions=None) -> None:
        """The keys and values of new tokens ([tokens, kv_heads, head_dim] at (token, head) element strides, None:
        contiguous) into their sequences' pages, keys and queries (q to q_out, which may be q) turned on the way.
        Sequence b's are rows token_starts[b] .. token_starts[b + 1] - 1 and its last positions."""
        d = cache.desc
        kt, kh = (d.kv_heads * d.head_dim, d.head_dim) if kv_strides is None else kv_strides
        qt, qh = (q_heads * d.head_dim, d.head_dim) if q_strides is None else q_strides
        ot, oh = (q_heads * d.head_dim, d.head_dim) if q_out_strides is None else q_out_strides
        check(_lib.load().zn_hip_paged_append(
            self.handle, cache.address, _dptr(token_starts), tokens, _dptr(k), _dptr(v), kt, kh, _dptr(q), _dptr(q_out), q_heads, qt, qh,
            ot, oh, _dptr(freq), rot_dim, _name_id(_lib.ROTARY_LAYOUTS, layout, "rotary layout"), scale, _dptr(positions)),
            "zn_hip_paged_append")

    def paged_attention(self, cache: PagedCache, token_starts, tokens, max_q_len, max_kv_len, q, out, lse, q_heads, scale,
                        causal=True, q_strides=None, out_strides=None) -> None:
        """Attention of the sequences' new tokens (rows as in paged_append; at most max_q_len of each) over the positions
        (at most max_kv_len) that their pages hold; q and out are [tokens, q_heads, head_dim] at (token, head) element
        strides (None: contiguous), lse [tokens x q_heads] or None."""
        d = cache.desc
        qt, qh = (q_heads * d.head_dim, d.head_dim) if q_strides is None else q_strides
        ot, oh = (q_heads * d.head_dim, d.head_dim) if out_strides is None else out_strides
        check(_lib.load().zn_hip_paged_attention(
            self.handle, cache.address, _dptr(token_starts), tokens, max_q_len, max_kv_len, _dptr(q), _dptr(out), _dptr(lse), q_heads,
            scale, int(causal), qt, qh, ot, oh), "zn_hip_paged_attention")

    def close(self) -> None:
        if self.handle:
            for g in list(self._graphs):  # zn_hip_destroy releases them
                g.handle = None
            _lib.load().zn_hip_destroy(self.handle)
            self.handle = None

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def __del__(self):  # pragma: no cover
        try:
            self.close()
        except Exception:
            pass


def _mha_strides(q_heads, kv_heads, q_len, kv_len, head_dim, q, kv, out):
    """The nine element strides of an mha call, contiguous [batch, heads, positions, dims] where not given."""
    q_own = (q_heads * q_len * head_dim, q_len * head_dim, head_dim)
    kv_own = (kv_heads * kv_len * head_dim, kv_len * head_dim, head_dim)
    return (*(q_own if q is None else q), *(kv_own if kv is None else kv), *(q_own if out is None else out))


def _rotary(call, handle, src, dst, freq, batch, heads, length, head_dim, rot_dim, layout, positions, position_stride, scale,
            src_strides, dst_strides) -> None:
    """Either direction's call; strides not given are contiguous [batch, heads, positions, dims]."""
    own = (heads * length * head_dim, length * head_dim, head_dim)
    sb, sh, ss = own if src_strides is None else src_strides
    db, dh, ds = own if dst_strides is None else dst_strides
    check(call(handle, _dptr(src), _dptr(dst), _dptr(freq), _dptr(positions), batch, heads, length, head_dim, rot_dim,
               _name_id(_lib.ROTARY_LAYOUTS, layout, "rotary layout"), scale, length if position_stride is None else position_stride,
               sb, sh, ss, db, dh, ds), call.__name__)


def _dptr(x) -> Optional[int]:
    if x is None or type(x) is int:
        return x
    if isinstance(x, DeviceBuffer):
        return x.ptr
    return int(x)


class Backend:
    """ZigNeuron ``Backend`` (src/backend.zig:15-325) with the HIP arm.

    Methods take host float32 arrays (the Zig slices) and write outputs in
    place; they return when the result is in host memory, like the
    reference's synchronous CUDA arms (src/cuda.zig:617).
    """

    def __init__(self, ctx: Context):
        self.ctx = ctx

    @classmethod
    def init(cls, device: int = 0) -> "Backend":
        """Backend.init + detect (src/backend.zig:43-94) with the HIP arm: raises
        NoDeviceError when no gfx950 device is present (no CPU fallback here)."""
        return cls(Context(device))

    def deinit(self) -> None:
        self.ctx.close()

    @property
    def _h(self):
        return self.ctx.handle

    # --- GEMM family
    def _gemm(self, fn, a, b, c, m, n, k, accumulate):
        a, b, c = _f32_in(a), _f32_in(b), _f32_out(c)
        check(fn(self._h, _ptr(a), a.size, _ptr(b), b.size, _ptr(c), c.size, m, n, k, int(bool(accumulate))),
              fn.__name__)

    def matMul(self, a, b, c, m, n, k, accumulate=False):
        """Backend.matMul (src/backend.zig:169-182): C (+)= A[m x k] . B[k x n]."""
        self._gemm(_lib.load().zn_hip_mat_mul, a, b, c, m, n, k, accumulate)

    def matMulBatch(self, a, b, c, batch_size, n, k, accumulate=False):
        """Backend.matMulBatch (src/backend.zig:186-195)."""
        self._gemm(_lib.load().zn_hip_mat_mul_batch, a, b, c, batch_size, n, k, accumulate)

    def matMulTransposeA(self, a, b, c, m, n, k, accumulate=False):
        """Backend.matMulTransposeA (src/backend.zig:298-307): C (+)= A^T . B, A is [k x m]."""
        self._gemm(_lib.load().zn_hip_mat_mul_transpose_a, a, b, c, m, n, k, accumulate)

    def matMulTransposeB(self, a, b, c, m, n, k, accumulate=False):
        """Backend.matMulTransposeB (src/backend.zig:310-325): C (+)= A . B^T, B is [n x k]."""
        self._gemm(_lib.load().zn_hip_mat_mul_transpose_b, a, b, c, m, n, k, accumulate)

    def _bias_gemm(self, fn, a, b, bias, c, batch_size, n, k):
        a, b, bias, c = _f32_in(a), _f32_in(b), _f32_in(bias), _f32_out(c)
        check(fn(self._h, _ptr(a), a.size, _ptr(b), b.size, _ptr(bias), bias.size, _ptr(c), c.size,
                 batch_size, n, k), fn.__name__)

    def matMulBias(self, a, b, bias, c, batch_size, n, k):
        """Backend.matMulBias (src/backend.zig:200-222)."""
        self._bias_gemm(_lib.load().zn_hip_mat_mul_bias, a, b, bias, c, batch_size, n, k)

    def matMulBiasRelu(self, a, b, bias, c, batch_size, n, k):
        """Backend.matMulBiasRelu (src/backend.zig:225-247)."""
        self._bias_gemm(_lib.load().zn_hip_mat_mul_bias_relu, a, b, bias, c, batch_size, n, k)

    def matMulBiasSigmoid(self, a, b, bias, c, batch_size, n, k):
        """Backend.matMulBiasSigmoid (src/backend.zig:250-272)."""
        self._bias_gemm(_lib.load().zn_hip_mat_mul_bias_sigmoid, a, b, bias, c, batch_size, n, k)

    def matMulBiasTanh(self, a, b, bias, c, batch_size, n, k):
        """Backend.matMulBiasTanh (src/backend.zig:275-295)."""
        self._bias_gemm(_lib.load().zn_hip_mat_mul_bias_tanh, a, b, bias, c, batch_size, n, k)

    # --- Dense epilogue / backward helpers
    def addBias(self, output, bias):
        """Backend.addBias (src/backend.zig:658-671)."""
        out, bias = _f32_out(output), _f32_in(bias)
        check(_lib.load().zn_hip_add_bias_host(self._h, _ptr(out), out.size, _ptr(bias), bias.size),
              "zn_hip_add_bias_host")

    def activationForward(self, act, inp, output):
        """Backend.activationForward (src/backend.zig:367-386)."""
        inp, out = _f32_in(inp), _f32_out(output)
        check(_lib.load().zn_hip_activation_forward_host(self._h, act_id(act), _ptr(inp), inp.size, _ptr(out),
                                                         out.size), "zn_hip_activation_forward_host")

    def activationBackward(self, act, inp, grad_output, grad_input):
        """Backend.activationBackward (src/backend.zig:390-399); `inp` is the activated output."""
        y, go, gi = _f32_in(inp), _f32_in(grad_output), _f32_out(grad_input)
        check(_lib.load().zn_hip_activation_backward_host(self._h, act_id(act), _ptr(y), y.size, _ptr(go),
                                                          go.size, _ptr(gi), gi.size),
              "zn_hip_activation_backward_host")

    def accumulateBias(self, grad_bias, grad_after_act):
        """Backend.accumulateBias (src/backend.zig:649-655)."""
        gb, gaa = _f32_out(grad_bias), _f32_in(grad_after_act)
        check(_lib.load().zn_hip_accumulate_bias_host(self._h, _ptr(gb), gb.size, _ptr(gaa), gaa.size),
              "zn_hip_accumulate_bias_host")

    # --- convolution and attention
    def conv2dForward(self, inp, weights, bias, output, in_channels, out_channels, kernel_h, kernel_w, input_h,
                      input_w, output_h, output_w, stride_h, stride_w, padding_h, padding_w):
        """Backend.conv2dForward (src/backend.zig:507-518), NCHW, batch = len(input) / (C*H*W)."""
        x, w, b, out = _f32_in(inp), _f32_in(weights), _f32_in(bias), _f32_out(output)
        check(_lib.load().zn_hip_conv2d_forward_host(
            self._h, _ptr(x), x.size, _ptr(w), w.size, _ptr(b), b.size, _ptr(out), out.size, in_channels,
            out_channels, kernel_h, kernel_w, input_h, input_w, output_h, output_w, stride_h, stride_w, padding_h,
            padding_w), "zn_hip_conv2d_forward_host")

    def conv2dBackward(self, inp, weights, grad_output, grad_input, grad_weights, grad_bias, in_channels,
                       out_channels, kernel_h, kernel_w, input_h, input_w, output_h, output_w, stride_h, stride_w,
                       padding_h, padding_w):
        """Backend.conv2dBackward (src/backend.zig:520, :3049-3095), batch = len(input) / (C*H*W)."""
        x, w, go = _f32_in(inp), _f32_in(weights), _f32_in(grad_output)
        gi, gw, gb = _f32_out(grad_input), _f32_out(grad_weights), _f32_out(grad_bias)
        check(_lib.load().zn_hip_conv2d_backward_host(
            self._h, _ptr(x), x.size, _ptr(w), w.size, _ptr(go), go.size, _ptr(gi), gi.size, _ptr(gw), gw.size,
            _ptr(gb), gb.size, in_channels, out_channels, kernel_h, kernel_w, input_h, input_w, output_h, output_w,
            stride_h, stride_w, padding_h, padding_w), "zn_hip_conv2d_backward_host")

    def attentionForward(self, q, k, v, output, scores_buffer, seq_len, d_k, scaling_factor):
        """Backend.attentionForward (src/backend.zig:631-638), one head [seq_len x d_k]."""
        q, k, v, out = _f32_in(q), _f32_in(k), _f32_in(v), _f32_out(output)
        sc = _f32_out(scores_buffer)
        check(_lib.load().zn_hip_attention_forward_host(
            self._h, _ptr(q), q.size, _ptr(k), k.size, _ptr(v), v.size, _ptr(out), out.size, _ptr(sc), sc.size,
            seq_len, d_k, float(scaling_factor)), "zn_hip_attention_forward_host")
