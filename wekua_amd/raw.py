"""Thin numpy helpers over the raw C ABI (device buffers, uploads, the two hot-path calls).

Used by bench.py and by the parity tests that drive `wk_gemm` / `wk_axpy` directly.
Everything here goes through libwekua_hip.so; nothing computes on the host.
"""
from __future__ import annotations

import ctypes

import numpy as np

from . import _capi
from ._capi import check

REAL_NAMES = ["i8", "u8", "i16", "u16", "i32", "u32", "i64", "u64", "f32", "f64"]
DTYPE_NAMES = REAL_NAMES + ["c" + n for n in REAL_NAMES]
# element formats beyond the reference's twenty; numpy holds bf16 and f8e4m3 as their bits
EXTRA_DTYPES = {"f16": 32, "bf16": 33, "f8e4m3": 34}
_NP_EXTRA = {"f16": np.float16, "bf16": np.uint16, "f8e4m3": np.uint8}
_NP_REAL = [np.int8, np.uint8, np.int16, np.uint16, np.int32, np.uint32, np.int64, np.uint64,
            np.float32, np.float64]


def dtype_id(name: str) -> int:
    return EXTRA_DTYPES[name] if name in EXTRA_DTYPES else DTYPE_NAMES.index(name)


def real_np_dtype(name: str) -> np.dtype:
    if name in _NP_EXTRA:
        return np.dtype(_NP_EXTRA[name])
    return np.dtype(_NP_REAL[dtype_id(name) % 10])


def is_complex(name: str) -> bool:
    return name.startswith("c")


def elem_size(name: str) -> int:
    return real_np_dtype(name).itemsize * (2 if is_complex(name) else 1)


def scalar_bytes(name: str, value):
    """ctypes buffer holding one element of dtype `name`, or None for an absent scalar."""
    if value is None:
        return None
    rd = real_np_dtype(name)
    if is_complex(name):
        if isinstance(value, complex):
            value = (value.real, value.imag)
        vals = list(value)
    else:
        vals = [value]
    if rd.kind in "iu":
        mask = (1 << (8 * rd.itemsize)) - 1
        arr = np.array([int(v) & mask for v in vals], dtype=np.uint64).astype(
            np.dtype("u%d" % rd.itemsize)).view(rd)
    else:
        arr = np.array(vals, dtype=rd)
    return ctypes.create_string_buffer(arr.tobytes(), arr.nbytes)


class Device:
    """One GPU and one in-order stream on it."""

    def __init__(self, ordinal: int = 0):
        self.lib = _capi.load()
        self.ordinal = ordinal
        self.dev = ctypes.c_void_p()
        check(self.lib.wk_device_open(ordinal, ctypes.byref(self.dev)), "wk_device_open")
        self.stream = ctypes.c_void_p()
        check(self.lib.wk_stream_create(self.dev, ctypes.byref(self.stream)), "wk_stream_create")
        self._live = []

    def props(self) -> _capi.WkProps:
        p = _capi.WkProps()
        check(self.lib.wk_device_props(self.dev, ctypes.byref(p)), "wk_device_props")
        return p

    def sync(self) -> None:
        check(self.lib.wk_stream_sync(self.stream), "wk_stream_sync")

    def malloc(self, nbytes: int) -> "DeviceBuffer":
        return DeviceBuffer(self, nbytes)

    def upload(self, arr: np.ndarray) -> "DeviceBuffer":
        arr = np.ascontiguousarray(arr)
        buf = DeviceBuffer(self, max(arr.nbytes, 1))
        check(self.lib.wk_copy_h2d_rect_async(self.stream, buf.ptr, arr.nbytes, 0, arr.ctypes.data, arr.nbytes, 0,
                                              arr.nbytes, 1, 1), "upload")
        self.sync()
        return buf

    def close(self) -> None:
        if self.stream:
            self.lib.wk_stream_destroy(self.stream)
            self.stream = None
        if self.dev:
            self.lib.wk_device_close(self.dev)
            self.dev = None

    def time_stream_ms(self, enqueue, iters: int) -> float:
        """Average duration in ms of `iters` calls of enqueue() measured with events recorded on
        this device's stream (the stream the kernels are launched on)."""
        e0, e1 = ctypes.c_void_p(), ctypes.c_void_p()
        check(self.lib.wk_event_create(self.dev, ctypes.byref(e0)), "wk_event_create")
        check(self.lib.wk_event_create(self.dev, ctypes.byref(e1)), "wk_event_create")
        try:
            check(self.lib.wk_event_record(e0, self.stream), "wk_event_record")
            for _ in range(iters):
                enqueue()
            check(self.lib.wk_event_record(e1, self.stream), "wk_event_record")
            check(self.lib.wk_event_sync(e1), "wk_event_sync")
            ms = ctypes.c_float()
            check(self.lib.wk_event_elapsed_ms(e0, e1, ctypes.byref(ms)), "wk_event_elapsed_ms")
        finally:
            self.lib.wk_event_destroy(e0)
            self.lib.wk_event_destroy(e1)
        return ms.value / iters

    # -- the hot path ---------------------------------------------------------------------
    def gemm(self, dtype: str, op_a: int, op_b: int, M: int, N: int, K: int, alpha, A: "DeviceBuffer", lda: int,
             B: "DeviceBuffer", ldb: int, beta, C: "DeviceBuffer", ldc: int, workspace: "DeviceBuffer | None" = None,
             b_kept: bool = False) -> None:
        """wk_gemm; b_kept: wk_gemm_packed_b_kept (the workspace still holds B's packed form)."""
        a, b = scalar_bytes(dtype, alpha), scalar_bytes(dtype, beta)
        entry = self.lib.wk_gemm_packed_b_kept if b_kept else self.lib.wk_gemm
        check(entry(self.stream, dtype_id(dtype), op_a, op_b, M, N, K,
                    ctypes.cast(a, ctypes.c_void_p) if a is not None else None, A.ptr, lda, B.ptr, ldb,
                    ctypes.cast(b, ctypes.c_void_p) if b is not None else None, C.ptr, ldc,
                    workspace.ptr if workspace is not None else None, workspace.nbytes if workspace is not None else 0),
              "wk_gemm")

    def axpy(self, dtype: str, shape3, x: "DeviceBuffer", xrp: int, xsp: int, alpha, y: "DeviceBuffer", yrp: int,
             ysp: int) -> None:
        a = scalar_bytes(dtype, alpha)
        s3 = (ctypes.c_uint64 * 3)(*shape3)
        check(self.lib.wk_axpy(self.stream, dtype_id(dtype), s3, x.ptr, xrp, xsp, y.ptr, yrp, ysp,
                               ctypes.cast(a, ctypes.c_void_p) if a is not None else None), "wk_axpy")

    # -- the token end of a network ---------------------------------------------------------
    # Buffers: DeviceBuffers, device addresses, or objects with data_ptr() whose memory is on this device and ready on
    # this stream (work of another stream on them is the caller's to wait for).
    def _address(self, buf):
        """The device address of a DeviceBuffer, of anything with data_ptr(), or a plain address; None (an operand that is not there) stays
        None.  Memory that is known to be elsewhere, or gone, is refused: the kernel would fault, or take it for an absent operand."""
        if buf is None or isinstance(buf, int):
            return buf
        if hasattr(buf, "data_ptr"):
            at, where = buf.data_ptr(), buf.get_device() if hasattr(buf, "get_device") else self.ordinal
        else:
            at, where = buf.ptr, buf.device.ordinal
        if not at or where != self.ordinal:
            raise ValueError("an operand has no memory" if not at else f"an operand is not on device {self.ordinal}")
        return at

    def dropout(self, dtype: str, shape3, x, xrp: int, xsp: int, y, yrp: int, ysp: int, p: float, seed: int, offset: int = 0,
                step=None) -> None:
        """wk_dropout; the backward pass is the same call on the gradient."""
        check(self.lib.wk_dropout(self.stream, dtype_id(dtype), (ctypes.c_uint64 * 3)(*shape3), self._address(x), xrp, xsp,
                                  self._address(y), yrp, ysp, p, seed, offset, self._address(step)), "wk_dropout")

    def f8_quantize(self, dtype: str, rows: int, cols: int, x, pitch: int, block_rows: int, q, q_pitch: int, scales,
                    scale_pitch: int) -> None:
        """wk_f8_quantize: 8-bit codes and a scale for each block of block_rows (1 or 128) x 128 elements."""
        check(self.lib.wk_f8_quantize(self.stream, dtype_id(dtype), rows, cols, self._address(x), pitch, block_rows, self._address(q), q_pitch,
                                      self._address(scales), scale_pitch), "wk_f8_quantize")

    def gemm_f8(self, M: int, N: int, K: int, A, lda: int, a_scales, a_scale_pitch: int, B, ldb: int, b_scales, b_scale_pitch: int,
                out_dtype: str, C, ldc: int, bias=None, kind: int = -1) -> None:
        """wk_gemm_f8: C = act(A B^T + bias) of 8-bit operands with block scales."""
        check(self.lib.wk_gemm_f8(self.stream, M, N, K, self._address(A), lda, self._address(a_scales), a_scale_pitch, self._address(B), ldb,
                                  self._address(b_scales), b_scale_pitch, dtype_id(out_dtype), self._address(C), ldc, self._address(bias), kind), "wk_gemm_f8")

    def token_logprobs_workspace_bytes(self, dtype: str, rows: int, vocab: int, top: int = 0) -> int:
        return int(self.lib.wk_token_logprobs_workspace_bytes(dtype_id(dtype), rows, vocab, top))

    def token_logprobs(self, dtype: str, rows: int, vocab: int, logits, pitch: int, targets, target_dtype: str = "i32", logprob=None,
                       lse=None, entropy=None, top: int = 0, top_ids=None, top_logprobs=None, workspace=None,
                       workspace_bytes: int = 0) -> None:
        """wk_token_logprobs; outputs that are None are not computed."""
        check(self.lib.wk_token_logprobs(self.stream, dtype_id(dtype), rows, vocab, self._address(logits), pitch, self._address(targets),
                                         dtype_id(target_dtype), self._address(logprob), self._address(lse), self._address(entropy), top,
                                         self._address(top_ids), self._address(top_logprobs), self._address(workspace), workspace_bytes), "wk_token_logprobs")

    def token_logprobs_grad(self, dtype: str, rows: int, vocab: int, logits, pitch: int, targets, target_dtype: str, lse, entropy,
                            logprob_grad, entropy_grad, logits_grad, grad_pitch: int) -> None:
        """wk_token_logprobs_grad: the gradient of the logits from those of the log probabilities and entropies."""
        check(self.lib.wk_token_logprobs_grad(self.stream, dtype_id(dtype), rows, vocab, self._address(logits), pitch, self._address(targets),
                                              dtype_id(target_dtype), self._address(lse), self._address(entropy), self._address(logprob_grad),
                                              self._address(entropy_grad), self._address(logits_grad), grad_pitch), "wk_token_logprobs_grad")


class DeviceBuffer:
    def __init__(self, device: Device, nbytes: int):
        self.device = device
        self.nbytes = nbytes
        self.ptr = ctypes.c_void_p()
        check(device.lib.wk_malloc(device.dev, nbytes, ctypes.byref(self.ptr)), "wk_malloc")

    def download(self, dtype: np.dtype, shape) -> np.ndarray:
        out = np.empty(shape, dtype=dtype)
        d = self.device
        check(d.lib.wk_copy_d2h_rect_async(d.stream, out.ctypes.data, out.nbytes, 0, self.ptr, out.nbytes, 0,
                                           out.nbytes, 1, 1), "download")
        d.sync()
        return out

    def write(self, arr: np.ndarray) -> None:
        arr = np.ascontiguousarray(arr)
        d = self.device
        check(d.lib.wk_copy_h2d_rect_async(d.stream, self.ptr, arr.nbytes, 0, arr.ctypes.data, arr.nbytes, 0,
                                           arr.nbytes, 1, 1), "write")
        d.sync()

    def free(self) -> None:
        if self.ptr:
            check(self.device.lib.wk_free(self.device.dev, self.ptr), "wk_free")
            self.ptr = None

    def __del__(self):
        try:
            if self.ptr and self.device.dev:
                self.device.lib.wk_free(self.device.dev, self.ptr)
        except Exception:
            pass
