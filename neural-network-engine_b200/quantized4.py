"""``QLinear4``: the 4-bit sibling of ``QLinear``.  Codes of four bits, one f32 scale for each group of 32, 64
or 128 consecutive inputs of a row.  The rounding rule is the one of the reference's int8 layer
(src/nn/quantized.rs:107-127) with 7 in the place of 127 and a group in the place of a row; the class
has the methods of ``QLinear``.  Every computation is a call through the ``nne_cuda`` C ABI.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional

import numpy as np

from . import _lib
from ._lib import NneError, check, load
from .quantized import (CudaContext, CudaQLinear, GpuError, InvalidArgument, Linear, ShapeMismatch, _ptr, _raise_mapped,
                        default_context)


def quantize_rows4_device(ctx: CudaContext, w_ptr: int, rows: int, cols: int, group: int, q_ptr: int, scales_ptr: int,
                          stream: int = 0) -> None:
    """Quantizes ``w [rows, cols]`` f32 on the device: codes ``[rows, (cols + 1) // 2]`` bytes (two's complement, the
    even column in the low four bits) and scales ``[rows, ceil(cols / group)]`` f32."""
    try:
        check(load().nne_quantize_rows4_dev(ctx.handle, w_ptr, rows, cols, group, q_ptr, scales_ptr, stream))
    except NneError as e:
        _raise_mapped(e)


class QLinear4:
    """4-bit linear layer; ``qweight`` (uint8 ``[out_features, (in_features + 1) // 2]``) and ``scales`` (f32
    ``[out_features, ceil(in_features / group)]``) and ``bias`` are host copies, fetched from the device when first asked
    for."""

    def __init__(self, handle, in_features: int, out_features: int, group: int, ctx: CudaContext):
        self._handle, self._ctx = handle, ctx
        self.in_features, self.out_features, self.group = int(in_features), int(out_features), int(group)
        self._host = None
        # bound once: a forward is one foreign call, without a look-up on its way
        self._forward, self._forward_strided = load().nne_qlinear4_forward_dev, load().nne_qlinear4_forward_dev_strided

    # -- construction --------------------------------------------------------------------------
    @classmethod
    def from_linear(cls, linear: Linear, group: int = 128, ctx: Optional[CudaContext] = None) -> "QLinear4":
        ctx = ctx or default_context()
        n, k = linear.out_features, linear.in_features
        w = np.ascontiguousarray(linear.weight, dtype=np.float32)
        b = None if linear.bias is None else np.array(linear.bias, dtype=np.float32)
        h = C.c_void_p()
        try:
            check(load().nne_qlinear4_create_from_f32(ctx.handle, _ptr(w), _ptr(b), n, k, group, C.byref(h)))
        except NneError as e:
            _raise_mapped(e)
        return cls(h, k, n, group, ctx)

    @classmethod
    def from_fields(cls, qweight, scales, bias, in_features: int, out_features: int, group: int,
                    ctx: Optional[CudaContext] = None) -> "QLinear4":
        """From host codes and scales in the public layout."""
        n, k = int(out_features), int(in_features)
        if group not in (32, 64, 128):
            raise InvalidArgument(f"group must be 32, 64 or 128 columns, got {group}")
        q = np.ascontiguousarray(qweight, dtype=np.uint8)
        s = np.ascontiguousarray(scales, dtype=np.float32)
        b = None if bias is None else np.array(bias, dtype=np.float32).reshape(-1)
        if q.size != n * ((k + 1) // 2) or s.size != n * -(-k // group) or (b is not None and b.size != n):
            raise InvalidArgument("field sizes do not match in_features/out_features/group")
        ctx = ctx or default_context()
        h = C.c_void_p()
        try:
            check(load().nne_qlinear4_create_from_i4(ctx.handle, _ptr(q), _ptr(s), _ptr(b), n, k, group, C.byref(h)))
        except NneError as e:
            _raise_mapped(e)
        return cls(h, k, n, group, ctx)

    @classmethod
    def from_packed_device(cls, ctx: CudaContext, q_ptr: int, scales_ptr: int, bias_ptr: int, n: int, k: int, group: int,
                           stream: int = 0) -> "QLinear4":
        """From codes and scales in the public layout that are on the device (``bias_ptr`` 0: none).  The buffers are
        not kept."""
        h = C.c_void_p()
        try:
            check(load().nne_qlinear4_create_from_i4_dev(ctx.handle, q_ptr, scales_ptr, bias_ptr or None, n, k, group, stream,
                                                         C.byref(h)))
        except NneError as e:
            _raise_mapped(e)
        return cls(h, k, n, group, ctx)

    @classmethod
    def from_linear_device(cls, ctx: CudaContext, w_ptr: int, bias_ptr: int, n: int, k: int, group: int = 128,
                           stream: int = 0) -> "QLinear4":
        """Quantizes f32 weights ``[n, k]`` that are on the device."""
        h = C.c_void_p()
        try:
            check(load().nne_qlinear4_create_from_f32_dev(ctx.handle, w_ptr, bias_ptr or None, n, k, group, stream, C.byref(h)))
        except NneError as e:
            _raise_mapped(e)
        return cls(h, k, n, group, ctx)

    # -- fields ----------------------------------------------------------------------------------
    def _live_handle(self):
        if self._handle is None:
            raise GpuError("layer has no device handle")
        return self._handle

    def _fields(self):
        if self._host is None:
            q = np.zeros((self.out_features, (self.in_features + 1) // 2), dtype=np.uint8)
            s = np.zeros((self.out_features, -(-self.in_features // self.group)), dtype=np.float32)
            try:
                has_bias = C.c_int()
                check(load().nne_qlinear4_info(self._live_handle(), None, None, None, C.byref(has_bias)))
                b = np.zeros(self.out_features, dtype=np.float32) if has_bias.value else None
                check(load().nne_qlinear4_download(self._live_handle(), _ptr(q), _ptr(s), _ptr(b)))
            except NneError as e:
                _raise_mapped(e)
            self._host = (q, s, b)
        return self._host

    @property
    def qweight(self) -> np.ndarray:
        return self._fields()[0]

    @property
    def scales(self) -> np.ndarray:
        return self._fields()[1]

    @property
    def bias(self) -> Optional[np.ndarray]:
        return self._fields()[2]

    def to_linear(self) -> Linear:
        """The f32 layer this one stands for, q * scale."""
        w = np.zeros((self.out_features, self.in_features), dtype=np.float32)
        try:
            check(load().nne_qlinear4_dequantize(self._live_handle(), _ptr(w)))
        except NneError as e:
            _raise_mapped(e)
        return Linear(w, None if self.bias is None else self.bias.copy())

    def memory_bytes(self) -> int:
        """Device bytes of codes, scales and bias."""
        return int(load().nne_qlinear4_memory_bytes(self._live_handle()))

    def parameters(self) -> list:
        return []

    # -- forward -------------------------------------------------------------------------------
    def forward(self, input: np.ndarray) -> np.ndarray:
        """The checks and shapes of ``QLinear.forward`` (src/nn/quantized.rs:146-197)."""
        x = np.asarray(input)
        if x.ndim < 2:
            raise InvalidArgument(f"QLinear forward expects tensor with at least 2 dimensions, got {list(x.shape)}")
        if x.shape[-1] != self.in_features:
            raise ShapeMismatch([self.in_features], [x.shape[-1]])
        rows = int(np.prod(x.shape[:-1], dtype=np.int64))
        xc = np.ascontiguousarray(x, dtype=np.float32)
        out = np.zeros(x.shape[:-1] + (self.out_features,), dtype=np.float32)
        try:
            check(load().nne_qlinear4_forward_host(self._live_handle(), _ptr(xc), rows, self.in_features, _ptr(out)))
        except NneError as e:
            _raise_mapped(e)
        return out

    def forward_device(self, x_ptr: int, m: int, y_ptr: int, stream: int = 0, ldy: Optional[int] = None) -> None:
        """Device-resident forward: x [m, in_features] and y [m, out_features] (row stride ``ldy`` floats) are device
        pointers; asynchronous on the CUDA stream ``stream``."""
        if ldy is None:
            status = self._forward(self._handle, x_ptr, m, self.in_features, y_ptr, stream)
        else:
            status = self._forward_strided(self._handle, x_ptr, m, self.in_features, y_ptr, ldy, stream)
        if status != _lib.OK:
            self._live_handle()
            _raise_mapped(NneError(status, _lib.last_error()))

    def to_gpu(self, ctx: Optional[CudaContext] = None) -> CudaQLinear:
        """The layer over device tensors, as ``QLinear.to_gpu``; the context is the layer's own."""
        if ctx is not None and ctx is not self._ctx:
            raise InvalidArgument("a QLinear4 stays on its own context")
        return CudaQLinear(self, self._ctx)

    def close(self):
        if self._handle is not None:
            load().nne_qlinear4_destroy(self._handle)
            self._handle = None

    def __del__(self):  # pragma: no cover - best effort
        try:
            self.close()
        except Exception:
            pass
