"""The LM head with low-rank adapters of many requests (ncb_adapter_head_* in
include/navsampler.h): the projection whose logits the samplers read, each row
with the adapter of its own request.

Like CudaTokenSampler, the handle owns packed adapters and scratch on its device
and the caller owns every input and output tensor; torch is the allocator and
stream provider only.
"""
from __future__ import annotations

import ctypes

from .native import check, load
from .sampler import _stream_ptr, dtype_code


def _rows_of(t, name: str, cols: int, dtype, device) -> int:
    """Row stride of a [*, cols] matrix with contiguous rows; ValueError otherwise."""
    if t.dim() != 2 or t.shape[1] != cols or t.dtype != dtype or t.device != device:
        raise ValueError(f"{name} must be [*, {cols}] {dtype} on {device}")
    if cols > 1 and t.stride(1) != 1:
        raise ValueError(f"{name}: a row's values must be contiguous")
    return t.stride(0) if t.shape[0] > 1 else cols


class CudaAdapterHead:
    """out[n, :] = weight x_n + scale_s b_s (a_s x_n), s the adapter of row n.

    `weight`: [out_features, in_features] float16 or bfloat16 on a GPU; it is kept and read in
    place (copied only where its rows do not start on 16-byte boundaries: after changing such a
    weight in place call set_weight again)."""

    def __init__(self, weight, max_rows: int, max_adapters: int = 0, max_rank: int = 0,
                 stream=None):
        self._h = None
        if weight.dim() != 2 or weight.device.type != "cuda":
            raise ValueError("weight must be [out_features, in_features] on a CUDA device")
        self._lib = load()
        self.out_features, self.in_features = weight.shape
        self.dtype, self.device = weight.dtype, weight.device
        self.max_rows, self.max_adapters, self.max_rank = max_rows, max_adapters, max_rank
        h = ctypes.c_void_p()
        check(self._lib.ncb_adapter_head_create(
            self.device.index, dtype_code(self.dtype), self.in_features, self.out_features,
            max_rows, max_adapters, max_rank, ctypes.byref(h)), "ncb_adapter_head_create")
        self._h = h
        self.set_weight(weight, stream)

    def close(self) -> None:
        if getattr(self, "_h", None) is not None and self._h.value:
            check(self._lib.ncb_adapter_head_destroy(self._h), "ncb_adapter_head_destroy")
            self._h = None

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def set_weight(self, weight, stream=None) -> None:
        """The shared weight, same shape, type and device as the one the head was made with. The
        head holds on to this tensor only: graphs captured with an earlier one still read that."""
        if weight.shape[0] != self.out_features:
            raise ValueError(f"weight must have {self.out_features} rows")
        ld = _rows_of(weight, "weight", self.in_features, self.dtype, self.device)
        check(self._lib.ncb_adapter_head_set_weight_device(
            self._h, weight.data_ptr(), ld, _stream_ptr(stream)),
            "ncb_adapter_head_set_weight_device")
        self._weight = weight  # read by every later call

    def set_adapter(self, slot: int, a, b, scale: float = 1.0, stream=None) -> None:
        """Copies an adapter into a slot: a [rank, in_features], b [out_features, rank]."""
        rank = a.shape[0]
        lda = _rows_of(a, "a", self.in_features, self.dtype, self.device)
        if b.shape[0] != self.out_features:
            raise ValueError(f"b must have {self.out_features} rows")
        ldb = _rows_of(b, "b", rank, self.dtype, self.device)
        check(self._lib.ncb_adapter_head_set_adapter_device(
            self._h, int(slot), a.data_ptr(), lda, b.data_ptr(), ldb, rank, float(scale),
            _stream_ptr(stream)), "ncb_adapter_head_set_adapter_device")

    def clear_adapter(self, slot: int, stream=None) -> None:
        """Empties a slot: rows that name it get the shared projection alone."""
        check(self._lib.ncb_adapter_head_clear_adapter_device(self._h, int(slot),
                                                              _stream_ptr(stream)),
              "ncb_adapter_head_clear_adapter_device")

    def project_device(self, x, adapter_ids, out, stream=None) -> None:
        """out [rows, out_features] (float32 or the head's type, any row stride) from x
        [rows, in_features]; adapter_ids: rows int32 slots (-1: none), or None for no adapters.
        Asynchronous on `stream` (None: the legacy default stream)."""
        device = self.device
        rows = x.shape[0]
        ldx = _rows_of(x, "x", self.in_features, self.dtype, device)
        if out.dtype != self.dtype and str(out.dtype) != "torch.float32":
            raise ValueError(f"out must be float32 or {self.dtype}")
        if out.shape[0] != rows:
            raise ValueError(f"out must have {rows} rows")
        ldo = _rows_of(out, "out", self.out_features, out.dtype, device)
        ids = None
        if adapter_ids is not None:
            if str(adapter_ids.dtype) != "torch.int32" or adapter_ids.numel() != rows \
                    or not adapter_ids.is_contiguous() or adapter_ids.device != device:
                raise ValueError(f"adapter_ids must be {rows} contiguous int32 on {device}")
            ids = adapter_ids.data_ptr()
        check(self._lib.ncb_adapter_head_project_device(
            self._h, x.data_ptr(), ldx, rows, ids, out.data_ptr(), dtype_code(out.dtype), ldo,
            _stream_ptr(stream)), "ncb_adapter_head_project_device")

    def check(self) -> None:
        """NcbError if a wait inside one of the head's kernels gave up, which leaves that call's
        output undefined. It waits for nothing: call it once the stream has been synchronised."""
        check(self._lib.ncb_adapter_head_status(self._h), "ncb_adapter_head_status")


__all__ = ["CudaAdapterHead"]
