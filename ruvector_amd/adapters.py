"""AdapterLinear: a shared projection with one low-rank adapter per row (rvx_adapter_linear_*).

One batch may hold rows of many tenants or requests, each with an adapter of its own — the query
embeddings of many users before one search, the tokens of many requests in one step.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional

from . import _lib as L
from .device import Buffer, dtype_code, int32, int64


class AdapterError(L.RvxError):
    pass


def _check(name, *args):
    try:
        L.call(name, *args)
    except L.RvxError as e:
        raise AdapterError(e.code, str(e).split(": ", 1)[-1]) from None


class AdapterLinear:
    """y[i] = W x[i] + bias + scale_r B_r (A_r x[i]), r = adapter_ids[i]: weight [out][in] and bias
    [out] of `dtype` are copied into the layer's layout, as are the adapters."""

    def __init__(self, in_features: int, out_features: int, weight: Buffer, bias: Optional[Buffer] = None,
                 max_rank: int = 16, max_adapters: int = 8, dtype: str = "f32"):
        self._h = None
        self.in_features, self.out_features, self.dtype = in_features, out_features, dtype
        self.max_rank, self.max_adapters = max_rank, max_adapters
        cfg = L.AdapterLinearConfig(int32(in_features, "in_features"), int32(out_features, "out_features"), dtype_code(dtype),
                                    int32(max_rank, "max_rank"), int32(max_adapters, "max_adapters"))
        h = C.c_void_p()
        _check("rvx_adapter_linear_create", C.byref(cfg), weight.handle, None if bias is None else bias.handle, C.byref(h))
        self._h = h

    def set_adapter(self, slot: int, rank: int, a: Buffer, b: Buffer, scale: float = 1.0) -> None:
        """Slot `slot` gets a [rank][in] and b [out][rank] of the layer's dtype (rank <= max_rank)."""
        _check("rvx_adapter_linear_set", self._h, int32(slot, "slot"), int32(rank, "rank"), a.handle, b.handle, float(scale))

    def clear_adapter(self, slot: int) -> None:
        """Rows of `slot` have no adapter from now on."""
        _check("rvx_adapter_linear_set", self._h, int32(slot, "slot"), 0, None, None, 1.0)

    def forward_device(self, x: Buffer, n: int, y: Buffer, adapter_ids: Optional[Buffer] = None) -> None:
        """x [n][in] -> y [n][out]; adapter_ids int32 [n], ids without an adapter (-1) get none."""
        _check("rvx_adapter_linear_forward_device", self._h, x.handle, int64(n, "n"), None if adapter_ids is None else adapter_ids.handle,
               y.handle)

    def __del__(self):
        try:
            if self._h:
                L.call("rvx_adapter_linear_destroy", self._h)
                self._h = None
        except Exception:
            pass
