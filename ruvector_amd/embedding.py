"""Rows of a learned table by id, and the gradient of the table (rvx_embedding_*).

The trainable side of the node and query embeddings that the layers of gnn.py read: ids are int64,
as cand_ids there, and an id outside the table is absent.
"""
from __future__ import annotations

from . import _lib as L
from .device import Buffer, dtype_code, int32, int64


class EmbeddingError(L.RvxError):
    pass


def _check(name, *args):
    try:
        L.call(name, *args)
    except L.RvxError as e:
        raise EmbeddingError(e.code, str(e).split(": ", 1)[-1]) from None


def embedding_forward_device(table: Buffer, rows: int, dim: int, ids: Buffer, n: int, out: Buffer,
                             scale: float = 1.0, dtype: str = "f32") -> None:
    """out[i] = scale * table[ids[i]] for i < n: table [rows][dim] and out [n][dim] of `dtype`
    ("f32", "f16", "bf16"), ids int64; the row of an id outside [0, rows) is zeros."""
    _check("rvx_embedding_forward_device", table.handle, dtype_code(dtype), int64(rows, "rows"), int32(dim, "dim"),
           ids.handle, int64(n, "n"), scale, out.handle)


def embedding_backward_device(grad_out: Buffer, ids: Buffer, n: int, rows: int, dim: int, grad_table: Buffer,
                              scale: float = 1.0, dtype: str = "f32", table_dtype: str = None,
                              accumulate: bool = False) -> None:
    """The gradient of the table: g[v] = scale * sum of grad_out[i] over ids[i] = v, grad_out [n][dim]
    of `dtype`. grad_table [rows][dim] of `table_dtype` (default: `dtype`) becomes g, or, with
    `accumulate`, grows by g: then the rows of ids that do not occur are left as they are. The sums
    are kept in 32 bits in an order given by the ids alone: the same bits every call."""
    code = dtype_code(dtype)
    _check("rvx_embedding_backward_device", grad_out.handle, code, ids.handle, int64(n, "n"), int64(rows, "rows"),
           int32(dim, "dim"), scale,
           1 if accumulate else 0, code if table_dtype is None else dtype_code(table_dtype), grad_table.handle)
