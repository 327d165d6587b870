"""Arguments that the typed operators refuse, without a GPU: what is wrong by itself is found
before any buffer or device is looked at."""
import pytest

import ruvector_amd as rv
from ruvector_amd import _lib as L


def _status(name, *args):
    lib = L.load()
    st = getattr(lib, name)(*args)
    return st, L.last_error()


@pytest.mark.parametrize("dtype,rows,dim,n,word", [
    (3, 8, 8, 8, "dtype"), (-1, 8, 8, 8, "dtype"), (0, 0, 8, 8, "rows"), (0, 2 ** 31 - 1, 8, 8, "rows"),
    (0, 8, 0, 8, "dim"), (0, 8, 65537, 8, "dim"), (0, 8, 8, -1, "n must"), (0, 8, 8, 2 ** 31, "n must"), (0, 8, 8, 8, "null")])
def test_embedding(dtype, rows, dim, n, word):
    st, msg = _status("rvx_embedding_forward_device", None, dtype, rows, dim, None, n, 1.0, None)
    assert st == 2 and word in msg
    st, msg = _status("rvx_embedding_backward_device", None, dtype, None, n, rows, dim, 1.0, 0, 0, None)
    assert st == 2 and word in msg


@pytest.mark.parametrize("scale", [float("inf"), float("nan")])
def test_embedding_scale(scale):
    assert _status("rvx_embedding_forward_device", None, 0, 8, 8, None, 8, scale, None)[0] == 2
    assert _status("rvx_embedding_backward_device", None, 0, None, 8, 8, 8, scale, 0, 0, None)[0] == 2


def test_numbers_past_32_bits():
    from ruvector_amd.device import int32
    assert int32(-2 ** 31, "k") == -2 ** 31
    for bad in (2 ** 31, -2 ** 31 - 1, 2 ** 32 + 8):
        with pytest.raises(rv.RvxError):
            int32(bad, "k")


def test_embedding_table_dtype():
    st, msg = _status("rvx_embedding_backward_device", None, 0, None, 8, 8, 8, 1.0, 0, 9, None)
    assert st == 2 and "dtype" in msg


@pytest.mark.parametrize("dtype,n,c,ld,temperature,k,word", [
    (7, 4, 8, 8, 1.0, 0, "dtype"), (0, -1, 8, 8, 1.0, 0, "n must"), (0, 2 ** 31, 8, 8, 1.0, 0, "n must"),
    (0, 4, 0, 8, 1.0, 0, "c must"), (0, 4, 2 ** 31, 2 ** 32, 1.0, 0, "c must"), (0, 4, 8, 7, 1.0, 0, "stride"),
    (0, 4, 8, 2 ** 41, 1.0, 0, "stride"), (0, 4, 8, 8, 0.0, 0, "temperature"), (0, 4, 8, 8, -1.0, 0, "temperature"),
    (0, 4, 8, 8, float("nan"), 0, "temperature"), (0, 4, 8, 8, float("inf"), 0, "temperature"),
    (0, 4, 8, 8, 1e-45, 0, "temperature"), (0, 4, 8, 8, 1.0, 0, "null")])
def test_log_probs(dtype, n, c, ld, temperature, k, word):
    st, msg = _status("rvx_log_probs_device", None, dtype, n, c, ld, temperature, None, k, *[None] * 6)
    assert st == 2 and word in msg
    st, msg = _status("rvx_log_probs_backward_device", None, dtype, n, c, ld, temperature, None, None, None, None, None, None, ld)
    assert st == 2 and word in msg


@pytest.mark.parametrize("k", [-1, 65])
def test_log_probs_k(k):
    st, msg = _status("rvx_log_probs_device", None, 0, 4, 8, 8, 1.0, None, k, *[None] * 6)
    assert st == 2 and "k must" in msg


def test_dtype_names():
    from ruvector_amd.device import dtype_code
    assert [dtype_code(d) for d in ("f32", "f16", "bf16")] == [0, 1, 2]
    for bad in ("f64", None, 2, []):
        with pytest.raises(rv.RvxError):
            dtype_code(bad)


@pytest.mark.parametrize("inp,out,dtype,rank,slots,word", [
    (0, 8, 0, 8, 1, "features"), (8, 0, 0, 8, 1, "features"), (65537, 8, 0, 8, 1, "features"), (8, 8, 3, 8, 1, "dtype"),
    (8, 8, 0, 0, 1, "max_rank"), (8, 8, 0, 129, 1, "max_rank"), (8, 8, 0, 8, -1, "max_adapters"), (8, 8, 0, 8, 65537, "max_adapters"),
    (8, 8, 0, 8, 1, "null weight")])
def test_adapter_linear(inp, out, dtype, rank, slots, word):
    import ctypes as C
    cfg, h = L.AdapterLinearConfig(inp, out, dtype, rank, slots), C.c_void_p()
    st, msg = _status("rvx_adapter_linear_create", C.byref(cfg), None, None, C.byref(h))
    assert st in (2, 4) and word in msg and not h.value
    assert _status("rvx_adapter_linear_set", None, 0, 4, None, None, 1.0)[0] == 2
    assert _status("rvx_adapter_linear_forward_device", None, None, 1, None, None)[0] == 2
    assert _status("rvx_adapter_linear_destroy", None)[0] == 0
