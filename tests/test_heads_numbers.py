"""Sizes that are no whole numbers of their C type are refused, not cut to ones that are (no GPU)."""
import math

import numpy as np
import pytest

import ruvector_amd as rv
from ruvector_amd.device import int32, int64


class Nothing:
    handle = None


def calls(v):
    b = Nothing()
    layer = rv.AdapterLinear.__new__(rv.AdapterLinear)
    layer._h = None
    yield lambda: rv.embedding_forward_device(b, 8, 8, b, v, b)
    yield lambda: rv.embedding_forward_device(b, v, 8, b, 8, b)
    yield lambda: rv.embedding_forward_device(b, 8, v, b, 8, b)
    yield lambda: rv.embedding_backward_device(b, b, v, 8, 8, b)
    yield lambda: rv.embedding_backward_device(b, b, 8, v, 8, b)
    yield lambda: rv.log_probs_device(b, v, 8)
    yield lambda: rv.log_probs_device(b, 8, v, ld=8)
    yield lambda: rv.log_probs_device(b, 8, 8, ld=v)
    yield lambda: rv.log_probs_device(b, 8, 8, k=v)
    yield lambda: rv.log_probs_backward_device(b, 8, 8, 1.0, b, b, ld=v)
    yield lambda: rv.log_probs_backward_device(b, 8, 8, 1.0, b, b, ld_grad=v)
    yield lambda: layer.forward_device(b, v, b)


@pytest.mark.parametrize("value", [2 ** 64 + 8, -2 ** 64 + 8, 2 ** 63, 8.5, np.float32(8.25)])
def test_refused(value):
    for call in calls(value):
        with pytest.raises(rv.RvxError, match="whole number"):
            call()


@pytest.mark.parametrize("value", [8, np.int64(8), np.int32(8), 8.0])
def test_taken(value):
    assert int32(value, "n") == int64(value, "n") == int(value)
    for call in calls(value):
        with pytest.raises(rv.RvxError, match="null"):  # the buffers are what is missing
            call()


@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_not_numbers(value):
    with pytest.raises((ValueError, OverflowError, rv.RvxError)):
        int64(value, "n")
