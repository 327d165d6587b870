"""What the tests of the typed operators share: element types, buffers from tensors, tolerances."""
import math

import torch

import ruvector_amd as rv

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
# half a step of each type, relative to the value
HALF = {k: torch.finfo(t).eps / 2 for k, t in DTYPES.items()}
# half of the smallest step of each type (subnormals)
TINY = {"f32": 2.0 ** -150, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}
F32 = 2.0 ** -24


def to_buffer(t: torch.Tensor) -> rv.Buffer:
    """A CPU tensor's bytes in a device buffer."""
    t = t.contiguous()
    b = rv.Buffer(max(t.numel() * t.element_size(), 1))
    if t.numel():
        b.upload(t.view(torch.uint8).reshape(-1).numpy() if t.dtype != torch.uint8 else t.numpy())
    return b


def out_buffer(shape, dtype, fill=0x7b) -> rv.Buffer:
    """A device buffer for an output, filled with a pattern."""
    n = max(math.prod(shape) * torch.empty((), dtype=dtype).element_size(), 1)
    return to_buffer(torch.full((n,), fill, dtype=torch.uint8))


def from_buffer(b: rv.Buffer, shape, dtype) -> torch.Tensor:
    n = math.prod(shape) * torch.empty((), dtype=dtype).element_size()
    import numpy as np
    raw = torch.from_numpy(b.download(np.uint8, (n,)))
    return raw.view(dtype).reshape(shape)


def assert_within(got, want, tol, what=""):
    """|got - want| <= tol elementwise, with equal infinities and NaN (want, tol in 64 bits)."""
    got, want = got.double(), want.double()
    assert got.shape == want.shape, what
    fine = torch.isfinite(want)
    assert torch.equal(fine, torch.isfinite(got)), what
    assert torch.equal(torch.isnan(want), torch.isnan(got)), what
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]), what
    tol = torch.as_tensor(tol, dtype=torch.float64).expand_as(want)
    over = ((got - want).abs() - tol)[fine]
    if over.numel():
        at = int(over.argmax())
        assert over.max() <= 0, f"{what}: off by {(got - want)[fine][at]:.3g}, {tol[fine][at]:.3g} allowed, value {want[fine][at]:.6g}"
