"""What a Buffer gives as a DLPack tensor: a view, a copy where one is asked for, nothing on another device."""
import os
import subprocess
import sys

import pytest

rv = pytest.importorskip("ruvector_amd")

# A process of its own: torch first, so that it and the library share one HIP runtime.
COPIES = """
import gc
import numpy as np
import torch
import ruvector_amd as rv
b = rv.Buffer.from_numpy(np.arange(64, dtype=np.float32))
view = torch.from_dlpack(b)
for again in range(2):
    copy = torch.from_dlpack(b, copy=True)
    assert copy.device == view.device and copy.dtype == torch.uint8 and copy.data_ptr() != view.data_ptr()
    assert torch.equal(copy, view)
    copy.fill_(3)
    torch.cuda.synchronize()
    assert torch.equal(view.view(torch.float32).cpu(), torch.arange(64, dtype=torch.float32))
assert torch.from_dlpack(b, copy=False).data_ptr() == view.data_ptr()
assert torch.from_dlpack(b, device="cuda:0").data_ptr() == view.data_ptr()
host = torch.from_dlpack(b, device="cpu")
assert host.device.type == "cpu" and torch.equal(host.view(torch.float32), torch.arange(64, dtype=torch.float32))
# behind what the consumer's stream writes, before what the library writes later
big = rv.Buffer(1 << 26)
t, side = torch.from_dlpack(big), torch.cuda.Stream()
torch.cuda.synchronize()
with torch.cuda.stream(side):
    torch.cuda._sleep(20_000_000)
    t.fill_(7)
    c = torch.from_dlpack(big, copy=True)
    big.zero()
    assert (c == 7).all()
    side.synchronize()
    rv.synchronize()
    assert not t.any()
# a copy outlives its Buffer, and goes with its tensor
big.free()
del t, big
gc.collect()
assert (c == 7).all()
capsule = b.__dlpack__(stream=-1, copy=True)   # nobody takes it
del capsule
large = rv.Buffer(1 << 30)
large.zero()
rv.synchronize()
free = torch.cuda.mem_get_info()[0]
held = torch.from_dlpack(large, copy=True)
assert torch.cuda.mem_get_info()[0] < free - (1 << 29)
del held
assert torch.cuda.mem_get_info()[0] > free - (1 << 29)
empty = torch.cuda.CUDAGraph()
with torch.cuda.graph(empty):
    view += 1
    try:
        torch.from_dlpack(b, copy=True)
        raise SystemExit("a stream being captured was taken")
    except rv.RvxError as e:
        assert "captured" in str(e), e
empty.replay()
torch.cuda.synchronize()
print("copies ok", flush=True)
"""


@pytest.mark.gpu
def test_copies():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-u", "-c", COPIES], cwd=root, capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and "copies ok" in r.stdout, r.stdout + r.stderr


@pytest.fixture
def freed():
    b = rv.Buffer.__new__(rv.Buffer)  # as after free(): no device is looked at
    b._h, b._device, b.nbytes = None, 1, 8
    return b


@pytest.mark.parametrize("where", [(1, 0), (10, 0), (2, 1)])
def test_another_device_is_refused(freed, where):
    with pytest.raises(BufferError):
        freed.__dlpack__(dl_device=where)


@pytest.mark.parametrize("more", [{}, dict(copy=True), dict(copy=False), dict(dl_device=(10, 1)), dict(max_version=(1, 0))])
def test_a_freed_buffer_is_refused(freed, more):
    with pytest.raises(rv.RvxError):
        freed.__dlpack__(**more)
    with pytest.raises(TypeError):
        freed.__dlpack__(**more, unknown=1)


def test_no_buffer():
    import ctypes as C
    from ruvector_amd import _lib as L
    p = C.c_void_p()
    for name in ("rvx_buffer_tensor", "rvx_buffer_copy_tensor"):
        assert getattr(L.load(), name)(None, C.byref(p)) == 2 and not p.value
