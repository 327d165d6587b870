"""Rows of a table by id and their gradient against sums in 64 bits."""
import math

import pytest
import torch

rv = pytest.importorskip("ruvector_amd")
from heads_ref import DTYPES, F32, HALF, TINY, assert_within, from_buffer, out_buffer, to_buffer  # noqa: E402

pytestmark = pytest.mark.gpu


def _ids(n, rows, kind, g):
    if kind == "same":
        return torch.full((n,), rows // 2, dtype=torch.int64)
    if kind == "zipf":
        u = torch.rand(n, generator=g, dtype=torch.float64)
        return ((torch.exp(u * math.log(rows + 1)) - 1).long()).clamp(0, rows - 1)
    ids = torch.randint(0, rows, (n,), generator=g)
    if kind == "absent":  # below, past the end, far away
        ids[::3] = -1
        ids[1::5] = rows
        if n > 2:
            ids[2] = 2 ** 40
            ids[-1] = -2 ** 63
    return ids


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,dim,n,kind", [
    (1, 1, 1, "uniform"), (7, 3, 64, "absent"), (1000, 128, 65, "uniform"), (500, 767, 333, "absent"),
    (300, 1025, 1000, "zipf"), (64, 8, 5000, "uniform"), (50, 65536, 3, "uniform")])
def test_forward(dtype, rows, dim, n, kind):
    g = torch.Generator().manual_seed(rows * 31 + n)
    table = torch.randn(rows, dim, generator=g).to(DTYPES[dtype])
    ids = _ids(n, rows, kind, g)
    for scale in (1.0, math.sqrt(dim)):
        out = out_buffer((n, dim), DTYPES[dtype])
        rv.embedding_forward_device(to_buffer(table), rows, dim, to_buffer(ids), n, out, scale=scale, dtype=dtype)
        got = from_buffer(out, (n, dim), DTYPES[dtype])
        there = (ids >= 0) & (ids < rows)
        s32 = torch.tensor(scale, dtype=torch.float32).double()
        want = table[ids.clamp(0, rows - 1)].double() * s32 * there[:, None]
        # one product in 32 bits, one rounding to the type
        assert_within(got, want, want.abs() * (HALF[dtype] + (F32 if dtype != "f32" else 0)) * (1 + 1e-6) + TINY[dtype])
        if scale == 1.0:
            assert torch.equal(got.double(), want)


def _grad_case(dtype, table_dtype, rows, dim, n, kind, accumulate, scale=1.5, seed=0):
    g = torch.Generator().manual_seed(rows * 7 + n + seed)
    dy = torch.randn(n, dim, generator=g).to(DTYPES[dtype])
    ids = _ids(n, rows, kind, g)
    start = torch.randn(rows, dim, generator=g).to(DTYPES[table_dtype])
    there = (ids >= 0) & (ids < rows)
    total = torch.zeros(rows, dim, dtype=torch.float64).index_add_(0, ids[there], dy[there].double())
    size = torch.zeros(rows, dim, dtype=torch.float64).index_add_(0, ids[there], dy[there].double().abs())
    count = torch.bincount(ids[there], minlength=rows)
    want = total * scale + (start.double() if accumulate else 0)
    # a sum of c values takes at most c - 1 roundings in 32 bits, each within F32 of a partial sum
    # (<= the sum of sizes); then the scale, the addition to the table, one rounding to its type
    tol = scale * size * F32 * (count[:, None] + 1) * 1.01 + want.abs() * (HALF[table_dtype] + F32) * 1.01 + TINY[table_dtype]
    if accumulate:
        tol = tol + (start.double().abs() + scale * size) * F32
        tol[count == 0] = 0
        want[count == 0] = start[count == 0].double()
    return dy, ids, start, want, tol


def _grad(dy, ids, start, dtype, table_dtype, accumulate, scale=1.5):
    n, dim = dy.shape
    rows = start.shape[0]
    buf = to_buffer(start) if accumulate else out_buffer(start.shape, start.dtype)
    rv.embedding_backward_device(to_buffer(dy), to_buffer(ids), n, rows, dim, buf, scale=scale, dtype=dtype,
                                 table_dtype=table_dtype, accumulate=accumulate)
    return from_buffer(buf, start.shape, start.dtype)


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("dtype,table_dtype", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16")])
@pytest.mark.parametrize("rows,dim,n,kind", [
    (1, 1, 1, "uniform"), (9, 5, 40, "absent"), (100, 130, 1024, "zipf"), (33, 512, 700, "same"),
    (100, 70, 1025, "uniform"), (3000, 129, 5000, "zipf"), (2048, 64, 3001, "absent"), (2047, 16, 3001, "uniform"),
    (17, 768, 9000, "same"), (5_000_000, 4, 4100, "zipf"), (5, 33, 70001, "uniform")])
def test_gradient(dtype, table_dtype, rows, dim, n, kind, accumulate):
    dy, ids, start, want, tol = _grad_case(dtype, table_dtype, rows, dim, n, kind, accumulate)
    got = _grad(dy, ids, start, dtype, table_dtype, accumulate)
    assert_within(got, want, tol)
    again = _grad(dy, ids, start, dtype, table_dtype, accumulate)
    assert torch.equal(got.view(torch.uint8), again.view(torch.uint8))


@pytest.mark.parametrize("length", [1, 2, 57, 58, 59, 61, 62, 63, 64, 65, 126, 127, 128, 129, 4096, 4097, 8500])
@pytest.mark.parametrize("before", [0, 1, 2, 62, 63, 64])
def test_gradient_runs_at_every_edge(length, before):
    """A run of one id that starts `before` entries into the sorted order, between runs of others."""
    rows, dim = 9, 5
    ids = torch.cat([torch.zeros(before, dtype=torch.int64), torch.full((length,), 3), torch.full((70,), 4),
                     torch.full((63,), 5), torch.arange(900) % 3 + 6])
    g = torch.Generator().manual_seed(length)
    ids = torch.cat([ids, torch.full((max(0, 1100 - len(ids)),), 8)])[torch.randperm(max(1100, len(ids)), generator=g)]
    # whole numbers: every sum is exact in 32 bits
    dy = torch.randint(-8, 9, (len(ids), dim), generator=g).float()
    want = torch.zeros(rows, dim).index_add_(0, ids, dy)
    assert torch.equal(_grad(dy, ids, torch.zeros(rows, dim), "f32", "f32", False, scale=1.0), want)
    assert torch.equal(_grad(dy, ids, torch.ones(rows, dim), "f32", "f32", True, scale=1.0), want + 1)


def test_gradient_without_positions():
    start = torch.randn(5, 6)
    assert torch.equal(_grad(torch.empty(0, 6), torch.empty(0, dtype=torch.int64), start, "f32", "f32", True), start)
    assert not _grad(torch.empty(0, 6), torch.empty(0, dtype=torch.int64), start, "f32", "f32", False).any()


def test_gradient_leaves_what_lies_behind_the_table():
    dy, ids = torch.randn(2000, 24), torch.randint(0, 10, (2000,))
    buf = out_buffer((12, 24), torch.float32, fill=0x55)
    rv.embedding_backward_device(to_buffer(dy), to_buffer(ids), 2000, 10, 24, buf)
    assert (from_buffer(buf, (12, 24), torch.float32)[10:].contiguous().view(torch.uint8) == 0x55).all()


def test_gradient_is_the_forward_pass_differentiated():
    """The forward pass is linear in the table: <dy, forward(t + d) - forward(t)> = <gradient, d>."""
    g = torch.Generator().manual_seed(3)
    rows, dim, n, scale = 300, 48, 2500, 0.5
    ids = torch.randint(0, rows, (n,), generator=g)
    t, d = torch.randn(rows, dim, generator=g), torch.randn(rows, dim, generator=g)
    dy = torch.randn(n, dim, generator=g)

    def forward(x):
        out = out_buffer((n, dim), torch.float32)
        rv.embedding_forward_device(to_buffer(x), rows, dim, to_buffer(ids), n, out, scale=scale)
        return from_buffer(out, (n, dim), torch.float32).double()
    grad = _grad(dy, ids, t, "f32", "f32", False, scale).double()
    left = (dy.double() * (forward(t + d) - forward(t))).sum()
    right = (grad * d.double()).sum()
    # roundings of t + d, of both forward passes (<= 3 F32 of |t| + |d| each) and of the gradient (31 F32 of its terms)
    size = scale * (dy.double().abs() * (t.double().abs() + d.double().abs())[ids]).sum()
    assert (left - right).abs() <= 40 * F32 * size


def test_refusals():
    t, ids, out = rv.Buffer(64 * 4), rv.Buffer(8 * 8), rv.Buffer(8 * 8 * 4)
    rv.embedding_forward_device(t, 8, 8, ids, 8, out)
    for bad in (dict(scale=math.inf), dict(scale=math.nan), dict(dim=2 ** 32 + 8), dict(rows=9), dict(dim=9), dict(n=9), dict(dtype="f64"), dict(dim=0), dict(rows=0), dict(n=-1),
                dict(out=t), dict(out=ids)):
        a = dict(dict(rows=8, dim=8, n=8, out=out, dtype="f32", scale=1.0), **bad)
        with pytest.raises(rv.RvxError):
            rv.embedding_forward_device(t, a["rows"], a["dim"], ids, a["n"], a["out"], dtype=a["dtype"], scale=a["scale"])
        with pytest.raises(rv.RvxError):
            rv.embedding_backward_device(t, ids, a["n"], a["rows"], a["dim"], t if a["out"] is t else a["out"], dtype=a["dtype"],
                                         scale=a["scale"])


# torch brings its own HIP runtime: it has to be loaded before librvx for the two to share the GPU
INTEROP = """
import gc
import torch
import ruvector_amd as rv
b = rv.Buffer.from_numpy(torch.arange(12, dtype=torch.float32).numpy())
assert b.__dlpack_device__()[0] == 10
v = torch.from_dlpack(b).view(torch.float32)
assert v.is_cuda and v.data_ptr() % 256 == 0 and torch.equal(v.cpu(), torch.arange(12, dtype=torch.float32))
side = torch.cuda.Stream()
rows, dim, n = 5000, 256, 20000
table, ids, out = rv.Buffer(rows * dim * 4), rv.Buffer(n * 8), rv.Buffer(n * dim * 4)
t = torch.from_dlpack(table).view(torch.float32).view(rows, dim)
i = torch.from_dlpack(ids).view(torch.int64)
o = torch.from_dlpack(out).view(torch.float32).view(n, dim)
torch.cuda.synchronize()
for step in range(3):
    # written on another stream, used by the library, read on that stream: ordered on the GPU alone
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        t.copy_(torch.randn(rows, dim, device="cuda"))
        i.copy_(torch.randint(0, rows, (n,), device="cuda"))
        rv.stream_wait(side.cuda_stream)
        rv.embedding_forward_device(table, rows, dim, ids, n, out, scale=2.0)
        rv.stream_signal(side.cuda_stream)
        assert torch.equal(o, t[i] * 2), step
graph, seven = torch.cuda.CUDAGraph(), torch.zeros(4, device="cuda")
with torch.cuda.graph(graph):
    seven += 7
    for order in (rv.stream_wait, rv.stream_signal):
        try:
            order(torch.cuda.current_stream().cuda_stream)
            raise SystemExit("a stream being captured was taken")
        except rv.RvxError as e:
            assert "captured" in str(e), e
graph.replay()                              # the capture went on undisturbed
graph.replay()
assert seven.tolist() == [14.0] * 4
b.free()
del b
gc.collect()
assert v.cpu()[3] == 3                      # the view keeps the memory
big = rv.Buffer(1 << 30)
w = torch.from_dlpack(big)
taken = torch.cuda.mem_get_info()[0]
del w                                       # the Buffer keeps it
assert torch.cuda.mem_get_info()[0] < taken + (1 << 29)
c = big.__dlpack__(stream=-1)               # a capsule nobody takes
big.free()
assert torch.cuda.mem_get_info()[0] < taken + (1 << 29)
del c
assert torch.cuda.mem_get_info()[0] >= taken + (1 << 29)
late = table.__dlpack__(stream=-1)          # this, and the views above, go with the interpreter
print("interop ok", flush=True)
"""


def test_dlpack_views_and_stream_order():
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-u", "-c", INTEROP], cwd=root, capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and "interop ok" in r.stdout, r.stdout + r.stderr


def test_offsets_past_32_bits():
    """A table of more than 2^31 elements: rows at its end, forward, and their gradient."""
    rows, dim = 2 ** 21 + 5, 1024
    table = rv.Buffer(rows * dim * 4)
    table.fill_uniform(rows * dim, 3)
    ids = torch.tensor([rows - 1, 0, rows - 2, rows, rows - 1, 2 ** 21], dtype=torch.int64)
    out = out_buffer((6, dim), torch.float32)
    rv.embedding_forward_device(table, rows, dim, to_buffer(ids), 6, out)
    want = torch.from_numpy(table.gather_rows(rows, dim, ids.clamp(0, rows - 1).numpy())).clone()
    want[3] = 0
    assert torch.equal(from_buffer(out, (6, dim), torch.float32), want)
    for n in (6, 1500):  # both ways of grouping
        many = ids.repeat(n // 6)
        g = torch.randint(-3, 4, (n, dim)).float()
        before = torch.from_numpy(table.gather_rows(rows, dim, [rows - 1, 2 ** 21, rows - 3]))
        rv.embedding_backward_device(to_buffer(g), to_buffer(many), n, rows, dim, table, accumulate=True)
        after = torch.from_numpy(table.gather_rows(rows, dim, [rows - 1, 2 ** 21, rows - 3]))
        assert_within(after[0], before[0].double() + g[many == rows - 1].double().sum(0), (after[0].abs() + 1).double() * F32)
        assert_within(after[1], before[1].double() + g[many == 2 ** 21].double().sum(0), (after[1].abs() + 1).double() * F32)
        assert torch.equal(after[2], before[2])


def test_calls_from_several_threads():
    import threading
    cases = [_grad_case("f32", "f32", 200 + t, 64, 3000 + 500 * t, "zipf", False, seed=t) for t in range(4)]
    fails = []

    def work(case):
        dy, ids, start, want, tol = case
        try:
            for _ in range(5):
                assert_within(_grad(dy, ids, start, "f32", "f32", False), want, tol)
        except Exception as e:  # noqa: BLE001
            fails.append(e)
    threads = [threading.Thread(target=work, args=(c,)) for c in cases]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not fails, fails
