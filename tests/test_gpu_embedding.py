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
    for bad in (dict(rows=9), dict(dim=9), dict(n=9), dict(dtype="f64"), dict(dim=0), dict(rows=0), dict(n=-1),
                dict(out=t), dict(out=ids)):
        a = dict(dict(rows=8, dim=8, n=8, out=out, dtype="f32"), **bad)
        with pytest.raises(rv.RvxError):
            rv.embedding_forward_device(t, a["rows"], a["dim"], ids, a["n"], a["out"], dtype=a["dtype"])
        with pytest.raises(rv.RvxError):
            rv.embedding_backward_device(t, ids, a["n"], a["rows"], a["dim"], t if a["out"] is t else a["out"], dtype=a["dtype"])


def test_dlpack_views_share_the_buffer():
    b = rv.Buffer.from_numpy(torch.arange(12, dtype=torch.float32).numpy())
    v = torch.from_dlpack(b).view(torch.float32)
    assert v.is_cuda and torch.equal(v.cpu(), torch.arange(12, dtype=torch.float32))
    v.mul_(2)
    rv.stream_wait(torch.cuda.current_stream().cuda_stream)
    assert torch.equal(from_buffer(b, (12,), torch.float32), 2 * torch.arange(12, dtype=torch.float32))
    del b
    assert v.cpu()[3] == 6
