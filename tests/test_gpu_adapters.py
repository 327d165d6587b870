"""AdapterLinear against the formula in 64 bits, and one pass through all the typed operators."""
import math

import numpy as np
import pytest
import torch

rv = pytest.importorskip("ruvector_amd")
from heads_ref import DTYPES, F32, HALF, TINY, assert_within, from_buffer, out_buffer, to_buffer  # noqa: E402

pytestmark = pytest.mark.gpu


def make(inp, out, n, ranks, dtype, bias=False, seed=0):
    """Weights, adapters of the given ranks (0 = a slot that is never set) and rows."""
    g = torch.Generator().manual_seed(seed + inp * 131 + out * 17 + n)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    T = DTYPES[dtype]
    m = dict(w=(r(out, inp) * inp ** -0.5).to(T), bias=r(out).to(T) if bias else None, x=r(n, inp).to(T),
             adapters=[((r(k, inp) * inp ** -0.5).to(T), r(out, k).to(T), 0.5 + s * 0.25) for s, k in enumerate(ranks)])
    m["ids"] = torch.randint(-1, len(ranks) + 1, (n,), generator=g).to(torch.int32)
    return m


def layer_of(m, max_rank, dtype):
    out, inp = m["w"].shape
    layer = rv.AdapterLinear(inp, out, to_buffer(m["w"]), bias=None if m["bias"] is None else to_buffer(m["bias"]),
                             max_rank=max_rank, max_adapters=len(m["adapters"]), dtype=dtype)
    for s, (a, b, scale) in enumerate(m["adapters"]):
        if a.shape[0]:
            layer.set_adapter(s, a.shape[0], to_buffer(a), to_buffer(b), scale)
    return layer


def run(layer, x, ids):
    n = x.shape[0]
    y = out_buffer((n + 1, layer.out_features), x.dtype)
    layer.forward_device(to_buffer(x), n, y, adapter_ids=None if ids is None else to_buffer(ids))
    got = from_buffer(y, (n + 1, layer.out_features), x.dtype)
    assert (got[n:].contiguous().view(torch.uint8) == 0x7b).all()  # the row behind the last one
    return got[:n]


def reference(m, ids, dtype):
    """y and how far it may be off."""
    x, w = m["x"].double(), m["w"].double()
    inp = x.shape[1]
    y, size = x @ w.T, x.abs() @ w.abs().T
    if m["bias"] is not None:
        y, size = y + m["bias"].double(), size + m["bias"].double().abs()
    # sums of `in` exact products in 32 bits, in any order: at most in - 1 roundings of partial sums
    tol = size * F32 * (inp + 4)
    for s, (a, b, scale) in enumerate(m["adapters"]):
        at = torch.nonzero(ids == s)[:, 0] if ids is not None else torch.empty(0, dtype=torch.long)
        if not len(at) or not a.shape[0]:
            continue
        a, b = a.double(), b.double()
        t, ts = scale * (x[at] @ a.T), scale * (x[at].abs() @ a.abs().T)
        y[at] += t @ b.T
        # t: the sum's roundings and the scale's; then t as two pieces of the type: 2^-17 (bf16), 2^-21 (f16)
        # of it, and the sum over the rank
        piece = dict(f32=0.0, bf16=2.0 ** -17, f16=2.0 ** -21)[dtype]
        tol[at] += (ts * F32 * (inp + 2) + t.abs() * piece) @ b.abs().T + (t.abs() @ b.abs().T) * F32 * (a.shape[0] + 4)
        if dtype == "f16":  # the row's largest |t| is scaled to [2^14, 2^15): pieces are off by 2^-25 steps of that
            tol[at] += t.abs().amax(1, keepdim=True) * 2.0 ** -38 * b.abs().sum(1)
    return y, tol * 1.01 + y.abs() * HALF[dtype] * 1.01 + TINY[dtype]


SHAPES = [  # in, out, n, ranks, max_rank
    (1, 1, 1, [1], 1), (64, 16, 1, [8, 4], 8), (768, 768, 1, [8], 8), (65, 33, 3, [3, 0, 16], 16), (128, 100, 16, [16, 1], 16),
    (127, 17, 17, [5], 8), (256, 272, 33, [32, 7, 20], 32), (512, 64, 64, [64, 3], 64), (96, 48, 65, [16, 0, 2], 16),
    (64, 130, 200, [128, 1], 128), (200, 257, 129, [24], 24), (320, 1000, 700, [8, 16, 33], 64), (192, 4100, 1100, [16] * 5, 16),
    (70, 300, 5000, [4, 12], 12)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("inp,out,n,ranks,max_rank", SHAPES)
def test_forward(dtype, inp, out, n, ranks, max_rank):
    m = make(inp, out, n, ranks, dtype, bias=n % 2 == 1)
    layer = layer_of(m, max_rank, dtype)
    for ids in (m["ids"], torch.sort(m["ids"]).values, None):
        got = run(layer, m["x"], ids)
        want, tol = reference(m, ids, dtype)
        assert_within(got, want, tol, f"ids {'none' if ids is None else 'given'}")
        assert torch.equal(run(layer, m["x"], ids), got)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_large_tiles(dtype):
    """Rounds of large tiles with edges, requests of many rows."""
    m = make(64, 4200, 4200, [16, 4, 9], dtype)
    layer = layer_of(m, 16, dtype)
    ids = torch.repeat_interleave(torch.tensor([0, -1, 2, 1, 3, 0, 2]), 600).to(torch.int32)  # requests of 600 rows
    got = run(layer, m["x"], ids)
    want, tol = reference(m, ids, dtype)
    assert_within(got, want, tol)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,out", [(4000, 4090), (1800, 4001), (1001, 4000), (3000, 2100)])
@pytest.mark.parametrize("inp", [40, 200, 300])
def test_every_tile(dtype, n, out, inp):
    """Row and output counts of each of the tiles' sizes; sums of fewer stages than are in flight, and more."""
    m = make(inp, out, n, [16, 40], dtype, bias=True)
    got = run(layer_of(m, 40, dtype), m["x"], m["ids"])
    want, tol = reference(m, m["ids"], dtype)
    assert_within(got, want, tol)


@pytest.mark.parametrize("n", [5, 300])
def test_rows_do_not_depend_on_each_other(n):
    """An adapter, or a row, with infinities and NaN changes its own rows alone."""
    m = make(128, 96, n, [8, 8], "bf16")
    ids = (torch.arange(n) % 2).to(torch.int32)
    clean = run(layer_of(m, 8, "bf16"), m["x"], ids)
    bad = dict(m, adapters=[m["adapters"][0], (m["adapters"][1][0] * math.inf, m["adapters"][1][1] * math.nan, 1.0)])
    got = run(layer_of(bad, 8, "bf16"), m["x"], ids)
    assert torch.equal(got[0::2], clean[0::2]) and not torch.isfinite(got[1::2]).any()
    x = m["x"].clone()
    x[n // 2] = math.nan
    got = run(layer_of(m, 8, "bf16"), x, ids)
    assert got[n // 2].isnan().all()
    keep = torch.arange(n) != n // 2
    assert torch.equal(got[keep], clean[keep])


@pytest.mark.parametrize("n", [4, 100])
def test_f16_intermediate_past_the_type(n):
    """t = A x may be larger than f16 holds while y is not."""
    inp, out = 64, 32
    x, a = torch.full((n, inp), 100.0).half(), torch.full((4, inp), 60.0).half()
    b = torch.zeros(out, 4).half()
    b[:, 0], b[:, 1] = 2.0 ** -10, -(2.0 ** -11)
    m = dict(w=torch.zeros(out, inp).half(), bias=None, x=x, adapters=[(a, b, 1.0)])
    ids = torch.zeros(n, dtype=torch.int32)
    want, tol = reference(m, ids, "f16")   # 384000 (2^-10 - 2^-11)
    assert_within(run(layer_of(m, 4, "f16"), x, ids), want, tol)


@pytest.mark.parametrize("n", [7, 200])
@pytest.mark.parametrize("size", [1e-30, 1e-18, 1e18, 1e30])
def test_f32_of_any_size(n, size):
    """Rows and weights of one size whose products stay in range; elsewhere exact zeros."""
    inp, out = 80, 50
    m = make(inp, out, n, [], "f32")
    m["x"][:, 40:] = 0
    m["x"] = m["x"].clamp(-1, 1) * size
    m["w"] = m["w"].clamp(-1, 1) / size
    m["w"][::2, :40] = 0                       # these outputs are 0: what they weigh is 0 in x
    m["w"][::2, 40:] = torch.tensor(size).clamp(max=1e30)
    got = run(layer_of(m, 8, "f32"), m["x"], None)
    want, tol = reference(m, None, "f32")
    assert (got[:, ::2] == 0).all()
    # as halves: a product is off by 3 2^-22 of the two rows' largest values, 40 of them
    most = m["x"].double().abs().amax(1)[:, None] * m["w"].double().abs().amax(1)
    assert_within(got[:, 1::2], want[:, 1::2], (tol + 40 * 3 * 2.0 ** -22 * most)[:, 1::2])


@pytest.mark.parametrize("n", [7, 200])
def test_bf16_intermediate_infinite(n):
    """A x past the largest float is infinite, and so is y, with B's sign."""
    m = make(64, 40, n, [1], "bf16")
    a, b, scale = m["adapters"][0]
    m["adapters"] = [((a.abs() + 0.1) * 1e30, b.sign() + 0.5, scale)]
    m["x"] = (m["x"].abs() + 0.1) * 1e30
    m["w"] *= 0
    m["ids"][:] = 0
    got = run(layer_of(m, 1, "bf16"), m["x"], m["ids"]).float()
    assert torch.equal(got, (math.inf * m["adapters"][0][1].float().T).expand(n, -1))


def test_adapters_replaced_and_cleared():
    m = make(96, 80, 70, [8, 8], "f32")
    layer = layer_of(m, 8, "f32")
    ids = (torch.arange(70) % 3 - 1).to(torch.int32)
    layer.clear_adapter(0)
    gone = dict(m, adapters=[(m["adapters"][0][0][:0], m["adapters"][0][1][:, :0], 1.0), m["adapters"][1]])
    want, tol = reference(gone, ids, "f32")
    assert_within(run(layer, m["x"], ids), want, tol)
    a, b = torch.randn(3, 96), torch.randn(80, 3)
    layer.set_adapter(1, 3, to_buffer(a), to_buffer(b), -2.0)  # a smaller rank in the place of a larger one
    new = dict(gone, adapters=[gone["adapters"][0], (a, b, -2.0)])
    want, tol = reference(new, ids, "f32")
    tol = tol.abs() + 0
    ref = m["x"].double() @ m["w"].double().T
    at = ids == 1
    ref[at] += -2.0 * (m["x"][at].double() @ a.double().T) @ b.double().T
    assert (want - ref).abs().max() < 1e-12
    size = m["x"].double().abs() @ m["w"].double().abs().T
    size[at] += 2.0 * (m["x"][at].double().abs() @ a.double().abs().T) @ b.double().abs().T
    assert_within(run(layer, m["x"], ids), ref, size * F32 * 110)  # at most 96 + 3 + scale, sum, addition


def test_ids_outside_the_slots():
    m = make(64, 64, 9, [4], "f32")
    layer = layer_of(m, 4, "f32")
    ids = torch.tensor([0, 1, -1, 2 ** 31 - 1, -2 ** 31, 0, 5, -7, 0], dtype=torch.int32)
    want, tol = reference(m, ids, "f32")
    assert_within(run(layer, m["x"], ids), want, tol)
    none = rv.AdapterLinear(64, 64, to_buffer(m["w"]), max_adapters=0)
    want, tol = reference(m, None, "f32")
    assert_within(run(none, m["x"], ids), want, tol)


def test_refusals():
    w = rv.Buffer(32 * 64 * 4)
    for bad in (dict(in_features=0), dict(out_features=65537), dict(max_rank=129), dict(max_rank=0), dict(max_adapters=-1),
                dict(in_features=65), dict(dtype="f8"), dict(bias=rv.Buffer(4))):
        a = dict(dict(in_features=64, out_features=32, weight=w), **bad)
        with pytest.raises(rv.RvxError):
            rv.AdapterLinear(**a)
    layer = rv.AdapterLinear(64, 32, w, max_rank=8, max_adapters=2)
    a, b = rv.Buffer(8 * 64 * 4), rv.Buffer(32 * 8 * 4)
    layer.set_adapter(1, 8, a, b)
    for slot, rank, scale in ((2, 8, 1.0), (-1, 8, 1.0), (0, 9, 1.0), (0, -1, 1.0), (0, 8, math.nan)):
        with pytest.raises(rv.RvxError):
            layer.set_adapter(slot, rank, a, b, scale)
    with pytest.raises(rv.RvxError):
        layer.set_adapter(0, 8, rv.Buffer(16), b)
    x, y, ids = rv.Buffer(4 * 64 * 4), rv.Buffer(4 * 32 * 4), rv.Buffer(4 * 4)
    layer.forward_device(x, 4, y, adapter_ids=ids)
    layer.forward_device(x, 0, y)
    for n, xx, yy, ii in ((5, x, y, ids), (4, x, x, ids), (4, y, y, ids), (-1, x, y, ids), (4, x, ids, ids), (4, x, rv.Buffer(8), ids),
                          (4, x, y, rv.Buffer(8))):
        with pytest.raises(rv.RvxError):
            layer.forward_device(xx, n, yy, adapter_ids=ii)


def test_a_query_tower_end_to_end():
    """Embedding rows -> the tenant's adapter -> scores against a table -> log probabilities, and
    back: the gradient of the loss by the scores and by the embeddings' table, against 64 bits."""
    g = torch.Generator().manual_seed(11)
    rows, dim, items, n, T = 400, 96, 700, 300, 0.5
    table, proj, corpus = (torch.randn(*s, generator=g) for s in ((rows, dim), (dim, dim), (items, dim)))
    proj, corpus = proj * dim ** -0.5, corpus * dim ** -0.5
    a, b = torch.randn(4, dim, generator=g) * dim ** -0.5, torch.randn(dim, 4, generator=g) * 0.5
    ids = torch.randint(0, rows, (n,), generator=g)
    tenants = torch.randint(-1, 1, (n,), generator=g).to(torch.int32)
    targets = torch.randint(0, items, (n,), generator=g)

    h, q, s, grad, ds = (rv.Buffer(n * d * 4) for d in (dim, dim, items, dim, items))
    stats, logp, dlogp, back = rv.Buffer(n * 8), rv.Buffer(n * 4), to_buffer(torch.full((n,), -1.0 / n)), rv.Buffer(rows * dim * 4)
    idb, tb = to_buffer(ids), to_buffer(targets)
    tower = rv.AdapterLinear(dim, dim, to_buffer(proj), max_rank=4, max_adapters=1)
    tower.set_adapter(0, 4, to_buffer(a), to_buffer(b), 1.5)
    scorer = rv.AdapterLinear(dim, items, to_buffer(corpus), max_adapters=0)
    by_query = rv.AdapterLinear(items, dim, to_buffer(corpus.T.contiguous()), max_adapters=0)     # dq = ds corpus
    by_row = rv.AdapterLinear(dim, dim, to_buffer(proj.T.contiguous()), max_rank=4, max_adapters=1)  # dh = dq (W + s B A)
    by_row.set_adapter(0, 4, to_buffer(b.T.contiguous()), to_buffer(a.T.contiguous()), 1.5)
    rv.embedding_forward_device(to_buffer(table), rows, dim, idb, n, h)
    tower.forward_device(h, n, q, adapter_ids=to_buffer(tenants))
    scorer.forward_device(q, n, s)
    rv.log_probs_device(s, n, items, T, targets=tb, logp=logp, stats=stats)
    rv.log_probs_backward_device(s, n, items, T, stats, ds, targets=tb, grad_logp=dlogp)
    by_query.forward_device(ds, n, q)
    by_row.forward_device(q, n, grad, adapter_ids=to_buffer(tenants))
    rv.embedding_backward_device(grad, idb, n, rows, dim, back)

    t64 = table.double().requires_grad_()
    e = t64[ids]
    query = e @ proj.double().T + 1.5 * (tenants >= 0).double()[:, None] * ((e @ a.double().T) @ b.double().T)
    lp = torch.log_softmax(query @ corpus.double().T / T, 1)[torch.arange(n), targets]
    (-lp.mean()).backward()
    # 64-bit values against a chain of five products of <= 700 terms in 32 bits: each relative to its
    # row's size within 700 F32, and the scores' error (|s| <= ~40 units of 1) enters p by 1 / T
    assert_within(from_buffer(logp, (n,), torch.float32), lp, 700 * F32 * 40)
    got = from_buffer(back, (rows, dim), torch.float32).double()
    assert (got - t64.grad).norm() <= 5 * 700 * F32 / T * t64.grad.norm()
