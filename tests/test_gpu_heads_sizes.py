"""The typed operators at the sizes where they take their other forms: sorts of several passes, rows of
several vectors a lane and several slabs, a wave a row over many steps, long sums, launches in slices."""
import math

import pytest
import torch

rv = pytest.importorskip("ruvector_amd")
from heads_ref import DTYPES, assert_within, from_buffer, out_buffer, to_buffer  # noqa: E402
import test_gpu_adapters as adapters  # noqa: E402
import test_gpu_embedding as embedding  # noqa: E402
import test_gpu_logprobs as logprobs  # noqa: E402

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- the table's gradient
@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("dtype,table_dtype", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16")])
@pytest.mark.parametrize("rows,dim,n,kind", [
    # more positions than one block sorts: digits of 12 to 14 bits (two passes), 17 (two), 23 (three); short runs
    # in rows of one vector a lane to four, and of two slabs; many rows without an id
    (3000, 300, 7000, "uniform"), (5000, 767, 8000, "zipf"), (2500, 1024, 9001, "uniform"), (4100, 1500, 6500, "zipf"),
    (2100, 2100, 7001, "absent"), (2600, 4200, 6145, "uniform"), (70000, 64, 20000, "uniform"), (70000, 33, 30011, "absent"),
    (4_300_000, 5, 30011, "uniform"), (9000, 520, 6144, "uniform"), (9000, 520, 1100, "zipf"), (20000, 130, 150_001, "zipf")])
def test_table_gradient(dtype, table_dtype, rows, dim, n, kind, accumulate):
    dy, ids, start, want, tol = embedding._grad_case(dtype, table_dtype, rows, dim, n, kind, accumulate)
    got = embedding._grad(dy, ids, start, dtype, table_dtype, accumulate)
    assert_within(got, want, tol)
    again = embedding._grad(dy, ids, start, dtype, table_dtype, accumulate)
    assert torch.equal(got.view(torch.uint8), again.view(torch.uint8))


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("rows", [1000, 100_000])
def test_table_gradient_of_more_than_one_launch(rows, accumulate):
    """2^24 positions a launch; whole numbers, so that every sum is exact."""
    n, dim = 2 ** 24 + 3001, 2
    g = torch.Generator().manual_seed(rows)
    ids = torch.randint(-1, rows, (n,), generator=g)
    dy = torch.randint(-8, 9, (n, dim), generator=g).float()
    there = ids >= 0
    want = torch.zeros(rows, dim, dtype=torch.float64).index_add_(0, ids[there], dy[there].double()) + accumulate
    assert torch.equal(embedding._grad(dy, ids, torch.ones(rows, dim), "f32", "f32", accumulate, scale=1.0).double(), want)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,dim,n", [(70000, 300, 20011), (5000, 4200, 3001), (300_000, 7, 100_003)])
def test_many_rows_by_id(dtype, rows, dim, n):
    g = torch.Generator().manual_seed(n)
    table = torch.randn(rows, dim, generator=g).to(DTYPES[dtype])
    ids = embedding._ids(n, rows, "absent", g)
    out = out_buffer((n + 1, dim), DTYPES[dtype])
    rv.embedding_forward_device(to_buffer(table), rows, dim, to_buffer(ids), n, out, dtype=dtype)
    got = from_buffer(out, (n + 1, dim), DTYPES[dtype])
    there = (ids >= 0) & (ids < rows)
    want = torch.where(there[:, None], table[ids.clamp(0, rows - 1)], torch.zeros((), dtype=DTYPES[dtype]))
    assert torch.equal(got[:n], want) and (got[n:].contiguous().view(torch.uint8) == 0x7b).all()


# ---------------------------------------------------------------- log probabilities: a wave a row
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,c,k,temperature", [
    (2100, 1500, 0, 1.0), (2100, 1500, 5, 0.07), (2503, 3001, 10, 1.0), (2048, 1025, 64, 2.0), (2049, 4097, 1, 0.7)])
def test_many_rows_of_many_steps(dtype, n, c, k, temperature):
    scores, targets = logprobs.make(n, c, dtype)
    targets[::4] = scores[::4].float().argmax(1)
    targets[1], targets[2] = -1, c
    logprobs.check(scores, targets, temperature, k, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("part", [0.1, 0.9])
@pytest.mark.parametrize("k", [0, 6, 40])
def test_many_rows_with_masks(dtype, part, k):
    n, c = 2200, 2100
    scores, targets = logprobs.make(n, c, dtype, seed=3)
    g = torch.Generator().manual_seed(2)
    scores.masked_fill_(torch.rand(n, c, generator=g) < part, -math.inf)
    scores[0] = scores[n // 2] = scores[n - 1] = -math.inf
    scores[1] = -math.inf
    scores[1, c - 1] = 2.0
    scores[2] = torch.finfo(DTYPES[dtype]).min
    scores[3, : c // 2] = torch.finfo(DTYPES[dtype]).min
    logprobs.check(scores, targets, 1.0, k, dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", ["equal", "up", "down", "two"])
@pytest.mark.parametrize("k", [5, 64])
def test_many_rows_in_order(dtype, shape, k):
    n, c = 2048, 2500
    base = dict(equal=torch.full((c,), 1.5), up=torch.arange(c) * 1e-3, down=-torch.arange(c) * 1e-3,
                two=(torch.arange(c) % 7 == 0) * 2.0)[shape]
    scores = base.float().expand(n, c).to(DTYPES[dtype]).contiguous()
    logprobs.check(scores, torch.arange(n) % c, 1.0, k, dtype)


@pytest.mark.parametrize("scale,temperature", [(1e8, 1.0), (3e38, 1.0), (3e38, 1e30), (1.0, 1e-7)])
def test_many_rows_of_any_size(scale, temperature):
    """Against the same rows a few at a time, whose values are held against 64 bits elsewhere."""
    n, c = 2060, 1300
    scores, targets = logprobs.make(n, c, "f32", spread=1.0)
    scores = (scores.clamp(-1, 1) * scale).float()
    scores[1, ::2] = -math.inf
    got = logprobs.forward(scores, targets, temperature, 7, "f32")
    want, _ = logprobs.reference(scores, targets, temperature, 7)
    assert torch.equal(got["top_ids"], want["top_ids"]) and torch.equal(got["rank"], want["rank"])
    assert_within(got["stats"][:, 0], want["stats"][:, 0], 0.0)
    _, s_err = logprobs.tolerances(scores, 1.0)
    row = s_err + 3 * 2.0 ** -24 * 40  # as there: what is over 40 below the best adds nothing
    assert_within(got["stats"][:, 1], want["stats"][:, 1], row)
    # log p may be -6e38 here: past 2^128 - 2^103 the nearest 32-bit number is an infinity
    logp = torch.where(want["logp"].float().isinf(), -math.inf, want["logp"])
    assert_within(got["logp"], logp, row + 4 * 2.0 ** -24 * logp.abs().nan_to_num(0, 0, 0))


def test_nan_and_infinities_among_many_rows():
    scores, targets = logprobs.make(2100, 1500, "f32")
    clean = logprobs.forward(scores, targets, 1.0, 4, "f32")
    scores[5, 700], scores[9, 1499], scores[2099, :] = math.nan, math.inf, math.nan
    got = logprobs.forward(scores, targets, 1.0, 4, "f32")
    keep = torch.ones(2100, dtype=torch.bool)
    keep[[5, 9, 2099]] = False
    for name in got:
        assert torch.equal(got[name][keep], clean[name][keep]), name
    for r in (5, 9, 2099):
        assert got["logp"][r].isnan() and got["entropy"][r].isnan() and got["stats"][r, 1].isnan()
    assert 700 not in got["top_ids"][5] and got["top_ids"][9, 0] == 1499 and (got["top_ids"][2099] == -1).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_log_probs_of_more_than_one_launch(dtype):
    """More rows than a launch takes (2^23; the gradient 2^25): the same rows over and over have the same results."""
    n, c, few = 2 ** 25 + 1009, 2, 1009
    scores, targets = logprobs.make(few, c, dtype)
    targets[::5] = -1
    gl = torch.randn(few, generator=torch.Generator().manual_seed(1))
    small = logprobs.forward(scores, targets, 0.5, 1, dtype)
    grad = logprobs.backward(scores, targets, 0.5, gl, None, dtype)
    over = lambda t: t.repeat((n + few - 1) // few, *[1] * (t.dim() - 1))[:n]  # noqa: E731
    big = logprobs.forward(over(scores), over(targets), 0.5, 1, dtype)
    for name in small:
        assert torch.equal(big[name], over(small[name])), name
    assert torch.equal(logprobs.backward(over(scores), over(targets), 0.5, over(gl), None, dtype), over(grad))


# ---------------------------------------------------------------- adapters: long sums
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("inp,out,n,ranks,max_rank", [
    (4096, 300, 1, [8, 16], 16), (4100, 200, 50, [64, 3], 64), (2050, 260, 70, [16, 0, 5], 16), (8192, 130, 200, [128, 9], 128),
    (1025, 520, 1100, [24] * 3, 24), (3001, 2100, 2300, [16, 40], 40), (65536, 40, 66, [4], 4), (65536, 20, 9, [33], 33),
    (40, 65536, 70, [16], 16)])
def test_adapters_with_long_sums(dtype, inp, out, n, ranks, max_rank):
    m = adapters.make(inp, out, n, ranks, dtype, bias=True)
    layer = adapters.layer_of(m, max_rank, dtype)
    for ids in (m["ids"], None):
        got = adapters.run(layer, m["x"], ids)
        want, tol = adapters.reference(m, ids, dtype)
        assert_within(got, want, tol)
        assert torch.equal(adapters.run(layer, m["x"], ids), got)


@pytest.mark.parametrize("n,c", [(3, 40), (3, 9000), (2100, 1500)])
def test_rank_of_a_nan(n, c):
    """A NaN counts before no target, and no score before a target that is NaN."""
    scores, targets = logprobs.make(n, c, "f32")
    targets[:] = c // 2
    clean = logprobs.forward(scores, targets, 1.0, 0, "f32")
    scores[0, c // 2] = math.nan
    scores[1, c - 1] = math.nan
    before = int(clean["rank"][1]) - int((logprobs.make(n, c, "f32")[0][1, c - 1] > scores[1, c // 2]))
    got = logprobs.forward(scores, targets, 1.0, 0, "f32")
    assert got["rank"][0] == 0 and got["logp"][0].isnan()
    assert got["rank"][1] == before and torch.equal(got["rank"][2:], clean["rank"][2:])
