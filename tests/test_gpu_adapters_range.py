"""AdapterLinear at the ends of the number range: results that the type holds are not lost on the
way to them, whatever the number of rows."""
import pytest
import torch

rv = pytest.importorskip("ruvector_amd")
from heads_ref import DTYPES, F32, HALF, TINY, assert_within, to_buffer  # noqa: E402
import test_gpu_adapters as adapters  # noqa: E402
from test_gpu_adapters import run  # noqa: E402

pytestmark = pytest.mark.gpu


def spread(g, *shape):
    """Values of either sign with magnitudes in [1/2, 1)."""
    v = torch.rand(*shape, generator=g) * 0.5 + 0.5
    return torch.where(torch.rand(*shape, generator=g) < 0.5, -v, v)


@pytest.mark.parametrize("n", [1, 64, 65, 200, 700])
@pytest.mark.parametrize("xe,we", [(-61, -61), (-20, -102), (-102, -20), (-58, -64), (60, 60), (100, -126), (-126, 100)])
@pytest.mark.parametrize("inp,out", [(100, 70), (4100, 40)])
def test_f32_products_near_the_ends(n, xe, we, inp, out):
    """max |x| max |W| from 2^-122 to 2^120: sums of such products are ordinary numbers."""
    g = torch.Generator().manual_seed(n * 1000 + xe + inp)
    x, w = spread(g, n, inp) * 2.0 ** xe, spread(g, out, inp) * 2.0 ** we
    layer = rv.AdapterLinear(inp, out, to_buffer(w), max_adapters=0)
    got = run(layer, x, None)
    x, w = x.double(), w.double()
    want, size = x @ w.T, x.abs() @ w.abs().T
    # sums of `in` products in 32 bits (no partial sum needs a step below the type's smallest), and each
    # product within 3 2^-22 of the two rows' largest values
    most = x.abs().amax(1)[:, None] * w.abs().amax(1)
    assert_within(got, want, size * F32 * (inp + 4) + inp * (3 * 2.0 ** -22 * most + TINY["f32"]))


def f32_forward(x, w):
    return run(rv.AdapterLinear(w.shape[1], w.shape[0], to_buffer(w), max_adapters=0), x, None)


def assert_f32(got, x, w):
    """Within what sums of `in` products in 32 bits may be off, whatever the values' sizes beside each other:
    in - 1 roundings of partial sums, 2^-24 of each product, and the last steps of the smallest numbers."""
    x, w = x.double(), w.double()
    inp = x.shape[1]
    assert_within(got, x @ w.T, (x.abs() @ w.abs().T) * F32 * (inp + 4) + inp * TINY["f32"])


@pytest.mark.parametrize("n", [1, 64, 65, 200, 700])
@pytest.mark.parametrize("inp,out", [(65, 64), (1000, 70)])
def test_f32_large_values_in_different_columns(n, inp, out):
    """What is large in x meets what is small in W: the small values of a row count in full."""
    x, w = torch.full((n, inp), 1.23 * 2.0 ** -26), torch.full((out, inp), 1.1)
    x[:, 0], w[:, 0] = 1, 2.0 ** -40
    assert_f32(f32_forward(x, w), x, w)


@pytest.mark.parametrize("n", [64, 65, 300])
@pytest.mark.parametrize("low,high", [(-5, 5), (-30, 30), (-62, 52), (-120, 0)])
def test_f32_rows_of_any_spread(n, low, high):
    """Magnitudes spread evenly over many powers of two, within a row and between rows."""
    g = torch.Generator().manual_seed(n + high)
    inp, out = 333, 90
    power = lambda *s: torch.randint(low, high + 1, s, generator=g).double()  # noqa: E731
    x = (spread(g, n, inp).double() * 2.0 ** power(n, inp)).float()
    w = (spread(g, out, inp).double() * 2.0 ** power(out, inp)).float()
    if high == 0:  # the small values of x beside the large ones of W
        x[:, ::2] = 0
        x[:, 0] = 1
        w[:, 0] = 2.0 ** -126
        w[:, 1:] = spread(g, out, inp - 1) * 2.0 ** 100
    assert_f32(f32_forward(x, w), x, w)


@pytest.mark.parametrize("n", [64, 65, 200])
@pytest.mark.parametrize("xe,we", [(-61, -61), (-20, -102), (60, 60), (100, -126), (-126, 100), (0, 0)])
def test_f32_as_exact_as_32_bits(n, xe, we):
    g = torch.Generator().manual_seed(n - xe)
    x, w = spread(g, n, 100) * 2.0 ** xe, spread(g, 70, 100) * 2.0 ** we
    assert_f32(f32_forward(x, w), x, w)


@pytest.mark.parametrize("n", [5, 100])
def test_f32_infinities_stay_in_their_rows(n):
    """A row with an infinity or a NaN is not finite; the others, and its own scale, are as without."""
    g = torch.Generator().manual_seed(n)
    x, w = spread(g, n, 80), spread(g, 50, 80) * 1e-20
    clean = f32_forward(x, w)
    x[2, 7], x[4, 9] = torch.inf, torch.nan
    got = f32_forward(x, w)
    keep = torch.ones(n, dtype=torch.bool)
    keep[[2, 4]] = False
    assert torch.equal(got[keep], clean[keep]) and not torch.isfinite(got[[2, 4]]).any() and got[4].isnan().all()


def adapted(x, a, b, dtype):
    """b (a x) alone: a layer with weights of zero and one adapter."""
    n, inp = x.shape
    layer = rv.AdapterLinear(inp, b.shape[0], to_buffer(torch.zeros(b.shape[0], inp, dtype=DTYPES[dtype])), max_rank=a.shape[0],
                             max_adapters=1, dtype=dtype)
    layer.set_adapter(0, a.shape[0], to_buffer(a), to_buffer(b))
    return run(layer, x, torch.zeros(n, dtype=torch.int32))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [1, 64, 65, 300])
@pytest.mark.parametrize("rank", [2, 40, 100])
@pytest.mark.parametrize("size", [1.0, 2.0 ** -9, 2.0 ** 8])
def test_a_x_in_32_bits(dtype, n, rank, size):
    """Pairs of nearly equal A x whose difference is y: what A x loses shows."""
    g = torch.Generator().manual_seed(n + rank)
    inp, out, T = 8, 20, DTYPES[dtype]
    x = (spread(g, n, inp) * size).to(T)
    a = spread(g, rank, inp).to(T)
    a[1::2] = a[0::2]
    a[1::2, 0] += a[0::2, 0] * 2.0 ** -6
    b = spread(g, out, rank).to(T)
    b[:, 1::2] = -b[:, 0::2]
    got = adapted(x, a, b, dtype)
    x, a, b = x.double(), a.double(), b.double()
    t, ts = x @ a.T, x.abs() @ a.abs().T
    # t: a sum of `in` products, and a step of 32 bits (f16: 2^-39 of the row's largest); then the sum of the
    # products with B, each of up to three pieces, and y's rounding
    off = ts * F32 * (inp + 1)
    if dtype == "f16":
        off = off + t.abs().amax(1, keepdim=True) * 2.0 ** -39
    want = t @ b.T
    tol = off @ b.abs().T + (t.abs() @ b.abs().T) * F32 * (3 * rank + 1)
    assert_within(got, want, tol * 1.01 + want.abs() * HALF[dtype] * 1.01 + TINY[dtype])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [3, 64, 65, 200])
@pytest.mark.parametrize("first,want", [((1, -1), torch.inf), ((-1, -1), -torch.inf), ((1, 0), torch.inf), ((0, 1), torch.nan)])
def test_an_infinite_a_x_beside_a_large_one(dtype, n, first, want):
    """A x = (inf, 384000): the second is past f16, yet no infinity."""
    T = DTYPES[dtype]
    a = torch.zeros(2, 64, dtype=T)
    a[0, 0], a[1] = torch.inf, 60
    got = adapted(torch.full((n, 64), 100.0, dtype=T), a, torch.tensor([first] * 20, dtype=T), dtype)
    assert torch.equal(got.float().nan_to_num(nan=1.0, posinf=2.0, neginf=-2.0),
                       torch.full((n, 20), want).nan_to_num(nan=1.0, posinf=2.0, neginf=-2.0))


@pytest.mark.parametrize("n", [3, 64, 65, 200])
@pytest.mark.parametrize("sign", [1, -1])
def test_bf16_a_x_next_to_the_largest_float(n, sign):
    """A x = 2^128 - 2^119, a float that is rounded to an infinite bf16."""
    a = torch.zeros(1, 64).bfloat16()
    a[0, 3], a[0, 40] = sign * 2.0 ** 127, sign * (2.0 ** 127 - 2.0 ** 119)
    got = adapted(torch.ones(n, 64).bfloat16(), a, torch.full((20, 1), 2.0 ** -100).bfloat16(), "bf16")
    assert torch.equal(got, torch.full((n, 20), sign * 2.0 ** 28).bfloat16())  # 2^28 - 2^19 in 8 bits


@pytest.mark.parametrize("n,out", [(9, 70), (64, 70), (65, 70), (200, 33), (700, 300), (1100, 4100)])
@pytest.mark.parametrize("inp", [37, 100, 200])
def test_f32_infinities(n, out, inp):
    """Infinite outputs are infinite with their sign, NaN only where the formula is, in rows and outputs of
    infinities and elsewhere, with bias and adapters."""
    m = adapters.make(inp, out, n, [4, 9], "f32", bias=True)
    x, w = m["x"], m["w"]
    w[:, 5], w[::3, 7] = torch.where(torch.arange(out) % 2 == 0, 1.0, -0.5), 0.0  # few bits: parts that are 0
    x[1, 5] = torch.inf
    x[2, 7] = -torch.inf
    x[n - 1, 5], x[n - 1, inp - 1] = torch.inf, -torch.inf
    x[n // 2, 6] = torch.nan
    x[4, 5], x[4, 6] = torch.inf, torch.nan
    x[5, 9], x[6, 9] = 0.0, 1.0
    w[out - 1, 9] = torch.inf
    w[3, 10], w[3, 11] = -torch.inf, torch.nan
    m["adapters"][1][1][7] = torch.inf
    layer = adapters.layer_of(m, 9, "f32")
    for ids in (None, m["ids"]):
        got = run(layer, x, ids)
        want = x.double() @ w.double().T + m["bias"].double()
        if ids is not None:
            for s, (a, b, scale) in enumerate(m["adapters"]):
                at = torch.nonzero(ids == s)[:, 0]
                want[at] += (scale * (x[at].double() @ a.double().T)) @ b.double().T
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(torch.where(got.isinf(), got.sign(), 0.0).double(), torch.where(want.isinf(), want.sign(), 0.0))
        assert torch.isfinite(got).sum() > n * out // 2 - 8 * out or n < 20


# Rows and outputs enough for the split into bf16 values, short sums and longer ones.
MANY = [(1100, 1000, 600), (2200, 1000, 100)]


@pytest.mark.parametrize("n,out,inp", MANY)
@pytest.mark.parametrize("xe,we", [(-61, -61), (-20, -102), (-102, -20), (-58, -64), (60, 60), (100, -126), (-126, 100), (0, 0)])
def test_f32_many_rows_near_the_ends(n, out, inp, xe, we):
    g = torch.Generator().manual_seed(n - xe)
    x, w = spread(g, n, inp) * 2.0 ** xe, spread(g, out, inp) * 2.0 ** we
    assert_f32(f32_forward(x, w), x, w)


@pytest.mark.parametrize("n,out,inp", MANY)
@pytest.mark.parametrize("low,high", [(-5, 5), (-30, 30), (-62, 52), (-120, 0)])
def test_f32_many_rows_of_any_spread(n, out, inp, low, high):
    g = torch.Generator().manual_seed(n + high)
    power = lambda *s: torch.randint(low, high + 1, s, generator=g).double()  # noqa: E731
    x = (spread(g, n, inp).double() * 2.0 ** power(n, inp)).float()
    w = (spread(g, out, inp).double() * 2.0 ** power(out, inp)).float()
    if high == 0:  # the small values of x beside the large ones of W
        x[:, ::2] = 0
        x[:, 0] = 1
        w[:, 0] = 2.0 ** -126
        w[:, 1:] = spread(g, out, inp - 1) * 2.0 ** 100
    assert_f32(f32_forward(x, w), x, w)


@pytest.mark.parametrize("n,out,inp", MANY)
def test_f32_many_rows_with_large_values_in_different_columns(n, out, inp):
    x, w = torch.full((n, inp), 1.23 * 2.0 ** -26), torch.full((out, inp), 1.1)
    x[:, 0], w[:, 0] = 1, 2.0 ** -40
    assert_f32(f32_forward(x, w), x, w)


@pytest.mark.parametrize("n,out,inp", MANY)
def test_f32_many_rows_with_infinities(n, out, inp):
    test_f32_infinities(n, out, inp)


@pytest.mark.parametrize("n,out,inp", [(1100, 1000, 600), (2200, 1000, 100), (2100, 4090, 300)])
def test_f32_many_rows_with_adapters(n, out, inp):
    """The three sizes of tiles, against the tolerances of f32's own roundings."""
    m = adapters.make(inp, out, n, [16, 0, 40], "f32", bias=True)
    layer = adapters.layer_of(m, 40, "f32")
    for ids in (m["ids"], torch.sort(m["ids"]).values):
        want, tol = adapters.reference(m, ids, "f32")
        assert_within(run(layer, m["x"], ids), want, tol)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("inp", [1, 2, 7, 15, 16, 17, 31, 33, 65])
@pytest.mark.parametrize("n,out", [(65, 1), (130, 2), (300, 33), (2100, 1030)])
def test_short_sums(dtype, inp, n, out):
    """Sums of one stage and less, by every form of the tiles."""
    m = adapters.make(inp, out, n, [1, 17], dtype, bias=True)
    layer = adapters.layer_of(m, 17, dtype)
    for ids in (m["ids"], None):
        want, tol = adapters.reference(m, ids, dtype)
        assert_within(run(layer, m["x"], ids), want, tol)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n", [64, 65, 66, 100, 127, 128, 129])
@pytest.mark.parametrize("inp,out", [(512, 40), (513, 40), (700, 130)])
def test_up_to_twice_64_rows(dtype, n, inp, out):
    m = adapters.make(inp, out, n, [3, 20, 0], dtype, bias=True)
    layer = adapters.layer_of(m, 20, dtype)
    for ids in (m["ids"], None):
        want, tol = adapters.reference(m, ids, dtype)
        assert_within(run(layer, m["x"], ids), want, tol)
