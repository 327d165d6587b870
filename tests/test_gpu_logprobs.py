"""Log probabilities, ranks, entropies and best alternatives of rows of scores, and their
gradient, against 64 bits."""
import math

import pytest
import torch

rv = pytest.importorskip("ruvector_amd")
from heads_ref import DTYPES, F32, HALF, TINY, assert_within, from_buffer, out_buffer, to_buffer  # noqa: E402

pytestmark = pytest.mark.gpu

OUTS = dict(logp=torch.float32, rank=torch.int64, entropy=torch.float32, stats=torch.float32, top_ids=torch.int64,
            top_logp=torch.float32)


def forward(scores, targets, temperature, k, dtype, ld=None, wanted=tuple(OUTS)):
    n, c = scores.shape
    shapes = dict(logp=(n,), rank=(n,), entropy=(n,), stats=(n, 2), top_ids=(n, k), top_logp=(n, k))
    bufs = {w: out_buffer(shapes[w], OUTS[w]) for w in wanted if k or not w.startswith("top")}
    stored = scores if ld is None else torch.nn.functional.pad(scores, (0, ld - c), value=1000.0)
    rv.log_probs_device(to_buffer(stored), n, c, temperature, targets=None if targets is None else to_buffer(targets), k=k,
                        ld=ld, dtype=dtype, **bufs)
    return {w: from_buffer(b, shapes[w], OUTS[w]) for w, b in bufs.items()}


def reference(scores, targets, temperature, k):
    s = scores.double()
    n, c = s.shape
    m = s.masked_fill(s.isnan(), -math.inf).amax(1)
    # from the largest score on: log(c) next to scores of -3e38 is lost in 64 bits too
    u = (s - torch.where(m == -math.inf, 0.0, m)[:, None]) / torch.tensor(temperature, dtype=torch.float32).double()
    log_sum = u.exp().sum(1).log()
    empty = log_sum == -math.inf
    lp = torch.where(empty[:, None], -math.inf, u - log_sum[:, None])
    has = (targets >= 0) & (targets < c)
    t = targets.clamp(0, c - 1)[:, None]
    st = s.gather(1, t)
    rank = ((s > st) | ((s == st) & (torch.arange(c) < t))).sum(1)
    entropy = -torch.where(lp == -math.inf, 0.0, lp.exp() * lp).sum(1)
    stats = torch.stack([m, log_sum], 1)
    out = dict(logp=torch.where(has, lp.gather(1, t)[:, 0], 0.0), rank=torch.where(has, rank, -1), entropy=entropy, stats=stats)
    if k:
        key = s.masked_fill(s.isnan(), -math.inf) + 0.0
        order = torch.sort(key, dim=1, descending=True, stable=True)
        ids, value = order.indices[:, :k], order.values[:, :k]
        top = lp.gather(1, ids)
        none = value == -math.inf
        out["top_ids"] = torch.nn.functional.pad(torch.where(none, -1, ids), (0, k - ids.shape[1]), value=-1)
        out["top_logp"] = torch.nn.functional.pad(torch.where(none, -math.inf, top), (0, k - ids.shape[1]), value=-math.inf)
    return out, lp


def tolerances(scores, temperature):
    """Each u = (s - m) / T is off by at most 3 roundings of |u|, and what differs by |u| > 30 adds
    nothing to S; e^u takes 2 more and S at most 6 + log2 parts of it again: S is within
    (U + 24) F32 of its value, U the weighted size of u (<= ln c, see below). The log adds
    one rounding of ln S and log p one of u."""
    s = scores.double()
    fin = s.masked_fill(~s.isfinite(), math.nan)
    spread = ((fin.nan_to_num(-1e30).amax(1) - fin.nan_to_num(1e30).amin(1)) / temperature).clamp(min=0)
    c = s.shape[1]
    chunk = math.ceil(c / 64) + 40               # additions in a row per lane, and joins
    # sum p |u| <= ln S + H <= 2 ln c
    s_err = F32 * (3 * 2 * math.log(max(c, 2)) + 4 + chunk)
    return spread, s_err


def check(scores, targets, temperature, k, dtype, **kw):
    got = forward(scores, targets, temperature, k, dtype, **kw)
    want, lp = reference(scores, targets, temperature, k)
    spread, s_err = tolerances(scores, temperature)
    log_c = math.log(max(scores.shape[1], 2))
    row = s_err + 3 * F32 * (log_c + 1)
    if "stats" in got:
        assert_within(got["stats"][:, 0], want["stats"][:, 0], 0.0, "largest score")
        assert_within(got["stats"][:, 1], want["stats"][:, 1], row, "log sum")
    if "logp" in got:
        assert_within(got["logp"], want["logp"], row + 4 * F32 * want["logp"].abs().nan_to_num(0, 0, 0), "logp")
        assert torch.equal(got["rank"], want["rank"])
    if "entropy" in got:
        # E = sum e^u u has the errors of e^u and of u on each term
        assert_within(got["entropy"], want["entropy"], 4 * (1 + 2 * log_c) * s_err + 8 * F32 * (log_c + 1), "entropy")
    if "top_ids" in got:
        assert torch.equal(got["top_ids"], want["top_ids"])
        assert_within(got["top_logp"], want["top_logp"], row + 4 * F32 * want["top_logp"].abs().nan_to_num(0, 0, 0), "top_logp")
    return got


def make(n, c, dtype, spread=3.0, seed=0):
    g = torch.Generator().manual_seed(seed + n * 1009 + c)
    return (torch.randn(n, c, generator=g) * spread).to(DTYPES[dtype]), torch.randint(0, c, (n,), generator=g)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,c,k,temperature", [
    (1, 1, 1, 1.0), (3, 2, 5, 0.5), (5, 63, 64, 1.0), (7, 64, 20, 2.0), (2, 1023, 5, 0.07), (4, 1025, 64, 1.0),
    (300, 257, 3, 1.0), (9, 10007, 10, 0.8), (1, 131072, 20, 1.0), (17, 40001, 0, 1.0), (5000, 33, 7, 1.0)])
def test_rows(dtype, n, c, k, temperature):
    scores, targets = make(n, c, dtype)
    targets[::4] = scores[::4].float().argmax(1)  # also the best one, and none
    if n > 2:
        targets[1], targets[2] = -1, c
    check(scores, targets, temperature, k, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n,c", [(6, 5), (6, 3001), (2, 70000)])
def test_masks(dtype, n, c):
    scores, targets = make(n, c, dtype, seed=5)
    g = torch.Generator().manual_seed(9)
    scores.masked_fill_(torch.rand(n, c, generator=g) < 0.6, -math.inf)
    scores[0] = -math.inf                                 # nothing is left
    scores[1] = -math.inf
    scores[1, c // 2] = 2.0                               # one is left
    low = torch.finfo(DTYPES[dtype]).min
    if n > 3:
        scores[2, : c // 2] = low                         # masked by the lowest value
        scores[3] = low                                   # all by the lowest value: equal scores
        targets[4] = int(torch.nonzero(scores[4] == -math.inf)[0]) if (scores[4] == -math.inf).any() else targets[4]
    for k in (1, 64):
        check(scores, targets, 1.0, k, dtype)
        check(scores, targets, 0.07, k, dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", ["equal", "up", "down", "two", "zeros"])
@pytest.mark.parametrize("n,c,k", [(3, 9000, 64), (2, 70001, 20)])
def test_ties_and_orders(dtype, shape, n, c, k):
    """Rows of equal scores, sorted rows (every score enters the list, or none after the first),
    two different scores, and both zeros."""
    base = dict(equal=torch.full((c,), 1.5), up=torch.arange(c) * 1e-3, down=-torch.arange(c) * 1e-3,
                two=(torch.arange(c) % 7 == 0) * 2.0, zeros=torch.where(torch.arange(c) % 2 == 0, -0.0, 0.0))[shape]
    scores = base.float().expand(n, c).to(DTYPES[dtype]).contiguous()
    targets = torch.tensor([0, c // 2 + 1, c - 1][:n])
    check(scores, targets, 1.0, k, dtype)


@pytest.mark.parametrize("scale,temperature", [(1e5, 1.0), (1e8, 1.0), (1e20, 1e18), (1e30, 1.0), (3e38, 1.0), (3e38, 1e30), (1.0, 1e-7), (1e-28, 1e-29),
                                               (1e3, 1e7), (10.0, 1e30), (1.0, 2.0 ** -100)])
@pytest.mark.parametrize("c", [70, 9000])
def test_scores_and_temperatures_of_any_size(scale, temperature, c):
    scores, targets = make(5, c, "f32", spread=1.0)
    scores = (scores.clamp(-1, 1) * scale).float()
    scores[0] += scale * 0.0 if scale > 1e37 else scale  # all positive
    scores[1, ::2] = -math.inf
    targets[:3] = scores[:3].argmax(1)
    got = forward(scores, targets, temperature, 3, "f32")
    want, _ = reference(scores, targets, temperature, 3)
    # u is off by 3 roundings of itself; what is over 40 below the best adds nothing, so log p is off by
    # that of the scores within 40 and by its own size's roundings, E (|u| e^u) as in check()
    _, s_err = tolerances(scores, 1.0)
    row = s_err + 3 * F32 * 40
    assert_within(got["stats"][:, 1], want["stats"][:, 1], row)
    assert_within(got["logp"], want["logp"], row + 4 * F32 * want["logp"].abs().nan_to_num(0, 0, 0))
    assert_within(got["entropy"], want["entropy"], 4 * (1 + 2 * math.log(c)) * s_err + 8 * F32 * 40)
    assert torch.equal(got["top_ids"], want["top_ids"]) and torch.equal(got["rank"], want["rank"])


def test_offsets_past_32_bits():
    """Rows more than 2^31 elements apart, of which 500 are used."""
    ld, c = 2 ** 31 + 64, 500
    big = rv.Buffer((ld + c) * 2)
    scores, targets = make(2, c, "bf16")
    for r in range(2):
        big.upload(scores[r].view(torch.uint8).numpy(), offset=r * ld * 2)
    outs = dict(logp=rv.Buffer(8), rank=rv.Buffer(16), stats=rv.Buffer(16), entropy=rv.Buffer(8))
    rv.log_probs_device(big, 2, c, 1.0, targets=to_buffer(targets), ld=ld, dtype="bf16", **outs)
    small = forward(scores, targets, 1.0, 0, "bf16")
    assert torch.equal(from_buffer(outs["logp"], (2,), torch.float32), small["logp"])
    assert torch.equal(from_buffer(outs["rank"], (2,), torch.int64), small["rank"])
    rv.log_probs_backward_device(big, 2, c, 1.0, outs["stats"], big, targets=to_buffer(targets), grad_logp=to_buffer(torch.ones(2)),
                                 ld=ld, dtype="bf16")
    import numpy as np
    want = backward(scores, targets, 1.0, torch.ones(2), None, "bf16")
    for r in range(2):
        got = torch.from_numpy(big.download(np.uint8, (c * 2,), offset=r * ld * 2)).view(torch.bfloat16)
        assert torch.equal(got, want[r])


def test_nan_and_inf():
    scores, targets = make(4, 3000, "f32")
    scores[0, 17] = math.nan
    scores[1, 2999] = math.inf
    scores[2, :] = math.nan
    got = forward(scores, targets, 1.0, 4, "f32")
    for r in (0, 1, 2):
        assert got["logp"][r].isnan() and got["entropy"][r].isnan() and got["stats"][r, 1].isnan()
    want, _ = reference(scores[3:], targets[3:], 1.0, 4)
    assert torch.equal(got["top_ids"][3], want["top_ids"][0])
    assert 17 not in got["top_ids"][0] and got["top_ids"][1, 0] == 2999 and (got["top_ids"][2] == -1).all()


@pytest.mark.parametrize("wanted", [("logp",), ("entropy",), ("stats",), ("top_ids",), ("top_logp",), ("rank", "top_ids"),
                                    ("entropy", "top_ids"), ("entropy", "logp", "rank"), ("rank", "logp")])
def test_each_output_alone(wanted):
    scores, targets = make(5, 2500, "bf16")
    full = forward(scores, targets, 1.0, 6, "bf16")
    some = forward(scores, targets, 1.0, 6, "bf16", wanted=wanted)
    for w in wanted:
        assert torch.equal(full[w], some[w])


def test_rows_with_a_stride():
    scores, targets = make(6, 1001, "f16")
    check(scores, targets, 1.0, 5, "f16", ld=1027)


def backward(scores, targets, temperature, gl, gh, dtype, ld=None, ld_grad=None, inplace=False):
    n, c = scores.shape
    f = forward(scores, targets if targets is not None else torch.zeros(n, dtype=torch.int64), temperature, 0, dtype)
    ld, ld_grad = ld or c, ld_grad or (ld or c)
    sb = to_buffer(torch.nn.functional.pad(scores, (0, ld - c), value=7.0))
    grad = sb if inplace else out_buffer((n, ld_grad), DTYPES[dtype])
    rv.log_probs_backward_device(sb, n, c, temperature, to_buffer(f["stats"]), grad,
                                 targets=None if targets is None else to_buffer(targets),
                                 grad_logp=None if gl is None else to_buffer(gl), entropy=to_buffer(f["entropy"]),
                                 grad_entropy=None if gh is None else to_buffer(gh), ld=ld, ld_grad=ld_grad, dtype=dtype)
    return from_buffer(grad, (n, ld_grad), DTYPES[dtype])


def grad_reference(scores, targets, temperature, gl, gh):
    n, c = scores.shape
    want, lp = reference(scores, targets, temperature, 0)
    p = lp.exp()
    has = ((targets >= 0) & (targets < c) & (want["stats"][:, 1] != -math.inf))[:, None]
    one = (torch.arange(c) == targets[:, None]).double()
    d = torch.zeros(n, c, dtype=torch.float64)
    if gl is not None:
        d = d + torch.where(has, gl.double()[:, None] * (one - p), 0.0)
    if gh is not None:
        d = d - gh.double()[:, None] * torch.where(p > 0, p * (lp + want["entropy"][:, None]), 0.0)
    return d / temperature, p, lp


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("entropy", [False, True])
@pytest.mark.parametrize("n,c,temperature", [(1, 1, 1.0), (4, 7, 0.5), (3, 1000, 1.0), (5, 4099, 0.07), (2, 70001, 1.0), (1500, 33, 1.0)])
def test_gradient(dtype, entropy, n, c, temperature):
    scores, targets = make(n, c, dtype, seed=2)
    g = torch.Generator().manual_seed(4)
    gl, gh = torch.randn(n, generator=g), torch.randn(n, generator=g) if entropy else None
    if n > 3:
        scores[1] = -math.inf
        scores[2, ::2] = -math.inf
        targets[3] = -1
    got = backward(scores, targets, temperature, gl, gh, dtype)
    want, p, lp = grad_reference(scores, targets, temperature, gl, gh)
    spread, s_err = tolerances(scores, temperature)
    log_c = math.log(max(c, 2))
    # p is off by the roundings of its exponent (5 of its size), of the log sum and of e
    p_err = p * (F32 * (6 * lp.abs().nan_to_num(0, 0, 0) + 6 + 4 * log_c) + s_err)
    gl_, gh_ = gl.abs().double()[:, None], (gh if entropy else torch.zeros(n)).abs().double()[:, None]
    inner = lp.abs().nan_to_num(0, 0, 0) + log_c
    tol = (gl_ * p_err + gh_ * (p_err * inner + p * (F32 * 8 * inner + 4 * (1 + 2 * log_c) * s_err))) / temperature
    tol = tol * 1.01 + want.abs() * (HALF[dtype] + 4 * F32) * 1.01 + gl_ * F32 / temperature + TINY[dtype]
    assert_within(got, want, tol)
    assert torch.equal(backward(scores, targets, temperature, gl, gh, dtype, inplace=True), got)


def test_gradient_by_entropy_alone_and_without_gradients():
    scores, _ = make(3, 500, "f32")
    gh = torch.randn(3)
    got = backward(scores, None, 1.0, None, gh, "f32")
    want, _, _ = grad_reference(scores, torch.full((3,), -1), 1.0, None, gh)
    assert_within(got, want, 3e-6 * want.abs().amax())  # 50 roundings of the largest term, see test_gradient
    assert not backward(scores, None, 1.0, None, None, "f32").any()


def test_gradient_against_differences():
    """Central differences of the 64-bit formula at the 32-bit gradient's inputs."""
    scores, targets = make(2, 40, "f32", seed=8)
    gl, gh = torch.tensor([0.7, -1.3]), torch.tensor([0.4, 0.9])

    def value(x):
        want, _ = reference(x, targets, 0.5, 0)
        return (want["logp"] * gl.double()).sum() + (want["entropy"] * gh.double()).sum()
    got = backward(scores, targets, 0.5, gl, gh, "f32").double()
    h = 1e-5
    for r, j in ((0, 0), (0, int(targets[0])), (1, 39), (1, int(targets[1])), (1, int(scores[1].argmax()))):
        d = torch.zeros(2, 40, dtype=torch.float64)
        d[r, j] = h
        slope = (value(scores.double() + d) - value(scores.double() - d)) / (2 * h)
        # differences: h^2 f''' / 6 with derivatives up to (2 / T)^3, and 1e-16 / h; the gradient: ~50 F32
        assert (got[r, j] - slope).abs() <= h * h * 64 + 1e-10 + 50 * F32 * 4


def test_gradient_leaves_the_row_padding():
    scores, targets = make(4, 101, "bf16")
    got = backward(scores, targets, 1.0, torch.ones(4), None, "bf16", ld=110, ld_grad=128)
    assert (got[:, 101:].contiguous().view(torch.uint8) == 0x7b).all()
    same = backward(scores, targets, 1.0, torch.ones(4), None, "bf16")
    assert torch.equal(got[:, :101], same)


def test_refusals():
    s, t, f = rv.Buffer(4 * 16 * 4), rv.Buffer(4 * 8), rv.Buffer(4 * 4)
    rv.log_probs_device(s, 4, 16, targets=t, logp=f)
    for bad in (dict(n=5), dict(c=17), dict(c=0), dict(ld=15), dict(temperature=0.0), dict(temperature=-1.0),
                dict(temperature=math.nan), dict(temperature=math.inf), dict(k=65), dict(k=-1), dict(k=2 ** 32), dict(dtype="int8"),
                dict(targets=None), dict(logp=s), dict(logp=t), dict(logp=f, entropy=f), dict(top_ids=f), dict(k=2, top_ids=f),
                dict(n=-1), dict(stats=f)):
        a = dict(dict(n=4, c=16, temperature=1.0, targets=t, logp=f), **bad)
        with pytest.raises(rv.RvxError):
            rv.log_probs_device(s, a.pop("n"), a.pop("c"), a.pop("temperature"), **a)
    st, g = rv.Buffer(4 * 8), rv.Buffer(4 * 16 * 4)
    rv.log_probs_backward_device(s, 4, 16, 1.0, st, g, targets=t, grad_logp=f)
    for bad in (dict(targets=None), dict(grad_entropy=f), dict(ld_grad=15), dict(grad=st), dict(grad=s, ld_grad=17),
                dict(n=5), dict(temperature=0.0)):
        a = dict(dict(n=4, temperature=1.0, grad=g, targets=t, grad_logp=f), **bad)
        with pytest.raises(rv.RvxError):
            rv.log_probs_backward_device(s, a.pop("n"), 16, a.pop("temperature"), st, a.pop("grad"), **a)
