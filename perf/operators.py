"""Cases of the training and serving operators around the graph layers: rows of a learned
table by id and their gradient, log probabilities of given ids over scores and their gradient,
and a shared projection with one low-rank adapter per row.

`listed()` names the cases, `prepare` makes what a program has in hand before the call, `run`
makes one pass: in elementary torch operations, or, where `own` is true, through ruvector_amd.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
DEVICE = "cuda" if torch.cuda.is_available() else "cpu"


# ---------------------------------------------------------------- cases
def listed():
    return [
        # the embeddings of one small re-rank batch: latency
        dict(name="rows f32 100000x128 n64", op="rows", dtype="f32", rows=100_000, dim=128, n=64, ids="uniform", scale=1.0),
        # one training batch of ids out of a large table, scaled by sqrt(dim)
        dict(name="rows bf16 1000000x768 n131072", op="rows", dtype="bf16", rows=1_000_000, dim=768, n=131_072, ids="uniform", scale=27.7128),
        # that batch's dense gradient, with ids as frequent as words are (id 0 has about one in 18)
        dict(name="table grad bf16 262144x1024 n65536", op="table_grad", dtype="bf16", table_dtype="bf16", rows=262_144, dim=1024, n=65_536, ids="zipf", scale=32.0, accumulate=False),
        # gradients of several micro-batches summed in 32 bits: only the rows looked up are touched
        dict(name="table grad f32 500009x768 n100003", op="table_grad", dtype="f32", table_dtype="f32", rows=500_009, dim=768, n=100_003, ids="uniform", scale=1.0, accumulate=True),
        # a decoding step: few rows of many scores
        dict(name="log_probs bf16 16x131072 k20", op="log_probs", dtype="bf16", n=16, c=131_072, k=20, temperature=0.8, masked=False),
        # a training batch over a vocabulary
        dict(name="log_probs bf16 8192x32000 k5", op="log_probs", dtype="bf16", n=8192, c=32_000, k=5, temperature=1.0, masked=False),
        # contrastive scores of one batch of queries against the rows of an index, removed rows masked
        dict(name="log_probs f32 2503x10007 k10", op="log_probs", dtype="f32", n=2503, c=10_007, k=10, temperature=0.07, masked=True),
        # the gradients of the two losses above
        dict(name="log_probs grad bf16 8192x32000", op="log_probs_grad", dtype="bf16", n=8192, c=32_000, temperature=1.0, masked=False, entropy=False),
        dict(name="log_probs grad f32 2503x10007", op="log_probs_grad", dtype="f32", n=2503, c=10_007, temperature=0.07, masked=True, entropy=True),
        # one query through its tenant's adapter before a search
        dict(name="adapters f32 768x768 n1", op="adapters", dtype="f32", inp=768, out=768, n=1, rank=8, adapters=4, requests="single", bias=False),
        # a decoding step of 64 requests, each with an adapter of its own choice
        dict(name="adapters bf16 4096x4096 n64", op="adapters", dtype="bf16", inp=4096, out=4096, n=64, rank=16, adapters=32, requests="single", bias=False),
        # 24 ragged prompts in one batch
        dict(name="adapters bf16 4096x4096 n8192", op="adapters", dtype="bf16", inp=4096, out=4096, n=8192, rank=32, adapters=24, requests="ragged", bias=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rows", "table_grad", "log_probs", "log_probs_grad", "adapters"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if op in ("rows", "table_grad"):
        dim = rng.choice([_log(rng, 16, 2048), 64 * rng.randint(1, 32)])
        rows = _log(rng, 100, min(1_000_000, 300_000_000 // dim))
        n = _log(rng, 1, min(131_072, 100_000_000 // dim))
        case = dict(op=op, dtype=dtype, rows=rows, dim=dim, n=n, ids=rng.choice(["uniform", "zipf"]),
                    scale=rng.choice([1.0, round(math.sqrt(dim), 4)]))
        if op == "table_grad":
            case["accumulate"] = rng.random() < 0.5
            case["table_dtype"] = "f32" if case["accumulate"] else dtype
        return case
    if op in ("log_probs", "log_probs_grad"):
        c = _log(rng, 2, 262_144)
        n = _log(rng, 1, max(2, min(8192, 260_000_000 // c)))
        case = dict(op=op, dtype=dtype, n=n, c=c, temperature=rng.choice([1.0, 0.7, 0.07]), masked=rng.random() < 0.3)
        if op == "log_probs":
            case["k"] = rng.choice([0, 1, 5, 20, 64])
        else:
            case["entropy"] = rng.random() < 0.5
        return case
    inp, out = (rng.choice([_log(rng, 16, 4096), 64 * rng.randint(1, 64)]) for _ in range(2))
    n = _log(rng, 1, 8192 if dtype != "f32" else 2048)
    return dict(op=op, dtype=dtype, inp=inp, out=out, n=n, rank=rng.choice([4, 8, 16, 32, 64]),
                adapters=rng.randint(1, 32), requests=rng.choice(["single", "ragged"]), bias=rng.random() < 0.5)


# ---------------------------------------------------------------- inputs
def _ids(case, g):
    u = torch.rand(case["n"], generator=g, device=DEVICE, dtype=torch.float64)
    rows = case["rows"]
    if case["ids"] == "zipf":  # P(id) ~ 1 / (id + 1)
        ids = (torch.exp(u * math.log(rows + 1)) - 1).long()
    else:
        ids = (u * rows).long()
    return ids.clamp(0, rows - 1)


def _normal(g, shape, dtype, std=1.0):
    return (torch.randn(shape, generator=g, device=DEVICE, dtype=torch.float32) * std).to(dtype)


def _inputs(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    op, dtype = case["op"], DTYPES[case["dtype"]]
    if op == "rows":
        return dict(table=_normal(g, (case["rows"], case["dim"]), dtype, 0.05), ids=_ids(case, g))
    if op == "table_grad":
        t = dict(grad_out=_normal(g, (case["n"], case["dim"]), dtype, 0.01), ids=_ids(case, g))
        shape = (case["rows"], case["dim"])
        t["grad_table"] = _normal(g, shape, torch.float32, 0.01) if case["accumulate"] else torch.empty(shape, device=DEVICE, dtype=DTYPES[case["table_dtype"]])
        return t
    if op in ("log_probs", "log_probs_grad"):
        n, c = case["n"], case["c"]
        spread = 3.0 * case["temperature"] ** 0.5
        t = dict(targets=torch.randint(0, c, (n,), generator=g, device=DEVICE))
        scores = _normal(g, (n, c), dtype, spread)
        # a trained model's scores: the target stands out in most rows
        lift = torch.rand((n, 1), generator=g, device=DEVICE) * 3 * spread
        scores.scatter_add_(1, t["targets"][:, None], lift.to(dtype))
        if case["masked"]:
            scores.masked_fill_(torch.rand((n, c), generator=g, device=DEVICE) < 0.1, -math.inf)
            scores[n // 2] = -math.inf           # a row whose mask leaves nothing
            t["targets"][: n // 8] = -1          # rows without a target
        t["scores"] = scores
        if op == "log_probs_grad":
            t["grad_logp"] = _normal(g, (n,), torch.float32, 1.0)
            t["grad_entropy"] = _normal(g, (n,), torch.float32, 0.1) if case["entropy"] else None
            t.update(_kept(scores, case["temperature"]))
        return t
    n, R, S = case["n"], case["rank"], case["adapters"]
    t = dict(x=_normal(g, (n, case["inp"]), dtype), w=_normal(g, (case["out"], case["inp"]), dtype, case["inp"] ** -0.5),
             bias=_normal(g, (case["out"],), dtype, 0.1) if case["bias"] else None,
             a=_normal(g, (S, R, case["inp"]), dtype, case["inp"] ** -0.5),
             b=_normal(g, (S, case["out"], R), dtype, 0.5 * R ** -0.5),
             scales=torch.rand((S,), generator=g, device=DEVICE) + 0.5)
    t["ranks"] = [max(1, R // 2) if s % 3 == 2 else R for s in range(S)]  # adapters of different ranks
    for s, r in enumerate(t["ranks"]):
        t["a"][s, r:] = 0
        t["b"][s, :, r:] = 0
    if case["requests"] == "single":  # a row a request; slot S stands for "no adapter"
        ids = torch.randint(0, S + 1, (n,), generator=g, device=DEVICE)
        if n == 1:
            ids.clamp_(max=S - 1)
    else:                             # requests of ragged lengths, one adapter each
        cuts = torch.rand((n,), generator=g, device=DEVICE) < max(1, S) / n
        ids = (torch.cumsum(cuts.long(), 0) * 5 + seed) % (S + 1)
    t["adapter_ids"] = torch.where(ids == S, -1, ids).to(torch.int32)
    return t


def _kept(scores, temperature):
    """What the forward pass leaves for the backward pass: the row's largest score and log sum, and its entropy."""
    n = scores.shape[0]
    stats, entropy = torch.empty((n, 2), device=scores.device), torch.empty((n,), device=scores.device)
    step = max(1, 32_000_000 // scores.shape[1])
    for i in range(0, n, step):
        z = scores[i:i + step].double()
        m = z.amax(1)
        u = (z - torch.where(m == -math.inf, 0.0, m)[:, None]) / temperature
        e = u.exp()
        total = e.sum(1)
        stats[i:i + step, 0], stats[i:i + step, 1] = m.float(), total.log().float()
        h = total.log() - torch.where(e > 0, e * u, 0.0).sum(1) / total
        entropy[i:i + step] = torch.where(m == -math.inf, 0.0, h).float()
    return dict(stats=stats, entropy=entropy)


# ---------------------------------------------------------------- the framework's side
def _buffer(t):
    """A tensor's copy in a buffer of the framework."""
    import ruvector_amd as rv
    t = t.contiguous()
    b = rv.Buffer(max(t.numel() * t.element_size(), 1))
    if t.numel():
        _view(b, t.shape, t.dtype).copy_(t)
    return b


def _view(b, shape, dtype):
    flat = torch.from_dlpack(b)
    size = math.prod(shape) * torch.empty((), dtype=dtype).element_size()
    return flat[:size].view(dtype).view(tuple(shape))


def _out(shape, dtype):
    import ruvector_amd as rv
    b = rv.Buffer(max(math.prod(shape) * torch.empty((), dtype=dtype).element_size(), 1))
    return b, _view(b, shape, dtype)


def _own_state(case, t):
    import ruvector_amd as rv
    op, dtype = case["op"], DTYPES[case["dtype"]]
    s = {k: _buffer(v) for k, v in t.items() if isinstance(v, torch.Tensor)}
    if op == "rows":
        s["out"], s["answer"] = _out((case["n"], case["dim"]), dtype)
    elif op == "table_grad":
        s["answer"] = _view(s["grad_table"], t["grad_table"].shape, t["grad_table"].dtype)
    elif op == "log_probs":
        n, k = case["n"], case["k"]
        s["answer"] = {}
        for name, shape, kind in (("logp", (n,), torch.float32), ("rank", (n,), torch.int64), ("entropy", (n,), torch.float32),
                                  ("stats", (n, 2), torch.float32), ("top_ids", (n, k), torch.int64), ("top_logp", (n, k), torch.float32)):
            if k or not name.startswith("top"):
                s[name], s["answer"][name] = _out(shape, kind)
    elif op == "log_probs_grad":
        s["grad"], s["answer"] = _out((case["n"], case["c"]), dtype)
    else:
        layer = rv.AdapterLinear(case["inp"], case["out"], s["w"], bias=s.get("bias"), max_rank=case["rank"],
                                 max_adapters=case["adapters"], dtype=case["dtype"])
        for slot, r in enumerate(t["ranks"]):
            layer.set_adapter(slot, r, _buffer(t["a"][slot, :r]), _buffer(t["b"][slot, :, :r]), float(t["scales"][slot]))
        s = dict(layer=layer, x=s["x"], adapter_ids=s["adapter_ids"])
        s["out"], s["answer"] = _out((case["n"], case["out"]), dtype)
    return s


def prepare(case, seed):
    t = _inputs(case, seed)
    if own:
        if torch.cuda.is_available():
            torch.cuda.synchronize()
        t = _own_state(case, t)
    return dict(case=case, t=t)


def _run_own(case, s):
    import ruvector_amd as rv
    op = case["op"]
    if op == "rows":
        rv.embedding_forward_device(s["table"], case["rows"], case["dim"], s["ids"], case["n"], s["out"], scale=case["scale"], dtype=case["dtype"])
    elif op == "table_grad":
        rv.embedding_backward_device(s["grad_out"], s["ids"], case["n"], case["rows"], case["dim"], s["grad_table"], scale=case["scale"],
                                     dtype=case["dtype"], table_dtype=case["table_dtype"], accumulate=case["accumulate"])
    elif op == "log_probs":
        rv.log_probs_device(s["scores"], case["n"], case["c"], case["temperature"], targets=s["targets"], k=case["k"], logp=s["logp"],
                            rank=s["rank"], entropy=s["entropy"], stats=s["stats"], top_ids=s.get("top_ids"), top_logp=s.get("top_logp"), dtype=case["dtype"])
    elif op == "log_probs_grad":
        rv.log_probs_backward_device(s["scores"], case["n"], case["c"], case["temperature"], s["stats"], s["grad"], targets=s["targets"],
                                     grad_logp=s["grad_logp"], entropy=s["entropy"], grad_entropy=s.get("grad_entropy"), dtype=case["dtype"])
    else:
        s["layer"].forward_device(s["x"], case["n"], s["out"], adapter_ids=s["adapter_ids"])
    return s["answer"]


# ---------------------------------------------------------------- the plain form
def _plain_rows(case, t):
    return (t["table"][t["ids"]].float() * case["scale"]).to(t["table"].dtype)


def _plain_table_grad(case, t):
    add = t["grad_out"].float() * case["scale"]
    if case["accumulate"]:
        return t["grad_table"].index_add_(0, t["ids"], add)
    total = torch.zeros(t["grad_table"].shape, device=add.device).index_add_(0, t["ids"], add)
    return t["grad_table"].copy_(total)


def _order(scores):
    """Distinct 64-bit keys that order a row's scores downwards, ties by the lowest index first."""
    f = scores.float()
    bits = (f + 0.0).view(torch.int32)
    bits = torch.where(bits >= 0, bits, bits ^ 0x7FFFFFFF).long()
    return (bits << 32) + (0xFFFFFFFF - torch.arange(scores.shape[1], device=scores.device))


def _plain_log_probs(case, t):
    s, target, k = t["scores"].float(), t["targets"], case["k"]
    n, c = s.shape
    m = s.amax(1)
    empty = m == -math.inf
    u = (s - torch.where(empty, 0.0, m)[:, None]) / case["temperature"]
    e = torch.exp(u)
    total = e.sum(1)
    log_sum = torch.log(total)
    entropy = torch.where(empty, 0.0, log_sum - torch.where(e > 0, e * u, 0.0).sum(1) / total)
    at = target.clamp(min=0)[:, None]
    logp = torch.where(empty, -math.inf, u.gather(1, at)[:, 0] - log_sum)
    st = s.gather(1, at)
    rank = ((s > st) | ((s == st) & (torch.arange(c, device=s.device) < at))).sum(1)
    out = dict(logp=torch.where(target < 0, 0.0, logp), rank=torch.where(target < 0, -1, rank), entropy=entropy, stats=torch.stack([m, log_sum], 1))
    if k:
        ids = torch.topk(_order(t["scores"]), min(k, c), dim=1).indices
        value = s.gather(1, ids)
        top = torch.where(value == -math.inf, -math.inf, u.gather(1, ids) - log_sum[:, None])
        out["top_ids"] = torch.full((n, k), -1, device=s.device)
        out["top_ids"][:, : ids.shape[1]] = torch.where(value == -math.inf, -1, ids)
        out["top_logp"] = torch.full((n, k), -math.inf, device=s.device)
        out["top_logp"][:, : ids.shape[1]] = top
    return out


def _plain_log_probs_grad(case, t):
    s, target, inv = t["scores"].float(), t["targets"], 1.0 / case["temperature"]
    m, log_sum = t["stats"][:, :1], t["stats"][:, 1:]
    empty = m == -math.inf
    lp = (s - torch.where(empty, 0.0, m)) * inv - torch.where(empty, 0.0, log_sum)
    p = torch.where(empty, 0.0, torch.exp(lp))
    gl = torch.where(target < 0, 0.0, t["grad_logp"])[:, None]
    d = -gl * p
    if t["grad_entropy"] is not None:
        d = d - t["grad_entropy"][:, None] * torch.where(p > 0, p * (lp + t["entropy"][:, None]), 0.0)
    d.scatter_add_(1, target.clamp(min=0)[:, None], torch.where(empty, 0.0, gl))
    return (d * inv).to(t["scores"].dtype)


def _plain_adapters(case, t):
    x, ids = t["x"].float(), t["adapter_ids"].long()
    S, R = case["adapters"], case["rank"]
    mine = (ids[:, None] == torch.arange(S, device=x.device)) * t["scales"]
    h = (x @ t["a"].float().view(S * R, -1).T).view(-1, S, R) * mine[:, :, None]
    y = x @ t["w"].float().T + h.view(-1, S * R) @ t["b"].float().permute(0, 2, 1).reshape(S * R, -1)
    if t["bias"] is not None:
        y = y + t["bias"].float()
    return y.to(t["x"].dtype)


PLAIN = dict(rows=_plain_rows, table_grad=_plain_table_grad, log_probs=_plain_log_probs, log_probs_grad=_plain_log_probs_grad, adapters=_plain_adapters)


def run(state):
    if own:
        return _run_own(state["case"], state["t"])
    return PLAIN[state["case"]["op"]](state["case"], state["t"])


# ---------------------------------------------------------------- bytes and operations
def _touched(case):
    """Expected number of different ids."""
    rows, n = case["rows"], case["n"]
    if case["ids"] == "uniform":
        return rows * -math.expm1(-n / rows)
    total, lo, width = 0.0, 0, 1
    while lo < rows:  # P(id) = log((id + 2) / (id + 1)) / log(rows + 1), over ids in groups of about the same P
        hi = min(rows, lo + width)
        p = math.log((hi + 1) / (lo + 1)) / (hi - lo) / math.log(rows + 1)
        total += (hi - lo) * -math.expm1(n * math.log1p(-p)) if p < 1 else hi - lo
        lo, width = hi, max(1, hi // 16)
    return total


def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2}
    e, op, n = size[case["dtype"]], case["op"], case["n"]
    if op == "rows":
        return dict(bytes=n * 8 + (_touched(case) + n) * case["dim"] * e, flops=n * case["dim"])
    if op == "table_grad":
        moved = 2 * _touched(case) if case["accumulate"] else case["rows"]
        return dict(bytes=n * 8 + (n * e + moved * size[case["table_dtype"]]) * case["dim"], flops=2 * n * case["dim"])
    if op == "log_probs":
        return dict(bytes=n * (case["c"] * e + 8 + 4 + 8 + 4 + 8 + 12 * case["k"]), flops=6 * n * case["c"])
    if op == "log_probs_grad":
        return dict(bytes=n * (2 * case["c"] * e + 8 + 8 + 4 + (8 if case["entropy"] else 0)), flops=6 * n * case["c"])
    i, o, R = case["inp"], case["out"], case["rank"]
    used = min(case["adapters"], n)
    return dict(bytes=e * (n * (i + o) + i * o + used * R * (i + o)) + 4 * n, flops=2 * n * (i * o + R * (i + o)))


# ---------------------------------------------------------------- the definition, in 64 bits
def exact(case, seed):
    t, op = _inputs(case, seed), case["op"]
    if op == "rows":
        return torch.index_select(t["table"], 0, t["ids"]).double().mul_(case["scale"])
    if op == "table_grad":
        order = torch.argsort(t["ids"], stable=True)
        ids, count = torch.unique_consecutive(t["ids"][order], return_counts=True)
        ends = torch.cumsum(count, 0)
        rows = t["grad_out"][order]
        out = t["grad_table"].double() if case["accumulate"] else torch.zeros(t["grad_table"].shape, device=DEVICE, dtype=torch.float64)
        step = max(1, 100_000_000 // case["n"])
        for j in range(0, case["dim"], step):  # running sums over the sorted rows, a slab of columns at a time
            run_sum = torch.cumsum(rows[:, j:j + step].double(), 0)[ends - 1]
            run_sum[1:] -= run_sum[:-1].clone()
            out[ids, j:j + step] += run_sum * case["scale"]
        return out
    if op in ("log_probs", "log_probs_grad"):
        parts = []
        step = max(1, 64_000_000 // case["c"])
        for i in range(0, case["n"], step):
            z = t["scores"][i:i + step].double() / case["temperature"]
            target = t["targets"][i:i + step]
            lse = torch.logsumexp(z, 1, keepdim=True)
            lp = z - torch.where(lse == -math.inf, 0.0, lse)
            p = lp.exp()
            plogp = torch.special.entr(p)
            h = plogp.sum(1)
            there = target >= 0
            if op == "log_probs":
                one = torch.zeros(z.shape[0], device=DEVICE, dtype=torch.float64)
                one[there] = torch.take_along_dim(lp[there], target[there][:, None], 1)[:, 0]
                m = t["scores"][i:i + step].double().max(1).values
                log_sum = torch.where(m == -math.inf, -math.inf, lse[:, 0] - m / case["temperature"])
                got = dict(logp=one, entropy=h, stats=torch.stack([m, log_sum], 1))
                if case["k"]:
                    top = torch.sort(lp, 1, descending=True).values[:, : case["k"]]
                    got["top_logp"] = torch.nn.functional.pad(top, (0, case["k"] - top.shape[1]), value=-math.inf)
            else:
                d = torch.zeros_like(z)
                d[there, target[there]] = 1.0
                d = (d - p * there[:, None]) * t["grad_logp"][i:i + step, None].double()
                if t["grad_entropy"] is not None:
                    d += t["grad_entropy"][i:i + step, None].double() * (plogp - p * h[:, None])
                got = torch.where(lse == -math.inf, 0.0, d / case["temperature"]).to(torch.float32 if case["dtype"] != "f32" else torch.float64)
            parts.append(got)
        if op == "log_probs_grad":
            return torch.cat(parts)
        got = {k: torch.cat([q[k] for q in parts]) for k in parts[0]}
        return {**got, "rank": None, "top_ids": None}
    y = t["x"].double() @ t["w"].double().T
    if t["bias"] is not None:
        y += t["bias"].double()
    for s in range(case["adapters"]):
        at = torch.nonzero(t["adapter_ids"] == s)[:, 0]
        y[at] += float(t["scales"][s]) * ((t["x"][at].double() @ t["a"][s].double().T) @ t["b"][s].double().T)
    return y
