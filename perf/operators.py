"""Operators on the rows of a table, as cases that can be timed and compared.

Five kinds of calls, through the entry points of `glide_b200.rows`:

  lookup        `lookup_rows`: rows of a table by ids (what a search returned, or tokens), times a scale
  lookup_grad   `lookup_rows_grad`: the gradient of the table, equal ids joined
  dispatch      `dispatch_rows`: rows sorted by the partitions (experts) that each of them chose
  combine       `combine_rows`: the sorted rows back in their places, weighted and added
  combine_grad  `combine_rows_grad`: gradients of the sorted rows and of the weights

Where `own` is false the same is computed from elementary torch operations. Data are drawn on the GPU from the
seed alone. Ids and choices are 32 bits wide, -1 (0xffffffff) stands for none.
"""
import math

import numpy as np
import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "u8": torch.uint8}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2, "u8": 1}
_CONTEXT = None


def _ctx():
    """One context per process, as a program that uses the package keeps one."""
    global _CONTEXT
    if _CONTEXT is None:
        from glide_b200 import api
        _CONTEXT = api.Context(0)
    return _CONTEXT


# ---- cases -----------------------------------------------------------------------------------------------

def _table(kind, ids, n, dim, count, width, dtype, scale, empty, grad="", name=None):
    case = dict(kind=kind, ids=ids, n=n, dim=dim, count=count, width=width, dtype=dtype, scale=scale, empty=empty)
    if grad:
        case["grad"] = grad
    return case if name is None else dict(case, name=name)


def _routed(kind, rows, dim, choices, partitions, dtype, padded, second, name=None):
    case = dict(kind=kind, rows=rows, dim=dim, choices=choices, partitions=partitions, dtype=dtype, padded=padded, second=second)
    return case if name is None else dict(case, name=name)


def listed():
    return [
        # the ten neighbours of one query fetched from a million rows: an interactive lookup, all latency
        _table("lookup", "results", 1_000_000, 128, 1, 10, "f32", 1.0, 0.0, name="lookup_one_query"),
        # the result lists of the headline batch (10,000 queries, ten neighbours), some places unfilled
        _table("lookup", "results", 1_000_000, 128, 10_000, 10, "f32", 1.0, 0.02, name="lookup_results"),
        # a batch of token sequences with the scale by the square root of the width, a table of 1 GB
        _table("lookup", "tokens", 131_072, 4096, 32_768, 1, "bf16", 64.0, 0.0, name="lookup_tokens"),
        # the gradient of the indexed rows from the same lists: hardly any id twice, most rows untouched
        _table("lookup_grad", "results", 1_000_000, 128, 10_000, 10, "f32", 1.0, 0.02, grad="f32", name="grad_results"),
        # the gradient of the token table: a few ids make up much of the batch
        _table("lookup_grad", "tokens", 131_072, 4096, 32_768, 1, "bf16", 64.0, 0.0, grad="bf16", name="grad_tokens"),
        # a step of serving: 64 tokens, eight of 256 experts each
        _routed("dispatch", 64, 2048, 8, 256, "bf16", 0.0, 1.0, name="dispatch_serving"),
        # a step of training: 16,384 tokens, eight of 64 experts each, a fiftieth of them padding without any
        _routed("dispatch", 16_384, 2048, 8, 64, "bf16", 0.02, 1.0, name="dispatch_tokens"),
        # rows (dimension 100) to the nearest of 1,024 partitions and, for a third of them, to the second nearest too
        _routed("dispatch", 200_003, 100, 2, 1024, "f32", 0.0, 0.33, name="dispatch_partitions"),
        # serving's way back for an odd number of tokens
        _routed("combine", 61, 2048, 8, 256, "bf16", 0.0, 1.0, name="combine_serving"),
        # training's way back
        _routed("combine", 16_384, 2048, 8, 64, "bf16", 0.02, 1.0, name="combine_tokens"),
        # its gradient
        _routed("combine_grad", 16_384, 2048, 8, 64, "bf16", 0.02, 1.0, name="combine_grad_tokens"),
        # the gradient for wide half-precision rows of an odd batch with two experts each (cfg2's dimension)
        _routed("combine_grad", 4_999, 960, 2, 32, "f16", 0.02, 1.0, name="combine_grad_odd"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the same ranges: one id to whole batches, 24 to 4,096 values a row, 5,000 to 2,000,000 table rows,
    1 to 2,048 partitions, all types; sizes of every alignment, with none of them beyond the largest listed case."""
    kind = rng.choice(["lookup", "lookup_grad", "dispatch", "combine", "combine_grad"])
    dim = _log_int(rng, 24, 4096)
    if rng.random() < 0.5:
        dim = max(32, dim // 32 * 32)
    if kind in ("lookup", "lookup_grad"):
        dtype = rng.choice(["f32", "f16", "bf16", "u8"] if kind == "lookup" else ["f32", "f16", "bf16"])
        grad = rng.choice(["f32", dtype]) if kind == "lookup_grad" else ""
        n = min(_log_int(rng, 5_000, 2_000_000), 800_000_000 // (dim * 4))
        ids = rng.choice(["results", "tokens"])
        width = rng.choice([1, 10, 32, 100]) if ids == "results" else 1
        count = max(1, min(_log_int(rng, 1, 100_000), 100_000_000 // (dim * width)))
        return _table(kind, ids, n, dim, count, width, dtype, rng.choice([1.0, round(math.sqrt(dim), 3)]), rng.choice([0.0, 0.02, 0.2]), grad)
    choices = rng.choice([1, 2, 3, 4, 6, 8])
    partitions = max(choices, _log_int(rng, 1, 2048))
    rows = max(1, min(_log_int(rng, 1, 200_000), 200_000_000 // (dim * choices)))
    return _routed(kind, rows, dim, choices, partitions, rng.choice(["f32", "f16", "bf16"]), rng.choice([0.0, 0.02, 0.3]),
                   rng.choice([1.0, 1.0, 0.33]))


# ---- inputs ----------------------------------------------------------------------------------------------

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _values(shape, dtype, g):
    if dtype == "u8":
        return torch.randint(0, 219, shape, generator=g, device="cuda", dtype=torch.uint8)
    return torch.randn(shape, generator=g, device="cuda").to(_TYPES[dtype])


def _make_ids(case, g):
    """results: any row of the table, unfilled places; tokens: the share of the v-th token is about 1 / (v + 1)."""
    n, shape = case["n"], (case["count"], case["width"])
    u = torch.rand(shape, generator=g, device="cuda", dtype=torch.float64)
    ids = (u * n if case["ids"] == "results" else torch.exp(u * math.log(n + 1)) - 1).long().clamp(0, n - 1)
    return torch.where(torch.rand(shape, generator=g, device="cuda") < case["empty"], -1, ids).int()


def _make_choice(case, g):
    """The most likely of the partitions for each row, likeliest first, and their weights; some partitions are more popular than
    others, some rows are padding and choose none, and choices after the first are made with probability `second`."""
    rows, k, parts = case["rows"], case["choices"], case["partitions"]
    popular = torch.randn((1, parts), generator=g, device="cuda")
    score, choice = (torch.randn((rows, parts), generator=g, device="cuda") + 0.5 * popular).topk(k, dim=1)
    weights = torch.softmax(score, dim=1)
    none = (torch.rand((rows, 1), generator=g, device="cuda") < case["padded"]).repeat(1, k)
    none[:, 1:] |= torch.rand((rows, k - 1), generator=g, device="cuda") >= case["second"]
    return torch.where(none, -1, choice).int(), weights


def _order(choice, partitions):
    """Flat places (t * k + j) sorted by partition, ties by place, those without a partition last; and the partition of each."""
    key = choice.reshape(-1).long()
    key = torch.where((key >= 0) & (key < partitions), key, partitions)
    key, order = torch.sort(key, stable=True)
    return key, order


def _positions(choice, partitions):
    key, order = _order(choice, partitions)
    at = torch.arange(order.numel(), device="cuda")
    position = torch.empty_like(order)
    position[order] = torch.where(key < partitions, at, -1)
    return position.reshape(choice.shape).int()


def prepare(case, seed):
    g = _generator(seed)
    kind, dim, dtype = case["kind"], case["dim"], case["dtype"]
    s = {"case": case}
    if kind in ("lookup", "lookup_grad"):
        s["ids"] = _make_ids(case, g)
        if kind == "lookup":
            s["table"] = _values((case["n"], dim), dtype, g)
        else:
            s["grad"] = _values((case["count"], case["width"], dim), dtype, g)
        return s
    rows, k, parts = case["rows"], case["choices"], case["partitions"]
    s["choice"], s["weights"] = _make_choice(case, g)
    if kind == "dispatch":
        s["rows"] = _values((rows, dim), dtype, g)
        s["out"] = torch.zeros((rows * k, dim), dtype=_TYPES[dtype], device="cuda")     # what no row comes to stays zero
        return s
    s["position"] = _positions(s["choice"], parts)                                       # as the way there has left them
    s["sorted"] = _values((rows * k, dim), dtype, g)
    if kind == "combine_grad":
        s["grad"] = _values((rows, dim), dtype, g)
        s["out"] = torch.zeros((rows * k, dim), dtype=_TYPES[dtype], device="cuda")
    return s


# ---- one pass --------------------------------------------------------------------------------------------

def run(state):
    case = state["case"]
    return _RUN[case["kind"]](state, case)


def _run_lookup(s, case):
    if own:
        from glide_b200 import rows
        return rows.lookup_rows(_ctx(), s["table"], s["ids"], case["scale"])
    ids = s["ids"].long()
    there = (ids >= 0) & (ids < case["n"])
    got = s["table"][torch.where(there, ids, 0)].float() * case["scale"]
    got = torch.where(there[..., None], got, 0.0)
    return got if case["dtype"] == "u8" else got.to(s["table"].dtype)


def _run_lookup_grad(s, case):
    if own:
        from glide_b200 import rows
        return rows.lookup_rows_grad(_ctx(), s["grad"], s["ids"], case["n"], case["scale"], dtype=_TYPES[case["grad"]])
    ids = s["ids"].reshape(-1).long()
    there = (ids >= 0) & (ids < case["n"])
    part = torch.where(there[:, None], s["grad"].reshape(-1, case["dim"]).float(), 0.0)
    total = torch.zeros((case["n"], case["dim"]), device="cuda")
    total.index_add_(0, torch.where(there, ids, 0), part)
    return (total * case["scale"]).to(_TYPES[case["grad"]])


def _run_dispatch(s, case):
    if own:
        from glide_b200 import rows
        d = rows.dispatch_rows(_ctx(), s["rows"], s["choice"], case["partitions"], out=s["out"])
        return {"sorted": d.d_sorted, "map": d.d_map, "position": d.d_position, "start": d.d_segment_start}
    parts, k = case["partitions"], case["choices"]
    key, order = _order(s["choice"], parts)
    there = key < parts
    row = order // k
    got = torch.where(there[:, None], s["rows"][row], 0.0)
    position = torch.empty_like(order)
    position[order] = torch.where(there, torch.arange(order.numel(), device="cuda"), -1)
    start = torch.searchsorted(key, torch.arange(parts + 1, device="cuda"))
    return {"sorted": got, "map": torch.where(there, row, -1).int(), "position": position.reshape(s["choice"].shape).int(),
            "start": start.int()}


def _run_combine(s, case):
    if own:
        from glide_b200 import rows
        return rows.combine_rows(_ctx(), s["sorted"], s["position"], s["weights"])
    at = s["position"].long()
    there = at >= 0
    got = s["sorted"][torch.where(there, at, 0)].float() * s["weights"][..., None]
    return torch.where(there[..., None], got, 0.0).sum(1).to(s["sorted"].dtype)


def _run_combine_grad(s, case):
    if own:
        from glide_b200 import rows
        return rows.combine_rows_grad(_ctx(), s["grad"], s["sorted"], s["position"], s["weights"], out=s["out"])
    at = s["position"].long()
    there = at >= 0
    safe = torch.where(there, at, 0)
    grad = s["grad"].float()[:, None, :]
    weights = torch.where(there, (grad * s["sorted"][safe].float()).sum(2), 0.0)
    rows = torch.zeros((s["sorted"].shape[0] + 1, case["dim"]), device="cuda")
    last = torch.where(there, at, s["sorted"].shape[0])                     # those without a place go behind the last row
    rows[last.reshape(-1)] = (grad * s["weights"][..., None]).reshape(-1, case["dim"])
    return rows[:-1].to(s["sorted"].dtype), weights


_RUN = {"lookup": _run_lookup, "lookup_grad": _run_lookup_grad, "dispatch": _run_dispatch, "combine": _run_combine,
        "combine_grad": _run_combine_grad}


# ---- work and exact values ---------------------------------------------------------------------------------

def _distinct(case):
    """How many different rows the ids of a lookup name, in the mean."""
    n, t = case["n"], case["count"] * case["width"] * (1 - case["empty"])
    if case["ids"] == "results":
        return n * -math.expm1(t * math.log1p(-1.0 / n)) if n > 1 else 1.0
    v = np.arange(n, dtype=np.float64)
    p = np.log((v + 2) / (v + 1)) / math.log(n + 1)
    return float((-np.expm1(t * np.log1p(-np.minimum(p, 1 - 1e-12)))).sum())


def work(case):
    kind, dim, e = case["kind"], case["dim"], _BYTES[case["dtype"]]
    if kind in ("lookup", "lookup_grad"):
        t = case["count"] * case["width"]
        if kind == "lookup":
            return {"bytes": 4 * t + _distinct(case) * dim * e + t * dim * (4 if case["dtype"] == "u8" else e), "flops": t * dim}
        return {"bytes": 4 * t + t * (1 - case["empty"]) * dim * e + case["n"] * dim * _BYTES[case["grad"]], "flops": 2 * t * dim}
    t, k = case["rows"], case["choices"]
    pairs = t * (1 - case["padded"]) * (1 + (k - 1) * case["second"])
    if kind == "dispatch":
        return {"bytes": t * (1 - case["padded"]) * dim * e + pairs * dim * e + 12 * t * k + 4 * (case["partitions"] + 1), "flops": 0}
    if kind == "combine":
        return {"bytes": pairs * dim * e + t * dim * e + 8 * t * k, "flops": 2 * pairs * dim}
    return {"bytes": t * (1 - case["padded"]) * dim * e + 2 * pairs * dim * e + 12 * t * k, "flops": 3 * pairs * dim}


def exact(case, seed):
    """The definitions in 64 bits, one choice (or a run of ids) at a time."""
    s = prepare(case, seed)
    kind, dim = case["kind"], case["dim"]
    if kind == "lookup":
        ids = s["ids"].reshape(-1).long()
        out = torch.zeros((ids.numel(), dim), dtype=torch.float64, device="cuda")
        at = torch.nonzero((ids >= 0) & (ids < case["n"])).reshape(-1)
        out[at] = torch.index_select(s["table"], 0, ids[at]).double() * float(case["scale"])
        return out.reshape(case["count"], case["width"], dim)
    if kind == "lookup_grad":
        ids = s["ids"].reshape(-1).long()
        at = torch.nonzero((ids >= 0) & (ids < case["n"])).reshape(-1)
        out = torch.zeros((case["n"], dim), dtype=torch.float64, device="cuda")
        flat = s["grad"].reshape(-1, dim)
        for part in torch.split(at, max(1, 200_000_000 // dim)):
            out.index_put_((ids[part],), flat[part].double(), accumulate=True)
        return out.mul_(float(case["scale"]))
    k, parts = case["choices"], case["partitions"]
    if kind == "dispatch":
        choice = s["choice"].cpu().numpy().reshape(-1).astype(np.int64)
        place = np.flatnonzero((choice >= 0) & (choice < parts))
        place = place[np.lexsort((place, choice[place]))]
        used = torch.from_numpy(place // k).cuda()
        got = torch.zeros((case["rows"] * k, dim), dtype=torch.float64, device="cuda")
        got[:place.size] = s["rows"][used].double()
        where = np.full(case["rows"] * k, -1, np.int32)
        where[:place.size] = place // k
        position = np.full(case["rows"] * k, -1, np.int32)
        position[place] = np.arange(place.size, dtype=np.int32)
        start = np.concatenate([[0], np.cumsum(np.bincount(choice[place], minlength=parts))]).astype(np.int32)
        return {"sorted": got, "map": torch.from_numpy(where).cuda(), "position": torch.from_numpy(position.reshape(-1, k)).cuda(),
                "start": torch.from_numpy(start).cuda()}
    if kind == "combine":
        out = torch.zeros((case["rows"], dim), dtype=torch.float64, device="cuda")
        for j in range(k):
            t = torch.nonzero(s["position"][:, j] >= 0).reshape(-1)
            out[t] += s["weights"][t, j, None].double() * s["sorted"][s["position"][t, j].long()].double()
        return out
    rows = torch.zeros((case["rows"] * k, dim), dtype=torch.float64, device="cuda")
    weights = torch.zeros((case["rows"], k), dtype=torch.float64, device="cuda")
    for j in range(k):
        t = torch.nonzero(s["position"][:, j] >= 0).reshape(-1)
        p, grad = s["position"][t, j].long(), s["grad"][t].double()
        rows[p] = grad * s["weights"][t, j, None].double()
        weights[t, j] = (grad * s["sorted"][p].double()).sum(1)
    return rows, weights
