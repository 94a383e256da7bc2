"""Cases of the operators that serve many streams from a bounded cache: decode over a shared prefix, the attention weight that
every cache row has received, and eviction of the rows that received least.  ``own = False`` computes them in elementary
torch operations, ``own = True`` makes the calls of the engine."""
import importlib.util
import math
import os
import sys

import numpy as np
import torch

own = False

D = 64
SCALE = 0.125
ROPE_BASE = 10000.0
LN2 = math.log(2.0)


# ---------------------------------------------------------------------------------------------------------------- cases

def _shared(name, streams, prefixes, prefix_len, own_len, heads=16, kv_heads=2, kind="f16", append=True, loners=False, empty=False):
    return {"name": name, "op": "decode_shared", "streams": streams, "prefixes": prefixes, "prefix_len": prefix_len, "own_len": own_len,
            "heads": heads, "kv_heads": kv_heads, "kind": kind, "append": append, "loners": loners, "empty": empty}


def _observe(name, streams, length, n_q, heads=16, kv_heads=2, kind="f16", given_lse=False, decay=1.0):
    return {"name": name, "op": "observe", "streams": streams, "length": length, "n_q": n_q, "heads": heads, "kv_heads": kv_heads,
            "kind": kind, "given_lse": given_lse, "decay": decay}


def _evict(name, layers, streams, length, budget, kv_heads=2, n_sink=4, n_recent=32, ragged=False):
    return {"name": name, "op": "evict", "layers": layers, "streams": streams, "length": length, "budget": budget, "kv_heads": kv_heads,
            "n_sink": n_sink, "n_recent": n_recent, "ragged": ragged}


def listed():
    return [
        # one listener of a short voice prompt, a few tokens in: what a call costs at the least
        _shared("shared, 1 short stream", 1, 1, 90, 24),
        # a small server: four voices, half a minute of speech each, lengths all different
        _shared("shared, 32 streams 4 voices", 32, 4, 700, 512),
        # odd numbers of everything: streams without a prompt, streams without a row of their own, six query heads per kv head
        _shared("shared, odd and ragged", 37, 5, 1001, 777, heads=18, kv_heads=3, append=False, loners=True, empty=True),
        # a narrator's long prompt in the quantised cache
        _shared("shared, 64 streams q8_0", 64, 1, 2048, 1024, kind="q8_0"),
        # a full card: the long prompt of two voices under all streams that one step takes
        _shared("shared, 256 streams long", 256, 2, 4096, 2048),
        # the step of a few streams: latency
        _observe("observe, 4 streams step", 4, 300, 1),
        # the step of a full card; the decode before it has returned the log-sum-exp
        _observe("observe, 256 streams step", 256, 4096, 1, given_lse=True),
        # the last tokens of a prompt look back over it, in the quantised cache
        _observe("observe, window q8_0", 16, 2000, 32, kind="q8_0", decay=0.9),
        # the longest prompts
        _observe("observe, long window", 8, 8192, 64),
        # one stream that has just passed its budget
        _evict("evict, 1 stream", 6, 1, 300, 256),
        # the steady state: every stream of a model's layers gives up one row a step
        _evict("evict, one row each", 30, 32, 1025, 1024),
        # long prompts cut to a quarter, lengths all different
        _evict("evict, prompts to a quarter", 30, 24, 2048, 512, ragged=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["decode_shared", "decode_shared", "observe", "evict"])
    while True:
        heads, kv_heads = rng.choice([(16, 2), (16, 2), (8, 8), (18, 3), (6, 1), (4, 2)])
        kind = rng.choice(["f16", "f16", "q8_0"])
        if op == "decode_shared":
            streams = _log_int(rng, 1, 256)
            c = _shared("", streams, rng.randint(1, min(streams, 8)), _log_int(rng, 1, 8192), _log_int(rng, 1, 4096), heads, kv_heads, kind,
                        rng.random() < 0.7, rng.random() < 0.3, False)
            c["empty"] = not c["append"] and rng.random() < 0.5
            if streams * heads * (c["prefix_len"] + c["own_len"]) > 256 * 16 * 6144 or streams * kv_heads * c["own_len"] > 256 * 2 * 2048:
                continue
        elif op == "observe":
            n_q = 1 if rng.random() < 0.5 else _log_int(rng, 2, 64)
            c = _observe("", _log_int(rng, 1, 256), _log_int(rng, max(n_q, 2), 8192), n_q, heads, kv_heads, kind, n_q == 1 and rng.random() < 0.4,
                         rng.choice([1.0, 0.9, 0.99]))
            if c["streams"] * kv_heads * c["length"] > 256 * 2 * 4096 or c["streams"] * n_q * heads * c["length"] > 64 * 16 * 8192 * 8:
                continue
        else:
            length = _log_int(rng, 40, 4096)
            budget = max(8, min(length - 1, rng.choice([length - 1, length // 2, length // 4, rng.randint(8, length - 1)])))
            c = _evict("", _log_int(rng, 1, 30), _log_int(rng, 1, 64), length, budget, kv_heads, rng.randint(0, 4), rng.randint(0, budget - 4),
                       rng.random() < 0.5)
            if c["layers"] * c["streams"] * kv_heads * length > 30 * 24 * 2 * 2048:
                continue
        del c["name"]
        return c


# --------------------------------------------------------------------------------------------------------------- inputs

def _spread(lo, hi, n):
    """n lengths from lo to hi in even steps (their sum does not depend on the seed; their order does)."""
    return np.round(np.linspace(lo, hi, n) if n > 1 else np.array([hi])).astype(np.int64)


def _own_lengths(case):
    lens = _spread(max(1, case["own_len"] // 8), case["own_len"], case["streams"])
    if case["empty"]:
        lens[:: 5] = 0
    return lens


def _prefix_lengths(case):
    return _spread((3 * case["prefix_len"] + 3) // 4, case["prefix_len"], case["prefixes"])


def _prefix_of(case):
    of = np.arange(case["streams"]) % case["prefixes"]
    if case["loners"]:
        of[3:: 7] = -1
    return of


def _rows(gen, shape, kind):
    """Cache rows as (values, scales): f16 values and None, or int8 values and an f16 scale for every 32 of them.  Every block of
    the quantised form holds a value of full scale, as quantising a row makes it."""
    if kind == "f16":
        return torch.randn(shape, generator=gen, device="cuda").half(), None
    blocks = (*shape[:-1], shape[-1] // 32, 32)
    q = torch.randn(blocks, generator=gen, device="cuda").mul_(42).round_().clamp_(-127, 127)
    q[..., 0] = 127.0
    d = torch.rand(blocks[:-1], generator=gen, device="cuda").mul_(0.01).add_(0.02).half()
    return q.to(torch.int8), d


def _values(rows):
    q, d = rows
    return q.float() if d is None else (q.float() * d.float()[..., None]).flatten(-2)


def _rope_table(pos):
    i = torch.arange(D // 2, device="cuda", dtype=torch.float64)
    a = pos.double()[:, None] * ROPE_BASE ** (-2.0 * i / D)
    return torch.stack([a.cos(), a.sin()], -1).float()


def _cap(n):
    return max(8, -(-int(n) // 8) * 8)


_kept = {}


def _package():
    if "package" not in _kept:
        name = "voxcpm_cpp_b200"
        if name not in sys.modules:
            at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "voxcpm.cpp_b200")
            spec = importlib.util.spec_from_file_location(name, os.path.join(at, "__init__.py"), submodule_search_locations=[at])
            sys.modules[name] = importlib.util.module_from_spec(spec)
            spec.loader.exec_module(sys.modules[name])
        _kept["package"] = sys.modules[name]
        _kept["engine"] = sys.modules[name].Engine(0)
    return _kept["package"], _kept["engine"]


def _cache(k, v, kind):
    """A cache that holds k, v [layers, streams, kv heads, rows, 64] (as _rows gives them)."""
    p, engine = _package()
    layers, streams, kv_heads, rows = k[0].shape[:4]
    cache = p.KVCache(engine, layers, streams, kv_heads, rows, p.F16 if kind == "f16" else p.Q8_0)
    for layer in range(layers):
        at = [(x[0][layer], None if x[1] is None else x[1][layer]) for x in (k, v)]
        kk, vv = (_values(x).transpose(1, 2).contiguous() for x in at)
        cache.append(layer, kk, vv)
    torch.cuda.synchronize()
    return cache


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    order = np.random.RandomState(seed % (1 << 31))
    S, HK = case["streams"], case["kv_heads"]
    s = {"case": case}

    def ints(a):
        return torch.tensor(np.ascontiguousarray(a), dtype=torch.int32, device="cuda")

    if case["op"] == "decode_shared":
        n = _own_lengths(case)[order.permutation(S)]
        s["prefix_of"] = _prefix_of(case)[order.permutation(S)].astype(np.int32)
        s["of"] = ints(s["prefix_of"])
        s["kv_len"], s["prefix_len"] = ints(n), ints(_prefix_lengths(case)[order.permutation(case["prefixes"])])
        s["k"], s["v"] = (_rows(gen, (1, S, HK, _cap(case["own_len"]), D), case["kind"]) for _ in "kv")
        s["pk"], s["pv"] = (_rows(gen, (1, case["prefixes"], HK, _cap(case["prefix_len"]), D), case["kind"]) for _ in "kv")
        s["q"] = 1.5 * torch.randn((S, case["heads"], D), generator=gen, device="cuda")
        if case["append"]:
            s["k_new"], s["v_new"] = (torch.randn((S, HK, D), generator=gen, device="cuda") for _ in "kv")
            has = torch.where(s["of"] >= 0, s["prefix_len"][s["of"].clamp(min=0).long()], 0)
            s["rope"] = _rope_table(s["kv_len"] + has - 1)
    elif case["op"] == "observe":
        n = _spread(max(case["n_q"], case["length"] // 4), case["length"], S)[order.permutation(S)]
        s["kv_len"] = ints(n)
        s["n_seen"] = s["kv_len"] + 1000
        s["k"], s["v"] = (_rows(gen, (1, S, HK, _cap(case["length"]), D), case["kind"]) for _ in "kv")
        s["q"] = 1.5 * torch.randn((S, case["n_q"], case["heads"], D), generator=gen, device="cuda")
        # what a few passes like this one have left
        s["score"] = torch.rand((S, HK, _cap(case["length"])), generator=gen, device="cuda").mul_(4 * case["n_q"] * case["heads"] / HK / case["length"])
        s["row_pos"] = torch.randint(0, 100000, s["score"].shape, generator=gen, device="cuda", dtype=torch.int32)
        s["lse"] = None
        if case["given_lse"]:  # of a softmax that other rows have a share in too
            s["lse"] = _lse(s["q"][:, 0], _values(s["k"])[0], s["kv_len"]) + torch.rand((S, case["heads"]), generator=gen, device="cuda")
    else:
        L, N = case["layers"], case["length"]
        n = _spread(max(1, case["budget"] // 2), N, S)[order.permutation(S)] if case["ragged"] else np.full(S, N)
        s["kv_len"] = ints(n)
        s["n_seen"] = s["kv_len"] + 500
        s["k"], s["v"] = (_rows(gen, (L, S, HK, _cap(N), D), "f16") for _ in "kv")
        # weights as sums of softmaxes leave them: few rows with much, many with little, some with nothing at all
        w = torch.rand((L, S, HK, _cap(N)), generator=gen, device="cuda").pow_(8)
        s["score0"] = torch.where(w < 1e-4, 0.0, w)
        pos = torch.arange(_cap(N), device="cuda")[None].repeat(S, 1)
        pos = torch.where(pos < 8, pos, pos + 500)  # what earlier evictions took is missing
        s["row_pos0"] = pos.to(torch.int32)[None, :, None].expand(L, S, HK, -1).contiguous()
        s["score"], s["row_pos"] = s["score0"].clone(), s["row_pos0"].clone()
        s["new_len"] = torch.zeros(S, dtype=torch.int32, device="cuda")
        s["kept"] = torch.full((L, S, HK, case["budget"]), -1, dtype=torch.int32, device="cuda")
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        p, engine = _package()
        s["cache"] = _cache(s["k"], s["v"], case.get("kind", "f16"))
        if case["op"] == "decode_shared":
            s["prefix"] = _cache(s["pk"], s["pv"], case["kind"])
            s["plan"] = p.PrefixPlan(engine, s["prefix_of"], case["prefixes"], case["heads"], case["kv_heads"])
        if case.get("kind", "f16") == "f16":
            s["planes"] = s["cache"].planes()
        for name in ("k", "v", "pk", "pv"):
            s.pop(name, None)
    return s


# ---------------------------------------------------------------------------------------------------------- the operators

def _rotate(x, table):
    a, b = x[..., : D // 2], x[..., D // 2:]
    c, s = table[:, None, :, 0], table[:, None, :, 1]
    return torch.cat([a * c - b * s, a * s + b * c], -1)


def _quantise(x):
    b = x.unflatten(-1, (-1, 32))
    d = b.abs().amax(-1) / torch.tensor(127.0, device="cuda")
    inverse = torch.where(d != 0, torch.tensor(1.0, device="cuda") / d, 0.0)
    y = b * inverse[..., None]
    return (y.sign() * (y.abs().double() + 0.5).floor()).to(torch.int8), d.half()


def _visible(n, rows):
    return torch.arange(rows, device="cuda") < n[..., None]


def _lse(q, k, kv_len):
    """The log-sum-exp of one query over its stream's rows: [streams, heads]."""
    S, H, _ = q.shape
    HK = k.shape[1]
    e = (q.view(S, HK, H // HK, D) * SCALE) @ k.transpose(-1, -2)
    e = e.masked_fill(~_visible(kv_len, k.shape[2])[:, None, None], -math.inf)
    top = e.amax(-1, keepdim=True)
    return (top + (e - top).exp().sum(-1, keepdim=True).log()).view(S, H)


def _plain_decode_shared(s):
    case, q, (k, ks), (v, vs) = s["case"], s["q"], s["k"], s["v"]
    S, H, HK = case["streams"], case["heads"], case["kv_heads"]
    if case["append"]:
        q, k_new = _rotate(q, s["rope"]), _rotate(s["k_new"], s["rope"])
        at, last = torch.arange(S, device="cuda"), s["kv_len"].long() - 1
        if ks is None:
            k[0, at, :, last], v[0, at, :, last] = k_new.half(), s["v_new"].half()
        else:
            (k[0, at, :, last], ks[0, at, :, last]), (v[0, at, :, last], vs[0, at, :, last]) = _quantise(k_new), _quantise(s["v_new"])
    of = s["of"].clamp(min=0).long()
    n_prefix = torch.where(s["of"] >= 0, s["prefix_len"][of], 0)
    kk = torch.cat([_values(s["pk"])[0][of], _values((k, ks))[0]], 2)
    vv = torch.cat([_values(s["pv"])[0][of], _values((v, vs))[0]], 2)
    seen = torch.cat([_visible(n_prefix, s["pk"][0].shape[3]), _visible(s["kv_len"], k.shape[3])], 1)[:, None, None]
    e = ((q * SCALE).view(S, HK, H // HK, D) @ kk.transpose(-1, -2)).masked_fill(~seen, -math.inf)
    top = e.amax(-1, keepdim=True)
    w = (e - top.clamp(min=-1e30)).exp()
    total = w.sum(-1, keepdim=True)
    out = (w @ vv) / torch.where(total > 0, total, 1.0)
    got = {"out": out.view(S, H, D), "lse": (top + total.log()).view(S, H)}
    if case["append"] and ks is None:
        got["k"], got["v"] = k, v
    return got


def _plain_observe(s):
    case, q = s["case"], s["q"]
    S, H, HK, n_q = case["streams"], case["heads"], case["kv_heads"], case["n_q"]
    k = _values(s["k"])[0]
    rows = k.shape[2]
    e = (q.transpose(1, 2).reshape(S, HK, H // HK * n_q, D) * SCALE) @ k.transpose(-1, -2)
    i = torch.arange(n_q, device="cuda").repeat(H // HK)
    seen = torch.arange(rows, device="cuda") <= (s["kv_len"][:, None] - n_q + i)[..., None]
    e = e.masked_fill(~seen[:, None], -math.inf)
    if s["lse"] is None:
        w = (e - e.amax(-1, keepdim=True)).exp()
        w = w / w.sum(-1, keepdim=True)
    else:
        w = (e - s["lse"].view(S, HK, -1, 1)).exp()
    j = torch.arange(rows, device="cuda")
    here = (j < s["kv_len"][:, None])[:, None]
    new = here & (j >= s["kv_len"][:, None] - n_q)[:, None]
    old = torch.where(new, 0.0, s["score"] * case["decay"])
    s["score"].copy_(torch.where(here, old + w.sum(2), s["score"]))
    s["row_pos"].copy_(torch.where(new, (s["n_seen"] - s["kv_len"])[:, None, None] + j, s["row_pos"]))
    return {"score": s["score"], "row_pos": s["row_pos"]}


def _plain_evict(s):
    case, budget = s["case"], s["case"]["budget"]
    s["score"].copy_(s["score0"])
    s["row_pos"].copy_(s["row_pos0"])
    rows = s["score"].shape[-1]
    j = torch.arange(rows, device="cuda")
    n = s["kv_len"][None, :, None, None]
    safe = (s["row_pos"] < case["n_sink"]) | (s["row_pos"] >= s["n_seen"][None, :, None, None] - case["n_recent"])
    key = torch.where(safe, math.inf, s["score"]).masked_fill(j >= n, -math.inf)
    rank = key.sort(stable=True, dim=-1, descending=True).indices.argsort(-1)  # the place of every row among the kept
    keep = (rank < budget) & (j < n) | (n <= budget)
    holes, movers = ~keep & (j < budget), keep & (j >= budget) & (n > budget)
    # the i-th mover's row, then the row that every place below the budget gets
    order = torch.where(movers, movers.cumsum(-1) - 1, rows)
    mover = torch.zeros((*order.shape[:-1], rows + 1), dtype=torch.int64, device="cuda").scatter_(-1, order, j.expand(order.shape).contiguous())
    at = torch.where(holes, mover.gather(-1, (holes.cumsum(-1) - 1).clamp(min=0)), j)[..., :budget]
    for x in (s["score"], s["row_pos"]):
        x[..., :budget] = x.gather(-1, at)
    for x in (s["k"][0], s["v"][0]):
        x[..., :budget, :] = x.gather(-2, at[..., None].expand(*at.shape, D))
    s["new_len"].copy_(s["kv_len"].clamp(max=budget))
    s["kept"].copy_(torch.where(j[:budget] < n, at, s["kept"]))
    return {"k": s["k"][0], "v": s["v"][0], "score": s["score"], "row_pos": s["row_pos"], "new_len": s["new_len"], "kept": s["kept"]}


def run(state):
    s, case = state, state["case"]
    if not own:
        return {"decode_shared": _plain_decode_shared, "observe": _plain_observe, "evict": _plain_evict}[case["op"]](s)
    if case["op"] == "decode_shared":
        lse = torch.empty((case["streams"], case["heads"]), dtype=torch.float32, device="cuda")
        out = s["cache"].decode_shared(0, s["q"], s["kv_len"], case["own_len"], prefix=s["prefix"], plan=s["plan"], prefix_len=s["prefix_len"],
                                       prefix_bound=case["prefix_len"], scale=SCALE, k_new=s.get("k_new"), v_new=s.get("v_new"),
                                       rope_table=s.get("rope"), lse=lse)
        got = {"out": out, "lse": lse}
        if case["append"] and case["kind"] == "f16":
            got["k"], got["v"] = s["planes"]
        return got
    if case["op"] == "observe":
        s["cache"].observe(0, s["q"], s["kv_len"], case["length"], s["score"], row_pos=s["row_pos"], n_seen=s["n_seen"], n_new=case["n_q"],
                           lse=s["lse"], decay=case["decay"], scale=SCALE)
        return {"score": s["score"], "row_pos": s["row_pos"]}
    s["score"].copy_(s["score0"])
    s["row_pos"].copy_(s["row_pos0"])
    s["cache"].evict(s["kv_len"], case["length"], case["budget"], s["score"], s["row_pos"], s["n_seen"], s["new_len"], n_sink=case["n_sink"],
                     n_recent=case["n_recent"], kept=s["kept"])
    k, v = s["planes"]
    return {"k": k, "v": v, "score": s["score"], "row_pos": s["row_pos"], "new_len": s["new_len"], "kept": s["kept"]}


def work(case):
    HK, row = case["kv_heads"], 128 if case.get("kind", "f16") == "f16" else 68
    if case["op"] == "decode_shared":
        S, H = case["streams"], case["heads"]
        n, P, of = _own_lengths(case), _prefix_lengths(case), _prefix_of(case)
        rows = int(n.sum()) + int(sum(P[g] for g in set(of[of >= 0].tolist())))
        pairs = int(n.sum()) + S * float((of >= 0).mean() * P.mean())
        new = S * HK * (2 * D * 4 + 2 * row) + S * D * 4 if case["append"] else 0
        return {"bytes": rows * HK * 2 * row + S * H * (2 * D + 1) * 4 + new, "flops": 4 * H * D * pairs}
    if case["op"] == "observe":
        S, H, n_q = case["streams"], case["heads"], case["n_q"]
        n = int(_spread(max(n_q, case["length"] // 4), case["length"], S).sum())
        lse = S * H * 4 if case["given_lse"] else 0
        return {"bytes": n * HK * (row + 8) + S * n_q * (H * D + HK) * 4 + lse, "flops": 2 * H * D * n_q * n}
    L, S, N, budget = case["layers"], case["streams"], case["length"], case["budget"]
    n = _spread(max(1, budget // 2), N, S) if case["ragged"] else np.full(S, N)
    cut = n[n > budget]
    # of the rows above the budget the share that is kept moves down: about budget / n of them, and all that are recent
    moved = float(np.minimum(cut - budget, np.maximum(case["n_recent"], (cut - budget) * budget / np.maximum(cut, 1))).sum()) if len(cut) else 0.0
    return {"bytes": L * HK * (float(n.sum()) * 8 + moved * 2 * (2 * 128 + 8) + float(np.minimum(n, budget).sum()) * 4), "flops": 0}


# ------------------------------------------------------------------------------------------------------------- in 64 bits

def exact(case, seed):
    """The definitions again, in 64 bits and one stream (or one cache row list) at a time."""
    s = _inputs(case, seed)
    H, HK = case.get("heads", 0), case["kv_heads"]

    def values(rows, *at):
        q, d = rows
        return q[at].double() if d is None else (q[at].double() * d[at].double().unsqueeze(-1)).flatten(-2)

    if case["op"] == "decode_shared":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        lse = torch.full(out.shape[:2], -math.inf, dtype=torch.float64, device="cuda")
        q = s["q"]
        if case["append"]:  # rotated in 32 bits by definition, and stored in the cache's type
            pairs = torch.stack([q[..., :32], q[..., 32:]])
            c, t = s["rope"][:, None, :, 0], s["rope"][:, None, :, 1]
            q = torch.cat([pairs[0] * c - pairs[1] * t, pairs[0] * t + pairs[1] * c], -1)
            x, y = s["k_new"][..., :32], s["k_new"][..., 32:]
            rotated = torch.cat([x * c - y * t, x * t + y * c], -1)
            for i in range(case["streams"]):
                last = int(s["kv_len"][i]) - 1
                for (rows, scales), new in ((s["k"], rotated[i]), (s["v"], s["v_new"][i])):
                    if scales is None:
                        rows[0, i, :, last] = new.half()
                    else:
                        rows[0, i, :, last], scales[0, i, :, last] = _quantise(new)
        q = q.double()
        for i in range(case["streams"]):
            n, g = int(s["kv_len"][i]), int(s["prefix_of"][i])
            k, v = values(s["k"], 0, i)[:, :n], values(s["v"], 0, i)[:, :n]
            if g >= 0:
                P = int(s["prefix_len"][g])
                k, v = torch.cat([k, values(s["pk"], 0, g)[:, :P]], 1), torch.cat([v, values(s["pv"], 0, g)[:, :P]], 1)
            if k.shape[1]:
                e = torch.einsum("hrd,hjd->hrj", q[i].view(HK, -1, D), k) * SCALE
                lse[i] = e.logsumexp(-1).flatten()
                out[i] = torch.einsum("hrj,hjd->hrd", e.softmax(-1), v).reshape(H, D)
        got = {"out": out, "lse": lse}
        if case["append"] and s["k"][1] is None:
            got["k"], got["v"] = s["k"][0].double(), s["v"][0].double()
        return got
    if case["op"] == "observe":
        score, n_q = s["score"].double(), case["n_q"]
        for i in range(case["streams"]):
            n = int(s["kv_len"][i])
            k = values(s["k"], 0, i)[:, :n]
            q = s["q"][i].double().view(n_q, HK, -1, D)
            e = torch.einsum("ihrd,hjd->hrij", q, k) * SCALE
            late = torch.arange(n, device="cuda")[None] - torch.arange(n_q, device="cuda")[:, None] > n - n_q
            e = e.masked_fill(late, -math.inf)
            w = e.softmax(-1) if s["lse"] is None else (e - s["lse"][i].double().view(HK, -1, 1, 1)).exp()
            score[i, :, : n - n_q] *= float(np.float32(case["decay"]))
            score[i, :, n - n_q: n] = 0
            score[i, :, :n] += w.sum((1, 2))
        return {"score": score, "row_pos": None}
    score, k, v = s["score0"].double(), s["k"][0].double(), s["v"][0].double()
    budget, at = case["budget"], s["row_pos0"].cpu().numpy()
    weight = s["score0"].cpu().numpy()
    for i in range(case["streams"]):
        n, seen = int(s["kv_len"][i]), int(s["n_seen"][i])
        if n <= budget:
            continue
        for layer in range(case["layers"]):
            for h in range(HK):
                w, p = weight[layer, i, h, :n], at[layer, i, h, :n]
                safe = (p < case["n_sink"]) | (p >= seen - case["n_recent"])
                best = np.lexsort((np.arange(n), -w, ~safe))[:budget]
                movers = np.sort(best[best >= budget])
                holes = np.setdiff1d(np.arange(budget), best)
                a, b = torch.from_numpy(holes).cuda(), torch.from_numpy(movers).cuda()
                for x in (score, k, v):
                    x[layer, i, h, a] = x[layer, i, h, b]
    return {"k": k, "v": v, "score": score, "row_pos": None, "new_len": None, "kept": None}
