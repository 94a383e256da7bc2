"""Decode over shared prefixes, the attention weight of cache rows and eviction by it, against their definitions in 64 bits.

Tolerances, from the arithmetic: a score is a sum of 64 products whose f32 additions round by at most 2^-24 of sums that stay
below 16 here (q of standard deviation 1.5, k of 1): at most 64 * 16 * 2^-24 = 6e-5 of a natural unit, typically an eighth of
that.  The operands lose nothing that counts beside it (q and the weights travel as two f16 parts: 2^-22; 2^x: 2^-22).  A weight
is off by that much relative to itself, a result (a mean of v by the weights) by at most twice that of its size: OUT = 1e-4 of
the output's RMS, LSE = 6e-5, WEIGHT = 1.2e-4 relative.  (One f16 rounding of the weights would be off by 5e-4 of the RMS.)"""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

OUT, LSE, WEIGHT = 1e-4, 6e-5, 1.2e-4
D = 64


def cuda(x, dtype=None):
    import torch
    return torch.as_tensor(np.ascontiguousarray(x), dtype=dtype, device="cuda")


def ints(x):
    import torch
    return cuda(np.asarray(x), torch.int32)


def gen(seed):
    import torch
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape):
    import torch
    return torch.randn(shape, generator=g, device="cuda")


def new_cache(engine, pkg, kind, layers, streams, kv_heads, rows):
    return pkg.KVCache(engine, layers, streams, kv_heads, -(-rows // 8) * 8, pkg.F16 if kind == "f16" else pkg.Q8_0)


def stored(cache, pkg, layer, stream, n):
    """The first n rows of a stream as the cache holds them: k, v [HK, n, 64] in 64 bits."""
    import torch
    out = []
    for x in cache.export(layer, stream, n):
        if cache.cfg.type == pkg.F16:
            out.append(torch.from_numpy(x.astype(np.float64)).cuda())
        else:
            blocks = x.reshape(*x.shape[:2], 2, 34)
            scale = np.ascontiguousarray(blocks[..., :2]).view(np.float16)[..., 0].astype(np.float64)
            out.append(torch.from_numpy((blocks[..., 2:].view(np.int8) * scale[..., None]).reshape(*x.shape[:2], D)).cuda())
    return out


def rotate(x, table):
    """f32, as the contract has it: x [S, heads, 64], table [S, 32, 2]."""
    import torch
    a, b, c, s = x[..., :32], x[..., 32:], table[:, None, :, 0], table[:, None, :, 1]
    return torch.cat([a * c - b * s, a * s + b * c], -1)


def attend(q, k, v, scale):
    """q [H, 64], k, v [HK, n, 64] in 64 bits -> out [H, 64], lse [H]."""
    import torch
    HK, n = k.shape[:2]
    if n == 0:
        return torch.zeros_like(q), torch.full(q.shape[:1], -torch.inf, dtype=torch.float64, device="cuda")
    e = torch.einsum("hrd,hjd->hrj", q.view(HK, -1, D), k) * scale
    return torch.einsum("hrj,hjd->hrd", e.softmax(-1), v).reshape(q.shape), e.logsumexp(-1).flatten()


def check_rows(out, lse, want_out, want_lse):
    import torch
    rms = want_out.square().mean().sqrt().clamp(min=1e-30)
    assert float((out.double() - want_out).abs().max() / rms) < OUT
    if lse is not None:
        assert torch.equal(torch.isinf(lse), torch.isinf(want_lse))
        seen = ~torch.isinf(want_lse)
        if seen.any():
            assert float((lse.double() - want_lse)[seen].abs().max()) < LSE


# name: kind, prefix of every stream, prefix lengths, own lengths, heads, kv heads
SHARED = {
    "one row of each": ("f16", [0], [1], [1], 16, 2),
    "no prefix row": ("f16", [0, 0], [0], [5, 70], 16, 2),
    "no own row": ("f16", [0, 1, 0], [130, 64], [0, 0, 0], 16, 2),
    "nothing at all": ("f16", [-1, 0, 1], [0, 9], [0, 0, 0], 16, 2),
    "tile edges": ("f16", [0, 1, 2, 3, 4, 5], [63, 64, 65, 127, 128, 129], [129, 128, 127, 65, 64, 63], 16, 2),
    "more streams than a row tile": ("f16", [0] * 33 + [1] * 16, [300, 511], list(range(0, 98, 2)), 16, 2),
    "mixed, some without": ("f16", [2, -1, 0, 2, -1, 1, 2, 0, 0, 2, 1], [700, 33, 1025], [5, 0, 300, 1, 66, 0, 8, 640, 17, 2, 90], 16, 2),
    "one head each": ("f16", [0] * 40 + [1] * 100, [77, 200], [3 + i % 50 for i in range(140)], 4, 4),
    "three heads": ("f16", [i % 3 for i in range(50)], [257, 100, 640], [1 + 7 * i for i in range(50)], 9, 3),
    "six heads": ("f16", [i % 2 for i in range(50)], [257, 1000], [1 + 7 * i for i in range(50)], 6, 1),
    "one stream, long prefix": ("f16", [0], [9000], [3], 16, 2),
    "few rows per tile, long": ("f16", [0, 0, 0, 1, 1], [4100, 2050], [1, 40, 500, 2, 3], 16, 2),
    "full row tiles, edges": ("f16", [i % 8 for i in range(128)], [1, 63, 64, 65, 127, 128, 129, 193], [i % 5 for i in range(128)], 16, 2),
    "full row tiles, long": ("f16", [i % 2 for i in range(40)], [5000, 1601], [1 + i for i in range(40)], 16, 2),
    "full row tiles, six heads": ("f16", [0] * 45, [777], [3] * 45, 6, 1),
    "full row tiles beside long streams": ("f16", [i % 8 for i in range(128)], [1, 63, 64, 65, 127, 128, 129, 400], [2500 - 19 * i for i in range(128)], 16, 2),
    "q8_0 full row tiles beside long streams": ("q8_0", [i % 8 for i in range(128)], [1, 63, 64, 65, 127, 128, 129, 400], [2500 - 19 * i for i in range(128)], 16, 2),
    "q8_0 one row of each": ("q8_0", [0], [1], [1], 16, 2),
    "q8_0 tile edges": ("q8_0", [0, 1, 2, 3, 4, 5], [63, 64, 65, 127, 128, 129], [129, 128, 127, 65, 64, 63], 16, 2),
    "q8_0 mixed": ("q8_0", [2, -1, 0, 2, -1, 1, 2, 0, 0, 2, 1], [700, 33, 1025], [5, 0, 300, 1, 66, 0, 8, 640, 17, 2, 90], 16, 2),
    "q8_0 full row tiles, edges": ("q8_0", [i % 8 for i in range(128)], [1, 63, 64, 65, 127, 128, 129, 193], [i % 5 for i in range(128)], 16, 2),
    "q8_0 full row tiles, long": ("q8_0", [i % 2 for i in range(40)], [5000, 1601], [1 + i for i in range(40)], 16, 2),
    "q8_0 many": ("q8_0", [0] * 70, [2000], [11 * i for i in range(70)], 16, 2),
    "q8_0 six heads": ("q8_0", [i % 2 for i in range(50)], [257, 1000], [1 + 7 * i for i in range(50)], 6, 1),
}


class SharedCase:
    def __init__(self, engine, pkg, case, seed=0, v_scale=1.0, layers=1, junk=True):
        self.pkg, self.engine = pkg, engine
        self.kind, self.of, self.P, self.n, self.H, self.HK = SHARED[case] if isinstance(case, str) else case
        g = gen(seed)
        S, G, self.layer = len(self.of), len(self.P), layers - 1
        self.cap, self.pcap = max(self.n) + 9, max(self.P) + 9
        self.own = new_cache(engine, pkg, self.kind, layers, S, self.HK, self.cap)
        self.prefix = new_cache(engine, pkg, self.kind, layers, G, self.HK, self.pcap)
        for cache, lens in ((self.own, self.n), (self.prefix, self.P)):
            rows = cache.cfg.max_len
            k, v = randn(g, len(lens), rows, self.HK, D), v_scale * randn(g, len(lens), rows, self.HK, D)
            if junk:  # what a stream before left behind its rows
                for s, n in enumerate(lens):
                    k[s, n:], v[s, n:] = float("inf") if self.kind == "q8_0" else float("nan"), float("inf")
            cache.append(self.layer, k, v)
        self.q = 1.5 * randn(g, S, self.H, D)
        self.kv_len, self.prefix_len = ints(self.n), ints(self.P)
        self.plan = pkg.PrefixPlan(engine, self.of, G, self.H, self.HK)

    def want(self, q=None, scale=0.125):
        import torch
        q, out, lse = self.q if q is None else q, [], []
        pre = [stored(self.prefix, self.pkg, self.layer, g, n) for g, n in enumerate(self.P)]
        for s, n in enumerate(self.n):
            kv = stored(self.own, self.pkg, self.layer, s, n)
            if self.of[s] >= 0:
                kv = [torch.cat([a, b], 1) for a, b in zip(pre[self.of[s]], kv)]
            o, e = attend(q[s].double(), *kv, scale)
            out.append(o)
            lse.append(e)
        return torch.stack(out), torch.stack(lse)

    def run(self, **kw):
        import torch
        kw = {"kv_bound": max(self.n), "prefix_bound": max(self.P), "lse": torch.full((len(self.of), self.H), 7.0, device="cuda")} | kw
        out = self.own.decode_shared(self.layer, kw.pop("q", self.q), self.kv_len, kw.pop("kv_bound"), prefix=self.prefix, plan=self.plan,
                                     prefix_len=self.prefix_len, **kw)
        return out, kw["lse"]

    def check(self, **kw):
        out, lse = self.run(**kw)
        self.engine.sync_status()
        check_rows(out, lse, *self.want(scale=kw.get("scale", 0.125)))
        return out, lse


@pytest.mark.parametrize("case", SHARED)
def test_shared_prefix_matches_the_definition(case, engine, pkg):
    SharedCase(engine, pkg, case).check()


@pytest.mark.parametrize("kind", ["f16", "q8_0"])
@pytest.mark.parametrize("v_scale", [1e-3, 300.0])
def test_shared_prefix_with_small_and_large_values(kind, v_scale, engine, pkg):
    """The two f16 parts of a weight (q8_0: times its row's scale) neither overflow nor fall below f16's normal range."""
    SharedCase(engine, pkg, (kind, [0, 0, 1], [300, 70], [40, 200, 3], 16, 2), v_scale=v_scale).check()
    SharedCase(engine, pkg, (kind, [0] * 16, [300], [40] * 16, 16, 2), v_scale=v_scale).check()


@pytest.mark.parametrize("streams", [2, 20, 40])
def test_shared_prefix_scales_that_grow_along_the_rows(streams, engine, pkg):
    """q8_0 scales over a range of 2^24 inside one softmax: the unit of the weights follows the largest so far."""
    import torch
    own = 3000 if streams == 40 else 200  # 40: the form that runs beside two decode CTAs per SM
    c = SharedCase(engine, pkg, ("q8_0", [0] * streams, [512], [own, 64] * (streams // 2), 16, 2), junk=False)
    for cache, n in ((c.own, 200), (c.prefix, 512)):
        rows = cache.cfg.max_len
        k = randn(gen(3), cache.cfg.n_streams, rows, 2, D)
        v = randn(gen(4), cache.cfg.n_streams, rows, 2, D) * torch.logspace(-4, 3, rows, device="cuda")[None, :, None, None]
        cache.append(0, k, v)
    c.check()


@pytest.mark.parametrize("kind", ["f16", "q8_0"])
@pytest.mark.parametrize("streams,heads,kv_heads", [(4, 16, 2), (12, 18, 3), (20, 4, 2)])
def test_long_prefixes_keep_their_precision(kind, streams, heads, kv_heads, engine, pkg):
    """7000 rows of a prefix under few streams: errors of single sums must not add up along it.  A result is a sum over eight shares of
    at most 896 keys, each a chain of 28 additions in f32 (half a step of 2^-23 each, random in sign: 6e-8 * sqrt(28)), of products
    truncated four times at the size of 32 keys' share: 1e-6 of the result's RMS holds all of it twice over."""
    c = SharedCase(engine, pkg, (kind, [0] * streams, [7000], [40] * streams, heads, kv_heads), junk=False)
    out, _ = c.run()
    engine.sync_status()
    want, _ = c.want()
    error = (out.double() - want).norm() / want.norm()
    assert float(error) < 1e-6


def test_shared_prefix_bounds_only_size_the_grid(engine, pkg):
    """Prefixes and streams longer than the bounds the host gave are attended in full; loose bounds change nothing but rounding."""
    c = SharedCase(engine, pkg, ("f16", [0, 1, 0, 1], [1500, 700], [90, 300, 0, 7], 16, 2))
    c.check(prefix_bound=300, kv_bound=40)
    c.check(prefix_bound=c.prefix.cfg.max_len, kv_bound=c.own.cfg.max_len)


def test_shared_prefix_bound_of_zero_reads_no_prefix(engine, pkg):
    c = SharedCase(engine, pkg, ("f16", [0, 0], [70], [9, 130], 16, 2))
    out, lse = c.run(prefix_bound=0)
    c.of = [-1, -1]
    check_rows(out, lse, *c.want())


def test_own_rows_only_is_decode_with_a_log_sum_exp(engine, pkg):
    import torch
    c = SharedCase(engine, pkg, ("f16", [0] * 7, [1], [1, 64, 700, 0, 65, 2000, 31], 16, 2))
    lse = torch.empty((7, 16), device="cuda")
    out = c.own.decode_shared(0, c.q, c.kv_len, 2000, lse=lse)
    c.of = [-1] * 7
    check_rows(out, lse, *c.want())


def test_own_rows_only_agrees_with_decode(engine, pkg):
    """On a cache without leftovers: vox_attn_decode asks that rows behind a stream's length are finite."""
    c = SharedCase(engine, pkg, ("f16", [0] * 7, [1], [1, 64, 700, 0, 65, 2000, 31], 16, 2), junk=False)
    out = c.own.decode_shared(0, c.q, c.kv_len, 2000)
    assert float((out - c.own.decode(0, c.q, c.kv_len, 2000)).abs().max()) < 1e-5


@pytest.mark.parametrize("kind", ["f16", "q8_0"])
def test_shared_prefix_with_the_arriving_row_and_rotary_table(kind, engine, pkg):
    """The step of a model: q and the new K row rotated for positions that count the prefix, the row stored by the launch."""
    c = SharedCase(engine, pkg, (kind, [0, 1, 0, -1, 1], [300, 65], [1, 64, 65, 129, 700], 16, 2))
    g = gen(9)
    k_new, v_new = randn(g, 5, 2, D), randn(g, 5, 2, D)
    table = engine.rope_table(ints([n + (c.P[p] if p >= 0 else 0) for n, p in zip(c.n, c.of)]), pos_offset=-1)
    out, lse = c.run(k_new=k_new, v_new=v_new, rope_table=table)
    engine.sync_status()
    q, k_rot = rotate(c.q, table), rotate(k_new, table)
    other = new_cache(engine, pkg, kind, 1, 5, 2, c.cap)
    other.append(0, k_rot[:, None].contiguous(), v_new[:, None].contiguous())
    for s, n in enumerate(c.n):
        for a, b in zip(c.own.export(0, s, n), other.export(0, s, 1)):
            assert np.array_equal(a[:, -1], b[:, 0])
    check_rows(out, lse, *c.want(q=q))


def test_prefixes_in_the_streams_own_cache_and_in_later_layers(engine, pkg):
    """Two streams of one cache are the prefixes of three others; the last of three layers."""
    import torch
    g = gen(5)
    cache = new_cache(engine, pkg, "f16", 3, 5, 2, 300)
    k, v = randn(g, 5, 300, 2, D), randn(g, 5, 300, 2, D)
    cache.append(2, k, v)
    cache.append(1, 9 * k, -v)
    n, of, P = [3, 70, 128], [4, 3, 4], [0, 0, 0, 290, 65]
    q = randn(g, 3, 16, D)
    plan = pkg.PrefixPlan(engine, of, 5)
    lse = torch.empty((3, 16), device="cuda")
    out = cache.decode_shared(2, q, ints(n), 128, prefix=cache, plan=plan, prefix_len=ints(P), prefix_bound=290, lse=lse)
    engine.sync_status()
    want = []
    for s in range(3):
        kv = [torch.cat([a, b], 1) for a, b in zip(stored(cache, pkg, 2, of[s], P[of[s]]), stored(cache, pkg, 2, s, n[s]))]
        want.append(attend(q[s].double(), *kv, 0.125))
    check_rows(out, lse, torch.stack([w[0] for w in want]), torch.stack([w[1] for w in want]))


def test_shared_prefix_agrees_with_one_cache_that_holds_everything(engine, pkg):
    import torch
    c = SharedCase(engine, pkg, ("f16", [0, 0, 1], [300, 129], [64, 1, 190], 16, 2))
    whole = new_cache(engine, pkg, "f16", 1, 3, 2, 500)
    for s in range(3):
        kv = [torch.cat([a, b], 1) for a, b in zip(stored(c.prefix, pkg, 0, c.of[s], c.P[c.of[s]]), stored(c.own, pkg, 0, s, c.n[s]))]
        whole.import_(0, s, *(x.half().cpu().numpy() for x in kv))
    want = whole.decode(0, c.q, ints([n + c.P[p] for n, p in zip(c.n, c.of)]), 500)
    out, _ = c.run()
    engine.sync_status()
    assert float((out - want).abs().max() / want.square().mean().sqrt()) < 2e-5


def test_shared_prefix_strided_queries_and_scale(engine, pkg):
    c = SharedCase(engine, pkg, ("f16", [0, 0, 0], [200], [20, 5, 130], 16, 2))
    wide = randn(gen(1), 3, 16, D + 2)
    c.q = wide[..., :D]
    c.check(scale=0.07)


def test_a_query_of_nan_gives_nan_and_leaves_the_others_alone(engine, pkg):
    import torch
    c = SharedCase(engine, pkg, ("f16", [0, 0, 0], [900], [700, 5, 0], 16, 2))
    clean, _ = c.run()
    c.q[1, 3, 5] = float("nan")
    out, lse = c.run()
    assert torch.isnan(out[1, 3]).all() and torch.isnan(lse[1, 3])
    keep = torch.ones(3, 16, dtype=torch.bool, device="cuda")
    keep[1, 3] = False
    assert torch.equal(out[keep], clean[keep])


def test_shared_prefix_is_the_same_in_every_run_and_counts_its_launches(engine, pkg):
    import torch
    c = SharedCase(engine, pkg, "mixed, some without")
    before = engine.launches
    a, la = c.run()
    assert engine.launches - before == 2
    for _ in range(5):
        b, lb = c.run()
        assert torch.equal(a, b) and torch.equal(la, lb)


def test_shared_prefix_captured_replayed_and_reassigned(engine, pkg):
    """A captured call follows the lengths and the plan as they are at replay; two graphs with workspaces of their own."""
    import torch
    c = SharedCase(engine, pkg, ("f16", [0, 1, 0, -1], [300, 65], [1, 64, 65, 129], 16, 2), junk=False)
    lse, dst = torch.empty((4, 16), device="cuda"), torch.empty((4, 16, D), device="cuda")
    ws = [torch.empty(64 << 20, dtype=torch.uint8, device="cuda") for _ in range(2)]
    c.run(lse=lse, dst=dst, workspace=ws[0])
    torch.cuda.synchronize()
    graphs = []
    for w in ws:
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(graph, stream=side):
            c.run(lse=lse, dst=dst, workspace=w, kv_bound=c.own.cfg.max_len, prefix_bound=c.prefix.cfg.max_len, stream=side)
        graphs.append(graph)
    for of, n, P in (([0, 1, 0, -1], [1, 64, 65, 129], [300, 65]), ([1, 1, -1, 1], [130, 0, 7, 70], [5, 250])):
        c.of, c.n, c.P = of, n, P
        c.plan.set(of)
        c.kv_len.copy_(ints(n))
        c.prefix_len.copy_(ints(P))
        for graph in graphs:
            dst.zero_()
            graph.replay()
            engine.sync_status()
            check_rows(dst, lse, *c.want())


def test_two_calls_on_two_streams(engine, pkg):
    import torch
    cases = [SharedCase(engine, pkg, name, seed=i) for i, name in enumerate(("mixed, some without", "few rows per tile, long"))]
    wants = [c.want() for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    ws = [torch.empty(64 << 20, dtype=torch.uint8, device="cuda") for _ in cases]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(10):
        for i, c in enumerate(cases):
            with torch.cuda.stream(streams[i]):
                got[i] = c.run(workspace=ws[i], stream=streams[i])
    torch.cuda.synchronize()
    for (out, lse), want in zip(got, wants):
        check_rows(out, lse, *want)


# ------------------------------------------------------------------------------------------------------------------ observe

OBSERVE = {  # kind, lengths, n_q, heads, kv heads
    "one row": ("f16", [1], 1, 16, 2),
    "empty and short": ("f16", [0, 1, 2, 63, 64, 65, 0], 1, 16, 2),
    "chunk edges": ("f16", [511, 512, 513, 1024, 1500], 1, 16, 2),
    "long": ("f16", [9001], 1, 16, 2),
    "longer than a cluster takes": ("f16", [24577, 600, 25100], 1, 16, 2),
    "as long as a cluster takes": ("q8_0", [24576, 20000, 1, 3000], 1, 8, 1),
    "many": ("f16", [3 * i for i in range(200)], 1, 16, 2),
    "one head each": ("f16", [100, 700], 1, 4, 4),
    "six heads": ("f16", [100, 700], 1, 6, 1),
    "q8_0": ("q8_0", [0, 1, 63, 64, 65, 700, 513], 1, 16, 2),
    "q8_0 six heads": ("q8_0", [130, 700], 1, 6, 1),
    "two queries": ("f16", [2, 65, 513], 2, 16, 2),
    "window": ("f16", [32, 33, 700, 1025], 32, 16, 2),
    "more queries than rows": ("f16", [0, 5, 40], 33, 16, 2),
    "largest window": ("f16", [64, 2050], 64, 16, 2),
    "three heads, odd window": ("f16", [90, 600], 7, 9, 3),
    "q8_0 window": ("q8_0", [17, 64, 700], 17, 16, 2),
    "q8_0 largest window": ("q8_0", [1000], 64, 16, 2),
    "few rows": ("f16", [0, 1, 3, 4, 511, 514, 4700], 4, 16, 2),
    "few rows, one head each": ("f16", [40, 600, 3000, 1], 64, 4, 4),
    "few rows, more queries than rows": ("f16", [3, 0, 9, 700], 10, 6, 1),
    "q8_0 few rows": ("q8_0", [0, 2, 17, 64, 700, 1300], 3, 16, 2),
    "q8_0 few rows, six heads": ("q8_0", [130, 5, 2100], 10, 6, 1),
    "nine heads, just too many rows": ("f16", [130, 700], 22, 9, 3),
}


class ObserveCase:
    def __init__(self, engine, pkg, case, seed=0, given_lse=False, layers=1):
        self.engine, self.pkg = engine, pkg
        self.kind, self.n, self.n_q, self.H, self.HK = OBSERVE[case] if isinstance(case, str) else case
        import torch
        g = gen(seed)
        S, self.layer = len(self.n), layers - 1
        self.cache = new_cache(engine, pkg, self.kind, layers, S, self.HK, max(self.n) + 9)
        rows = self.cache.cfg.max_len
        k = randn(g, S, rows, self.HK, D)
        for s, n in enumerate(self.n):
            k[s, n:] = float("inf") if self.kind == "q8_0" else float("nan")
        self.cache.append(self.layer, k, randn(g, S, rows, self.HK, D))
        self.q = 1.5 * randn(g, S, self.n_q, self.H, D)
        self.score = torch.rand((S, self.HK, rows + 3), generator=g, device="cuda")[..., :rows]
        self.row_pos = torch.full((S, self.HK, rows + 3), -5, dtype=torch.int32, device="cuda")[..., :rows]
        self.kv_len = ints(self.n)
        self.n_seen = self.kv_len + 1000
        self.lse = 3 + randn(g, S, self.H) if given_lse else None

    def want(self, n_new, decay):
        import torch
        score, pos = self.score.double(), self.row_pos.clone()
        for s, n in enumerate(self.n):
            if n == 0:
                continue
            k, _ = stored(self.cache, self.pkg, self.layer, s, n)
            e = torch.einsum("ihrd,hjd->hrij", self.q[s].double().view(self.n_q, self.HK, -1, D), k) * 0.125
            i, j = torch.arange(self.n_q, device="cuda")[:, None], torch.arange(n, device="cuda")
            e = e.masked_fill(j > n - self.n_q + i, -torch.inf)
            w = torch.nan_to_num(e.softmax(-1)) if self.lse is None else (e - self.lse[s].double().view(self.HK, -1, 1, 1)).exp()
            fresh = j >= n - n_new
            score[s, :, :n] = torch.where(fresh, 0.0, float(np.float32(decay)) * score[s, :, :n]) + w.sum((1, 2))
            pos[s, :, :n] = torch.where(fresh, 1000 + j.to(torch.int32), pos[s, :, :n])
        return score, pos

    def run(self, n_new=1, decay=1.0, **kw):
        kw = {"kv_bound": max(self.n)} | kw
        self.cache.observe(self.layer, self.q, self.kv_len, kw.pop("kv_bound"), self.score, row_pos=self.row_pos, n_seen=self.n_seen, n_new=n_new,
                           lse=self.lse, decay=decay, **kw)

    def check(self, n_new=1, decay=1.0, **kw):
        import torch
        score, pos = self.want(n_new, decay)
        self.run(n_new, decay, **kw)
        self.engine.sync_status()
        assert torch.equal(self.row_pos, pos)
        assert bool(((self.score.double() - score).abs() <= WEIGHT * score.abs() + 1e-9).all())


@pytest.mark.parametrize("case", OBSERVE)
def test_weights_match_the_definition(case, engine, pkg):
    n_q = OBSERVE[case][2]
    ObserveCase(engine, pkg, case).check(n_new=n_q, decay=0.75)


@pytest.mark.parametrize("case", ["empty and short", "chunk edges", "q8_0", "one head each"])
def test_weights_against_a_given_log_sum_exp(case, engine, pkg):
    ObserveCase(engine, pkg, case, given_lse=True).check()


@pytest.mark.parametrize("given_lse", [True, False])
@pytest.mark.parametrize("kind,streams,rows", [("f16", 128, 4700), ("q8_0", 64, 9300)])
def test_weights_of_many_long_streams(kind, streams, rows, given_lse, engine, pkg):
    """Enough keys for a block to take several chunks of a stream one after the other: lengths on both sides of every chunk's end."""
    lens = [min(rows, max(0, 512 * (i % 11) + (0, 1, -1, 64, 257)[i % 5])) for i in range(streams - 2)] + [rows, rows - 1]
    ObserveCase(engine, pkg, (kind, lens, 1, 4, 2), given_lse=given_lse).check(decay=0.5)


@pytest.mark.parametrize("kind,streams,rows", [("f16", 128, 4700), ("q8_0", 64, 9300)])
def test_few_query_rows_over_many_long_streams(kind, streams, rows, engine, pkg):
    lens = [min(rows, max(0, 512 * (i % 11) + (0, 1, -1, 64, 257)[i % 5])) for i in range(streams - 2)] + [rows, rows - 1]
    ObserveCase(engine, pkg, (kind, lens, 3, 4, 2)).check(n_new=2, decay=0.5)
    ObserveCase(engine, pkg, (kind, lens, 46, 4, 2)).check(n_new=46)
    ObserveCase(engine, pkg, (kind, lens, 49, 4, 2)).check(n_new=46)


@pytest.mark.parametrize("kind", ["f16", "q8_0"])
@pytest.mark.parametrize("n_q,heads,kv_heads", [(n, 16, 2) for n in (13, 20, 28, 36, 40, 44, 48, 52, 60, 64)] + [(43, 18, 3), (64, 6, 1), (50, 4, 4)])
def test_windows_of_every_width_over_several_tiles(n_q, heads, kv_heads, kind, engine, pkg):
    """Every number of score tiles to a key tile, for blocks that walk several key tiles, one list of rows after the other."""
    for streams in (73, 160):
        lens = [4 * ((i * 37) % 97) + 1 for i in range(streams)]
        ObserveCase(engine, pkg, (kind, lens, n_q, heads, kv_heads)).check(n_new=2, decay=0.5)


@pytest.mark.parametrize("n_new", [0, 3, 1000])
def test_new_rows_start_from_nothing(n_new, engine, pkg):
    """n_new rows (none, some, all of them) take the weight alone, whatever their score held: NaN included."""
    import torch
    c = ObserveCase(engine, pkg, ("f16", [1, 2, 70, 600], 1, 16, 2))
    for s, n in enumerate(c.n):
        c.score[s, :, max(0, n - n_new): n] = float("nan")
    score, pos = c.want(n_new, 1.0)
    for s, n in enumerate(c.n):  # 0 * NaN in the formula's place of "nothing"
        assert not torch.isnan(score[s, :, :n]).any()
    c.check(n_new=n_new)


def test_weights_with_a_rotary_table_and_strided_queries(engine, pkg):
    c = ObserveCase(engine, pkg, ("f16", [3, 200, 65], 1, 16, 2))
    table = engine.rope_table(ints([2, 199, 64]))
    wide = 1.5 * randn(gen(2), 3, 1, 16, D + 2)
    raw = wide[..., :D]
    c.q = rotate(raw[:, 0], table)[:, None]
    score, _ = c.want(1, 1.0)
    c.q = raw
    c.run(rope_table=table)
    assert bool(((c.score.double() - score).abs() <= WEIGHT * score.abs() + 1e-9).all())


@pytest.mark.parametrize("kind", ["f16", "q8_0"])
@pytest.mark.parametrize("n_q", [1, 3, 20])
def test_a_query_of_nan_touches_the_keys_it_sees(n_q, kind, engine, pkg):
    """Weights of a NaN query are NaN for the keys that it sees; later keys and other streams have the others' weights."""
    import torch
    c = ObserveCase(engine, pkg, (kind, [200, 700, 5], n_q, 16, 2))
    score, _ = c.want(1, 1.0)
    c.q[1, 0] = float("nan")
    seen = 700 - n_q + 1  # rows that the first query sees
    c.run()
    engine.sync_status()
    assert bool(c.score[1, :, :seen].isnan().all()) and not bool(c.score[1, :, seen:].isnan().any())
    for s in (0, 2):
        assert bool(((c.score[s].double() - score[s]).abs() <= WEIGHT * score[s].abs() + 1e-9).all())
    later = slice(seen, None)  # rows that the first query does not see: they never had its weight
    assert bool(((c.score[1, :, later].double() - score[1, :, later]).abs() <= WEIGHT * score[1, :, later].abs() + 1e-9).all())


def test_weights_of_every_stream_add_up_to_its_heads(engine, pkg):
    """Over a whole softmax the weights of a query sum to one: 8 heads give 8 per kv head."""
    c = ObserveCase(engine, pkg, ("f16", [700, 64, 9], 1, 16, 2))
    c.score.zero_()
    c.run(n_new=0)
    got = c.score.sum(-1)
    assert float((got - 8).abs().max()) < 1e-5


def test_a_longer_stream_than_the_bound_is_left_alone_and_reported(engine, pkg):
    import torch
    c = ObserveCase(engine, pkg, ("f16", [700, 64], 1, 16, 2))
    score, pos = c.score.clone(), c.row_pos.clone()
    c.run(kv_bound=100)
    with pytest.raises(pkg.VoxError) as err:
        engine.sync_status()
    assert err.value.status_name == "DEVICE_STATE"
    assert torch.equal(c.score[0], score[0]) and torch.equal(c.row_pos[0], pos[0])
    assert not torch.equal(c.score[1], score[1])
    engine.sync_status()


def test_weights_are_the_same_in_every_run(engine, pkg):
    import torch
    got = []
    for _ in range(3):
        c = ObserveCase(engine, pkg, "window")
        c.run(n_new=0)
        got.append(c.score.clone())
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])


# -------------------------------------------------------------------------------------------------------------------- evict

def evict_reference(score, pos, n, seen, budget, n_sink, n_recent):
    """kept[i] = former index of the row at place i, for one row list (numpy)."""
    if n <= budget:
        return np.arange(n)
    score, pos = score[:n], pos[:n]
    safe = (pos < n_sink) | (pos >= seen - n_recent)
    number = np.where(np.isnan(score), -np.inf, score)
    best = np.lexsort((np.arange(n), -number, np.isnan(score) & ~safe, ~safe))
    if safe.any():  # protected rows are all alike
        best = np.concatenate([np.flatnonzero(safe), best[~safe[best]]])
    best = best[:budget]
    at = np.arange(budget)
    at[np.setdiff1d(at, best)] = np.sort(best[best >= budget])
    return at


class EvictCase:
    def __init__(self, engine, pkg, kind, lens, layers, heads, rows, seed=0):
        import torch
        self.engine, self.pkg, self.n = engine, pkg, lens
        g = gen(seed)
        S = len(lens)
        self.cache = new_cache(engine, pkg, kind, layers, S, heads, rows)
        self.rows = self.cache.cfg.max_len
        for layer in range(layers):
            self.cache.append(layer, randn(g, S, self.rows, heads, D), randn(g, S, self.rows, heads, D))
        w = torch.rand((layers, S, heads, self.rows), generator=g, device="cuda")
        self.score = torch.where(w < 0.3, 0.0, (w * 16).round() / 16)  # many ties
        pos = torch.arange(self.rows, device="cuda") * 2
        self.row_pos = pos.to(torch.int32).expand(layers, S, heads, -1).contiguous()
        self.kv_len, self.n_seen = ints(lens), ints([2 * n for n in lens])

    def check(self, budget, n_sink=0, n_recent=0, kv_bound=None, with_kept=True):
        import torch
        L, S, HK, rows = self.score.shape
        before = [[self.cache.export(layer, s, rows) for s in range(S)] for layer in range(L)]
        score, pos = self.score.cpu().numpy(), self.row_pos.cpu().numpy()
        kept = torch.full((L, S, HK, budget), -1, dtype=torch.int32, device="cuda") if with_kept else None
        new_len = torch.full((S,), -1, dtype=torch.int32, device="cuda")
        self.cache.evict(self.kv_len, max(self.n) if kv_bound is None else kv_bound, budget, self.score, self.row_pos, self.n_seen, new_len,
                         n_sink=n_sink, n_recent=n_recent, kept=kept)
        self.engine.sync_status()
        assert new_len.tolist() == [min(n, budget) for n in self.n]
        seen = self.n_seen.tolist()
        for layer in range(L):
            for s in range(S):
                after = self.cache.export(layer, s, rows)
                for h in range(HK):
                    at = evict_reference(score[layer, s, h], pos[layer, s, h], self.n[s], seen[s], budget, n_sink, n_recent)
                    whole = np.concatenate([at, np.arange(len(at), rows)])
                    if with_kept:
                        got = kept[layer, s, h].cpu().numpy()
                        assert np.array_equal(got[:len(at)], at) and (got[len(at):] == -1).all()
                    assert np.array_equal(self.score[layer, s, h].cpu().numpy(), score[layer, s, h][whole], equal_nan=True)
                    assert np.array_equal(self.row_pos[layer, s, h].cpu().numpy(), pos[layer, s, h][whole])
                    for a, b in zip(after, before[layer][s]):
                        assert np.array_equal(a[h].view(np.uint8), b[h][whole].view(np.uint8))
        return kept


@pytest.mark.parametrize("kind", ["f16", "q8_0"])
@pytest.mark.parametrize("lens,budget,n_sink,n_recent", [
    ([1], 1, 0, 0),
    ([2], 1, 0, 1),
    ([0, 5, 64, 65, 66], 64, 2, 8),
    ([700, 64, 300, 513, 1025], 256, 4, 32),
    ([700, 701, 3], 699, 4, 690),
    ([600, 512, 530], 8, 0, 0),
    ([600, 512, 530], 8, 8, 0),
    ([600, 512, 530], 40, 0, 40),
    ([5000, 4100], 4000, 4, 32),
    ([700, 701, 699, 3, 702], 699, 4, 690),
    ([9, 10, 11, 12, 8, 7], 8, 1, 2),
    ([5, 4, 3, 2, 1, 0], 1, 0, 0),
    ([1025, 1026, 1027, 1028], 1024, 4, 32),
    ([5000, 2100], 900, 4, 32),
    ([4, 5, 6, 7] * 12, 3, 0, 0),
    ([36, 35, 34, 33] * 6, 32, 0, 0),
])
def test_eviction_matches_the_definition(kind, lens, budget, n_sink, n_recent, engine, pkg):
    EvictCase(engine, pkg, kind, lens, 2, 2, max(lens) + 9).check(budget, n_sink, n_recent)


@pytest.mark.parametrize("pad,offset", [(1, 0), (4, 1), (4, 2), (2, 1)])
@pytest.mark.parametrize("lens,budget", [([700, 64, 300, 513, 1026], 256), ([1025, 1026, 1027, 1028, 7], 1024), ([5000, 4100, 3, 4099], 900)])
def test_eviction_of_scores_off_the_vector_grid(lens, budget, pad, offset, engine, pkg):
    """Row lists of scores and positions that do not start on 16 bytes, some or all of them."""
    import torch
    c = EvictCase(engine, pkg, "f16", lens, 2, 2, max(lens) + 9)
    for name in ("score", "row_pos"):
        x = getattr(c, name)
        wide = torch.zeros((*x.shape[:3], x.shape[3] + pad), dtype=x.dtype, device="cuda")
        wide[..., offset: offset + x.shape[3]] = x
        setattr(c, name, wide[..., offset: offset + x.shape[3]])
    c.check(budget, 4, 32)


@pytest.mark.parametrize("budget", [24000, 49000, 50])
@pytest.mark.parametrize("spread", ["ties", "close", "wide"])
def test_eviction_from_the_longest_row_lists(budget, spread, engine, pkg):
    """Lists whose keys do not fit shared memory beside the moving rows (24000 of 49152), scores that are all alike, that differ in
    their last bits alone, and that span all magnitudes."""
    import torch
    c = EvictCase(engine, pkg, "f16", [49152], 1, 1, 49152)
    w = torch.rand(c.score.shape, generator=gen(2), device="cuda")
    c.score.copy_({"ties": torch.where(w < 0.7, 0.25, 0.5), "close": 1 + (w * 3000).floor() * 2.0 ** -23, "wide": torch.exp2(w * 250 - 125)}[spread])
    c.check(budget, 4, 32)


@pytest.mark.parametrize("heads", [1, 3])
def test_eviction_without_the_list_of_rows(heads, engine, pkg):
    EvictCase(engine, pkg, "f16", [300, 90], 1, heads, 320).check(100, 4, 16, kv_bound=320, with_kept=False)


def test_eviction_orders_special_scores(engine, pkg):
    """NaN goes before -inf, -0 ties with 0, and a protected row outlives +inf."""
    c = EvictCase(engine, pkg, "f16", [64], 1, 1, 64)
    special = [float("nan"), float("-inf"), -1.0, -0.0, 0.0, 1e-45, 1.0, float("inf")]
    c.score[0, 0, 0] = cuda(np.array([special[i % 8] for i in range(64)], np.float32))
    for budget in (60, 52, 44, 36, 20, 9):
        c.check(budget, 2, 3)
        c.n = [budget]
        c.kv_len.copy_(ints(c.n))


def test_eviction_again_and_again(engine, pkg):
    """One row a step, as a bounded stream gives it up: rows end up in any order, the protected ones never go."""
    import torch
    c = EvictCase(engine, pkg, "f16", [65], 1, 2, 80)
    g = gen(1)
    n_seen = 130
    for step in range(40):
        c.check(64, 4, 16)
        here = c.row_pos[0, 0, :, :64]
        for h in range(2):
            have = set(here[h].tolist())
            assert {p for p in range(0, 4, 2)} <= have
            assert {p for p in range(n_seen - 16, n_seen) if p % 2 == 0 or p > 130} <= have | {p for p in range(131) if p % 2}
        n_seen += 1
        c.cache.append(0, randn(g, 1, 1, 2, D), randn(g, 1, 1, 2, D), pos0=64)
        c.score[0, 0, :, 64], c.row_pos[0, 0, :, 64] = torch.rand(2, generator=g, device="cuda"), n_seen - 1
        c.n_seen.fill_(n_seen)


def test_eviction_leaves_a_longer_stream_than_the_bound(engine, pkg):
    import torch
    c = EvictCase(engine, pkg, "f16", [300, 90], 1, 2, 320)
    score, new_len = c.score.clone(), torch.zeros(2, dtype=torch.int32, device="cuda")
    c.cache.evict(c.kv_len, 100, 50, c.score, c.row_pos, c.n_seen, new_len, n_recent=8)
    with pytest.raises(pkg.VoxError) as err:
        engine.sync_status()
    assert err.value.status_name == "DEVICE_STATE"
    assert new_len.tolist() == [300, 50] and torch.equal(c.score[:, 0], score[:, 0])
    engine.sync_status()


def test_positions_default_to_the_index(engine, pkg):
    """n_seen NULL: a cache that has never given up a row."""
    import torch
    c = EvictCase(engine, pkg, "f16", [200], 1, 1, 200)
    c.row_pos[:] = torch.arange(200, device="cuda", dtype=torch.int32)
    new_len = torch.zeros(1, dtype=torch.int32, device="cuda")
    c.cache.evict(c.kv_len, 200, 50, c.score, c.row_pos, None, new_len, n_sink=3, n_recent=10)
    engine.sync_status()
    have = set(c.row_pos[0, 0, 0, :50].tolist())
    assert {0, 1, 2} <= have and set(range(190, 200)) <= have


def test_rows_beyond_four_gigabytes(engine, pkg):
    """Offsets past 32 bits: the last layer and stream of a 10 GB cache."""
    L, S, rows = 40, 64, 8192
    cache = pkg.KVCache(engine, L, S, 2, rows, pkg.F16)
    try:
        planes = cache.planes()
        g = gen(8)
        for x in planes:
            x[-1, -1] = randn(g, 2, rows, D).half()
        import torch
        n = torch.zeros(S, dtype=torch.int32, device="cuda")
        n[-1] = rows
        q = 1.5 * randn(g, S, 1, 16, D)
        score, pos = torch.zeros((1, S, 2, rows), device="cuda"), torch.zeros((1, S, 2, rows), dtype=torch.int32, device="cuda")
        cache.observe(L - 1, q, n, rows, score[0], row_pos=pos[0], n_new=rows)
        engine.sync_status()
        e = torch.einsum("hrd,hjd->hrj", q[-1, 0].double().view(2, 8, D), planes[0][-1, -1].double()) * 0.125
        want = e.softmax(-1).sum(1)
        assert bool(((score[0, -1].double() - want).abs() <= WEIGHT * want + 1e-9).all())
        assert torch.equal(pos[0, -1, 0], torch.arange(rows, device="cuda", dtype=torch.int32))
        k = planes[0][-1, -1].clone()
        kept, new_len = torch.full((1, S, 2, 1000), -1, dtype=torch.int32, device="cuda"), torch.empty(S, dtype=torch.int32, device="cuda")
        w, p = score[0, -1].cpu().numpy(), pos[0, -1].cpu().numpy()
        cache.evict(n, rows, 1000, score, pos, None, new_len, kept=kept, layer0=L - 1)
        engine.sync_status()
        for h in range(2):
            at = evict_reference(w[h], p[h], rows, rows, 1000, 4, 32)
            assert np.array_equal(kept[0, -1, h].cpu().numpy(), at)
            assert torch.equal(planes[0][-1, -1, h, :1000], k[h][cuda(at)])
    finally:
        cache.close()


def test_views_of_a_cache_keep_it_alive(engine, pkg):
    import gc
    import weakref
    cache = pkg.KVCache(engine, 2, 1, 2, 64, pkg.F16)
    k, v = cache.planes()
    assert k.shape == (2, 1, 2, 64, 64)
    alive = weakref.ref(cache)
    del cache, k
    gc.collect()
    assert alive() is not None and float(v[:, :, :, 3:9].float().sum()) == 0.0
    del v
    gc.collect()
    assert alive() is None


# ----------------------------------------------------------------------------------------------------------------- together

@pytest.mark.parametrize("kind", ["f16", "q8_0"])
def test_streams_of_one_voice_in_a_bounded_cache(kind, engine, pkg):
    """As a server runs them: streams under shared prompts decode, note the weights against the whole softmax and give up rows
    once they are past their budget, step after step; every step's results against 64 bits over the rows that are left."""
    import torch
    S, budget, P, layers = 5, 70, [130, 64], 2
    of = [0, 1, 0, -1, 0]
    own, prefix = new_cache(engine, pkg, kind, layers, S, 2, 128), new_cache(engine, pkg, kind, layers, 2, 2, 136)
    g = gen(77)
    n = np.array([60, 69, 3, 70, 66])
    seen = n.copy()
    for layer in range(layers):
        own.append(layer, randn(g, S, 128, 2, D), randn(g, S, 128, 2, D))
        prefix.append(layer, randn(g, 2, 136, 2, D), randn(g, 2, 136, 2, D))
    plan, prefix_len = pkg.PrefixPlan(engine, of, 2), ints(P)
    score, pos = torch.zeros((layers, S, 2, 128), device="cuda"), torch.zeros((layers, S, 2, 128), dtype=torch.int32, device="cuda")
    pos[:] = torch.arange(128, device="cuda", dtype=torch.int32)
    kv_len, n_seen, new_len = ints(n), ints(seen), ints(n)
    for step in range(12):
        n, seen = n + 1, seen + 1
        kv_len.copy_(ints(n))
        n_seen.copy_(ints(seen))
        table = engine.rope_table(n_seen + ints([P[p] if p >= 0 else 0 for p in of]), pos_offset=-1)
        for layer in range(layers):
            q, k_new, v_new = 1.5 * randn(g, S, 16, D), randn(g, S, 2, D), randn(g, S, 2, D)
            lse, before = torch.empty((S, 16), device="cuda"), score[layer].clone()
            out = own.decode_shared(layer, q, kv_len, 128, prefix=prefix, plan=plan, prefix_len=prefix_len, prefix_bound=136, k_new=k_new,
                                    v_new=v_new, rope_table=table, lse=lse, cache_stable=layer > 0)
            own.observe(layer, q[:, None], kv_len, 128, score[layer], row_pos=pos[layer], n_seen=n_seen, lse=lse, rope_table=table)
            engine.sync_status()
            qr = rotate(q, table).double()
            for s in range(S):
                k, v = stored(own, pkg, layer, s, int(n[s]))
                kk, vv = k, v
                if of[s] >= 0:
                    kk, vv = (torch.cat([a, b], 1) for a, b in zip(stored(prefix, pkg, layer, of[s], P[of[s]]), (k, v)))
                want, want_lse = attend(qr[s], kk, vv, 0.125)
                check_rows(out[s], lse[s], want, want_lse)
                w = (torch.einsum("hrd,hjd->hrj", qr[s].view(2, 8, D), k) * 0.125 - want_lse.view(2, 8, 1)).exp().sum(1)
                w[:, :-1] += before[s, :, : int(n[s]) - 1].double()
                assert bool(((score[layer, s, :, : int(n[s])].double() - w).abs() <= WEIGHT * w + 1e-9).all())
                assert (pos[layer, s, :, int(n[s]) - 1] == int(seen[s]) - 1).all()
        own.evict(kv_len, 128, budget, score, pos, n_seen, new_len, n_sink=2, n_recent=8)
        engine.sync_status()
        n = np.minimum(n, budget)
        assert new_len.tolist() == n.tolist()
    assert n.max() == budget and seen.max() > budget


@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("streams", [1, 2, 12])
def test_lengths_of_an_eviction_feed_the_next_call_directly(streams, shared, engine, pkg):
    """new_len as the kv_len of the launch behind it, which may be scheduled while the eviction still runs: few f16 streams (a
    cluster per pair) and more."""
    import torch
    g = gen(6)
    cache = new_cache(engine, pkg, "f16", 1, streams, 2, 2048)
    cache.append(0, randn(g, streams, 2048, 2, D), randn(g, streams, 2048, 2, D))
    q, full, cut = randn(g, streams, 16, D), ints([2000] * streams), ints([1500] * streams)
    score = torch.rand((1, streams, 2, 2048), generator=g, device="cuda")
    pos = torch.arange(2048, dtype=torch.int32, device="cuda").expand(1, streams, 2, 2048).contiguous()
    new_len = ints([0] * streams)

    def decode(n):
        return cache.decode_shared(0, q, n, 2048) if shared else cache.decode(0, q, n, 2048)

    for _ in range(20):
        new_len.fill_(40)
        torch.cuda.synchronize()
        cache.evict(full, 2048, 1500, score, pos, None, new_len)
        out = decode(new_len)
        engine.sync_status()
        assert new_len.tolist() == [1500] * streams
        assert torch.equal(out, decode(cut))


@pytest.mark.parametrize("kind", ["f16", "q8_0"])
@pytest.mark.parametrize("streams", [2, 40])
def test_a_captured_step_follows_its_inputs(kind, streams, engine, pkg):
    """Decode, the weights of a step and of a window, eviction and the next decode as one graph, each launch right behind the one whose
    results it takes; replayed with other lengths and queries it gives what the calls give one at a time."""
    import torch
    rows, budget = 900, 500

    def start(seed):
        g = gen(seed)
        c = new_cache(engine, pkg, kind, 1, streams, 2, rows)
        c.append(0, randn(g, streams, c.cfg.max_len, 2, D), randn(g, streams, c.cfg.max_len, 2, D))
        n = torch.randint(1, rows + 1, (streams,), generator=g, device="cuda", dtype=torch.int32)
        return {"cache": c, "q": randn(g, streams, 16, D), "window": randn(g, streams, 20, 16, D), "n": n,
                "score": torch.rand((1, streams, 2, rows + 4), generator=g, device="cuda"),
                "pos": torch.arange(rows + 4, device="cuda", dtype=torch.int32).expand(1, streams, 2, -1).contiguous(),
                "new": torch.full((streams,), 7, dtype=torch.int32, device="cuda"), "lse": torch.zeros((streams, 16), device="cuda"),
                "ws": torch.zeros(1 << 24, dtype=torch.uint8, device="cuda")}

    def step(s, wait):
        def then():
            if wait:
                engine.sync_status()
        c, out = s["cache"], []
        out.append(c.decode_shared(0, s["q"], s["n"], rows, lse=s["lse"], workspace=s["ws"])); then()
        c.observe(0, s["q"][:, None], s["n"], rows, s["score"][0], row_pos=s["pos"][0], lse=s["lse"], workspace=s["ws"]); then()
        c.observe(0, s["window"], s["n"], rows, s["score"][0], n_new=0, workspace=s["ws"]); then()
        c.evict(s["n"], rows, budget, s["score"], s["pos"], None, s["new"]); then()
        c.observe(0, s["window"], s["new"], rows, s["score"][0], n_new=0, decay=0.5, workspace=s["ws"]); then()
        c.observe(0, s["q"][:, None], s["new"], rows, s["score"][0], n_new=0, workspace=s["ws"]); then()
        out.append(c.decode_shared(0, s["q"], s["new"], rows, lse=s["lse"], workspace=s["ws"])); then()
        return out

    captured = start(0)
    step(captured, True)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        out = step(captured, False)
    for seed in (1, 2, 3):
        fresh, refill = start(seed), start(seed)
        want = step(fresh, True)
        for name in ("q", "window", "n", "score", "pos", "lse"):
            captured[name].copy_(refill[name])
        captured["new"].fill_(3)
        g = gen(seed)
        captured["cache"].append(0, randn(g, streams, fresh["cache"].cfg.max_len, 2, D), randn(g, streams, fresh["cache"].cfg.max_len, 2, D))
        torch.cuda.synchronize()
        graph.replay()
        engine.sync_status()
        assert torch.equal(captured["new"], fresh["new"]) and torch.equal(captured["pos"], fresh["pos"])
        assert torch.equal(captured["score"], fresh["score"]) and torch.equal(captured["lse"], fresh["lse"])
        assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.parametrize("kind", ["f16", "q8_0"])
@pytest.mark.parametrize("prefix,rows", [(200, 700), (900, 60), (1500, 900)])
def test_full_row_tiles_of_three_streams_at_once(prefix, rows, kind, engine, pkg):
    """Calls whose prefix kernels (full row tiles, clusters, all of an SM's tensor memory) may meet on the same SMs."""
    import torch
    cases = [SharedCase(engine, pkg, (kind, [s % 2 for s in range(96)], [prefix, prefix - 9], [(rows * (s % 7 + 1)) // 7 for s in range(96)], 16, 2),
                        seed=i) for i in range(3)]
    ws = [torch.zeros(1 << 24, dtype=torch.uint8, device="cuda") for _ in cases]
    want = [c.run(workspace=w)[0].clone() for c, w in zip(cases, ws)]
    engine.sync_status()
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(20):
        got = []
        for c, w, st in zip(cases, ws, streams):
            with torch.cuda.stream(st):
                got.append(c.run(workspace=w)[0])
        torch.cuda.synchronize()
        engine.sync_status()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_a_captured_call_outlives_a_larger_workspace(pkg):
    """A graph captured with the engine's workspace is replayed after a larger call has made the engine take another one."""
    import torch
    engine = pkg.Engine(0)
    c = SharedCase(engine, pkg, ("f16", [0, 0, 0], [300], [500, 9, 0], 16, 2))
    want, lse = c.run()
    dst, graph, side = torch.empty_like(want), torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        c.run(dst=dst, lse=lse)
    before = engine.workspace(0)
    size, at = before.numel(), before.data_ptr()
    del before
    assert engine.workspace(size + 1).data_ptr() != at
    others = [torch.zeros(size, dtype=torch.uint8, device="cuda") for _ in range(64)]
    assert all(o.data_ptr() >= at + size or o.data_ptr() + size <= at for o in others)
    graph.replay()
    engine.sync_status()
    assert torch.equal(dst, want) and not any(bool(o.any()) for o in others)


def test_a_prefix_longer_than_its_cache_is_reported(engine, pkg):
    c = SharedCase(engine, pkg, ("f16", [0, 0], [20], [5, 9], 16, 2))
    c.prefix_len.fill_(c.prefix.cfg.max_len + 1)
    with pytest.raises(pkg.VoxError) as err:
        c.run()
        engine.sync_status()
    assert err.value.status_name == "DEVICE_STATE"
    engine.sync_status()


# ----------------------------------------------------------------------------------------------------------------- refusals

def test_refusals(engine, pkg):
    """Every refusal comes from the host, before a launch, with a reason."""
    import torch
    L = pkg.lib()
    c = SharedCase(engine, pkg, ("f16", [0, 0], [20], [5, 9], 16, 2))
    other_engine = pkg.Engine(0)
    q8 = new_cache(engine, pkg, "q8_0", 1, 1, 2, 32)
    heads = new_cache(engine, pkg, "f16", 1, 1, 4, 32)
    foreign = pkg.KVCache(other_engine, 1, 1, 2, 32)
    launches = engine.launches

    def refused(status, reason, call):
        with pytest.raises(pkg.VoxError, match=reason) as err:
            call()
        assert err.value.status_name == status, str(err.value)

    def shared(**kw):
        a = {"prefix": c.prefix, "plan": c.plan, "prefix_len": c.prefix_len, "prefix_bound": 20, "layer": 0, "q": c.q, "kv_bound": 9} | kw
        return lambda: c.own.decode_shared(a.pop("layer"), a.pop("q"), c.kv_len, a.pop("kv_bound"), **a)

    refused("INVALID_ARGUMENT", "given together", shared(plan=None))
    refused("INVALID_ARGUMENT", "given together", shared(prefix=None))
    refused("INVALID_ARGUMENT", "given together", shared(prefix_len=None))
    refused("INVALID_ARGUMENT", "type or heads", shared(prefix=q8))
    refused("INVALID_ARGUMENT", "type or heads", shared(prefix=heads))
    refused("INVALID_ARGUMENT", "another engine", shared(prefix=foreign))
    refused("INVALID_ARGUMENT", "prefix_bound", shared(prefix_bound=1000))
    refused("INVALID_ARGUMENT", "prefix_bound", shared(prefix_bound=-1))
    refused("INVALID_ARGUMENT", "layer 1 out of range", shared(layer=1))
    refused("INVALID_ARGUMENT", "arranges 3 streams", shared(plan=pkg.PrefixPlan(engine, [0, 0, 0], 1)))
    refused("INVALID_ARGUMENT", "names 2 prefixes", shared(plan=pkg.PrefixPlan(engine, [0, 0], 2)))
    refused("INVALID_ARGUMENT", "heads per kv head", shared(plan=pkg.PrefixPlan(engine, [0, 0], 1, 8, 2)))
    refused("WORKSPACE_TOO_SMALL", "workspace", shared(workspace=torch.empty(16, dtype=torch.uint8, device="cuda")))
    refused("INVALID_ARGUMENT", "kv_bound", shared(kv_bound=5000))
    refused("INVALID_ARGUMENT", "overlap", shared(dst=c.q))
    for of, G in (([0, 1], 1), ([-2, 0], 1)):
        refused("INVALID_ARGUMENT", "prefix_of", lambda: pkg.PrefixPlan(engine, of, G))
    refused("INVALID_ARGUMENT", "must be in", lambda: pkg.PrefixPlan(engine, [], 1))
    refused("INVALID_ARGUMENT", "multiple", lambda: pkg.PrefixPlan(engine, [0], 1, 15, 2))
    refused("UNSUPPORTED", "GQA", lambda: pkg.PrefixPlan(engine, [0], 1, 32, 2))
    refused("INVALID_ARGUMENT", "prefix_of", lambda: c.plan.set([0, 4]))

    o = ObserveCase(engine, pkg, ("f16", [5, 9], 1, 16, 2))
    launches = engine.launches - (launches - launches)

    def observe(n_q=1, **kw):
        q = randn(gen(0), 2, n_q, kw.pop("H", 16), D)
        a = {"layer": 0, "kv_bound": 9} | kw
        return lambda: o.cache.observe(a.pop("layer"), a.pop("q", q), o.kv_len, a.pop("kv_bound"), a.pop("score", o.score), **a)

    refused("UNSUPPORTED", "at most 64", observe(n_q=65))
    refused("UNSUPPORTED", "n_q == 1", observe(n_q=2, lse=torch.zeros(2, 16, device="cuda")))
    refused("UNSUPPORTED", "n_q == 1", observe(n_q=2, rope_table=torch.zeros(2, 32, 2, device="cuda")))
    refused("INVALID_ARGUMENT", "layer", observe(layer=1))
    refused("INVALID_ARGUMENT", "layer", observe(layer=-1))
    refused("INVALID_ARGUMENT", "multiple", observe(H=15))
    refused("UNSUPPORTED", "GQA", observe(H=32))
    refused("INVALID_ARGUMENT", "kv_bound", observe(kv_bound=1 << 20))
    refused("INVALID_ARGUMENT", "n_new", observe(n_new=-1))
    refused("INVALID_ARGUMENT", "8-byte aligned", observe(q=randn(gen(0), 2, 1, 16, D + 1)[..., 1:]))
    refused("WORKSPACE_TOO_SMALL", "workspace", observe(n_q=2, workspace=torch.empty(8, dtype=torch.uint8, device="cuda")))

    for view in (o.score[:, :1].expand(2, 2, -1), o.score[:1].expand(2, 2, -1), o.score.as_strided(o.score.shape, (o.score.stride(0), 4, 1))):
        refused("INVALID_ARGUMENT", "rows overlap", observe(score=view))

    v = EvictCase(engine, pkg, "f16", [30, 20], 2, 2, 32)
    n2 = ints([0, 0])

    def evict(kv_bound=30, budget=10, new_len=n2, **kw):
        return lambda: v.cache.evict(v.kv_len, kv_bound, budget, v.score, v.row_pos, v.n_seen, new_len, **{"n_sink": 0, "n_recent": 0} | kw)

    refused("INVALID_ARGUMENT", "budget", evict(budget=0))
    refused("INVALID_ARGUMENT", "budget", evict(n_sink=6, n_recent=5))
    refused("INVALID_ARGUMENT", "budget", evict(n_sink=-1))
    refused("INVALID_ARGUMENT", "budget", evict(n_sink=2**31 - 1, n_recent=2**31 - 1))
    refused("INVALID_ARGUMENT", "layers", evict(layer0=1))
    refused("INVALID_ARGUMENT", "kv_bound", evict(kv_bound=33))
    for dim in range(3):
        score, pos = (x.narrow(dim, 0, 1).expand_as(x) for x in (v.score, v.row_pos))
        refused("INVALID_ARGUMENT", "rows overlap", lambda: v.cache.evict(v.kv_len, 30, 10, score, pos, v.n_seen, n2, n_sink=0, n_recent=0))
    refused("INVALID_ARGUMENT", "overlap", evict(new_len=v.kv_len))
    refused("INVALID_ARGUMENT", "overlap", evict(new_len=v.n_seen))
    refused("INVALID_ARGUMENT", "overlap", evict(new_len=v.kv_len[1:]))
    other_engine.close()
    out, lse = c.run()
    engine.sync_status()
    check_rows(out, lse, *c.want())


def test_a_plan_is_not_set_inside_a_capture(engine, pkg):
    import torch
    plan = pkg.PrefixPlan(engine, [0, 0], 1)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    x = torch.zeros(4, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        x += 1
        with pytest.raises(pkg.VoxError, match="outside a capture") as err:
            plan.set([0, -1], stream=side)
    assert err.value.status_name == "UNSUPPORTED"
    graph.replay()
    torch.cuda.synchronize()
    assert x.tolist() == [1.0] * 4
