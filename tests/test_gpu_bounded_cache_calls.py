"""Calls of the bounded-cache operators that must be refused, and what the operators promise about calls in a row: beside
test_gpu_bounded_cache.py, whose cases and definitions these use."""
import contextlib
import ctypes

import numpy as np
import pytest
import test_gpu_bounded_cache as cases
from test_bounded_cache_border import scores_with_a_bin_of
from test_gpu_bounded_cache import OBSERVE, WEIGHT, D, EvictCase, ObserveCase, SharedCase, gen, ints, new_cache, randn

pytestmark = pytest.mark.gpu


def refuses(engine, pkg, reason, call, status="INVALID_ARGUMENT"):
    """The host refuses, with a reason, and nothing is launched."""
    launches = engine.launches
    with pytest.raises(pkg.VoxError, match=reason) as err:
        call()
    assert err.value.status_name == status, str(err.value)
    assert engine.launches == launches


def test_half_a_prefix_is_refused(engine, pkg):
    """Neither a prefix nor a plan, but lengths of prefixes or a bound of them: not a call for the streams' own rows."""
    c = SharedCase(engine, pkg, ("f16", [0, 0], [20], [5, 9], 16, 2))

    def call(**kw):
        return lambda: c.own.decode_shared(0, c.q, c.kv_len, 9, **kw)

    refuses(engine, pkg, "given together", call(prefix_len=c.prefix_len))
    refuses(engine, pkg, "given together", call(prefix_bound=20))
    refuses(engine, pkg, "given together", call(prefix_len=c.prefix_len, prefix_bound=20))
    call()()
    engine.sync_status()


def test_a_stream_that_is_appended_to_is_no_prefix_of_the_call(engine, pkg):
    """The row that arrives would be stored while the prefix is read.  Without one the streams may be each other's prefixes."""
    import torch
    cache = new_cache(engine, pkg, "f16", 1, 4, 2, 64)
    cache.append(0, randn(gen(1), 4, 64, 2, D), randn(gen(2), 4, 64, 2, D))
    q, new, n, P = randn(gen(3), 2, 16, D), randn(gen(4), 2, 2, D), [20, 33], [30, 40, 50, 60]

    def call(of, **kw):
        return lambda: cache.decode_shared(0, q, ints(n), 64, prefix=cache, plan=pkg.PrefixPlan(engine, of, 4), prefix_len=ints(P), prefix_bound=60, **kw)

    for of in ([0, 2], [3, 1], [-1, 0]):
        refuses(engine, pkg, "is a prefix and one of the 2", call(of, k_new=new, v_new=new))
    plan = pkg.PrefixPlan(engine, [2, 3], 4)
    plan.set([2, 1])
    refuses(engine, pkg, "is a prefix", lambda: cache.decode_shared(0, q, ints(n), 64, prefix=cache, plan=plan, prefix_len=ints(P), prefix_bound=60,
                                                                    k_new=new, v_new=new))
    for of in ([1, 0], [2, 3]):
        out = call(of)()
        engine.sync_status()
        for s in range(2):
            kv = [torch.cat([a, b], 1) for a, b in zip(cases.stored(cache, pkg, 0, of[s], P[of[s]]), cases.stored(cache, pkg, 0, s, n[s]))]
            want, _ = cases.attend(q[s].double(), *kv, 0.125)
            cases.check_rows(out[s], None, want, None)
    call([2, 3], k_new=new, v_new=new)()
    call([-1, -1], k_new=new, v_new=new)()
    engine.sync_status()


# what else lies over one another is tried on the host's own look at it: test_row_lists.py

def colliding(torch, lists, rows, dtype=None):
    """Lists whose last two extents have the same stride, one row list each: the second stream's first head is the first's second."""
    flat = torch.zeros(8 * rows, device="cuda", dtype=dtype)
    return flat.as_strided((*lists, rows), (*[lists[-1] * lists[-2] * rows] * (len(lists) - 2), rows, rows, 1))


def test_row_lists_over_one_another_are_refused_by_observe(engine, pkg):
    import torch
    c = ObserveCase(engine, pkg, ("f16", [5, 9], 1, 16, 2))
    rows = c.score.shape[2]

    def call(score, **kw):
        a = {"kv_len": c.kv_len, "row_pos": None} | kw
        return lambda: c.cache.observe(0, c.q, a.pop("kv_len"), 9, score, **a)

    both = torch.zeros((2, 2, 2, rows), device="cuda")  # scores and positions, list beside list
    score, pos = both[:, :, 0], both.view(torch.int32)[:, :, 1]
    refuses(engine, pkg, "rows overlap", call(colliding(torch, (2, 2), rows)))
    refuses(engine, pkg, "score and row_pos overlap", call(score, row_pos=score.view(torch.int32)))
    refuses(engine, pkg, "score and row_pos overlap", call(score, row_pos=both.view(torch.int32).as_strided(score.shape, score.stride(), 8)))
    refuses(engine, pkg, "not overlap kv_len", call(score, kv_len=score.view(torch.int32)[1, 1, 7:9]))
    refuses(engine, pkg, "not overlap kv_len", call(score, row_pos=pos, n_seen=pos[0, 1, :2]))
    refuses(engine, pkg, "not overlap lse", call(both.view(2, 2, 2 * rows)[..., :rows], lse=both.view(-1)[rows - 1: rows + 31].view(2, 16)))
    call(score, row_pos=pos, n_seen=ints([5, 9]), n_new=9)()
    engine.sync_status()
    assert pos[0, 0, :5].tolist() == list(range(5)) and float((score[1, 1, :9].sum() - 8).abs()) < 1e-5


def test_row_lists_over_one_another_are_refused_by_evict(engine, pkg):
    import torch
    c = EvictCase(engine, pkg, "f16", [30, 20], 2, 2, 32)
    n2, kept = ints([0, 0]), torch.zeros((2, 2, 2, 10), dtype=torch.int32, device="cuda")

    def call(score=c.score, row_pos=c.row_pos, new_len=n2, kv_len=c.kv_len, kept=kept, **kw):
        return lambda: c.cache.evict(kv_len, 30, 10, score, row_pos, c.n_seen, new_len, n_sink=0, n_recent=0, kept=kept, **kw)

    flat = c.score.view(torch.int32).view(-1)
    refuses(engine, pkg, "rows overlap", call(colliding(torch, (2, 2, 2), 32), colliding(torch, (2, 2, 2), 32, torch.int32)))
    refuses(engine, pkg, "score and row_pos overlap", call(row_pos=c.score.view(torch.int32)))
    refuses(engine, pkg, "kept must not overlap score", call(kept=flat[40:120].view(2, 2, 2, 10)))
    refuses(engine, pkg, "kept must not overlap score", call(kept=c.row_pos.view(-1)[:80].view(2, 2, 2, 10)))
    refuses(engine, pkg, "not overlap kv_len", call(new_len=flat[3:5]))
    refuses(engine, pkg, "not overlap kv_len", call(kv_len=c.row_pos[1, 1, 1, 28:30]))
    refuses(engine, pkg, "kept must not overlap kv_len", call(new_len=kept.view(-1)[7:9]))
    refuses(engine, pkg, "kept must not overlap kv_len", call(kv_len=kept.view(-1)[78:]))
    c.check(10)


@pytest.mark.parametrize("kind", ["f16", "q8_0"])
def test_a_captured_loop_loses_no_row_that_it_keeps(kind, engine, pkg):
    """A step as it is documented, one graph: kv_len = new_len + 1 and n_seen + 1 on the device, decode with the arriving row, weights,
    eviction.  Replayed far past the budget, every row that is left is the one that its position was given when it arrived, the newest
    among them, and the outputs are those of the calls made one at a time with lengths from the host."""
    import torch
    S, budget, rows, layers, of, P = 4, 40, 64, 2, [0, 1, -1, 0], [70, 9]
    start = np.array([3, 39, 40, 20])
    prefix = new_cache(engine, pkg, kind, layers, 2, 2, 72)
    for layer in range(layers):
        prefix.append(layer, randn(gen(layer), 2, 72, 2, D), randn(gen(9 + layer), 2, 72, 2, D))
    plan, prefix_len, behind = pkg.PrefixPlan(engine, of, 2), ints(P), ints([P[p] if p >= 0 else 0 for p in of])

    class State:
        def __init__(self):
            self.cache = new_cache(engine, pkg, kind, layers, S, 2, rows)
            for layer in range(layers):
                self.cache.append(layer, randn(gen(20 + layer), S, rows, 2, D), randn(gen(30 + layer), S, rows, 2, D))
            self.score = torch.zeros((layers, S, 2, rows), device="cuda")
            self.pos = torch.arange(rows, dtype=torch.int32, device="cuda").expand(layers, S, 2, -1).contiguous()
            self.kv_len, self.new_len, self.n_seen = ints(start * 0), ints(start), ints(start)
            self.q, self.k, self.v = (torch.zeros((layers, S, n, D), device="cuda") for n in (16, 2, 2))
            self.lse, self.out = torch.zeros((layers, S, 16), device="cuda"), torch.zeros((layers, S, 16, D), device="cuda")
            self.ws = torch.zeros(1 << 22, dtype=torch.uint8, device="cuda")

        def step(self):
            table = engine.rope_table(self.n_seen + behind, pos_offset=-1)
            for layer in range(layers):
                self.cache.decode_shared(layer, self.q[layer], self.kv_len, rows, prefix=prefix, plan=plan, prefix_len=prefix_len, prefix_bound=72,
                                         k_new=self.k[layer], v_new=self.v[layer], rope_table=table, lse=self.lse[layer], dst=self.out[layer],
                                         workspace=self.ws)
                self.cache.observe(layer, self.q[layer][:, None], self.kv_len, rows, self.score[layer], row_pos=self.pos[layer],
                                   n_seen=self.n_seen, lse=self.lse[layer], rope_table=table, workspace=self.ws)
            self.cache.evict(self.kv_len, rows, budget, self.score, self.pos, self.n_seen, self.new_len, n_sink=1, n_recent=6)

        def step_on_device(self):
            torch.add(self.new_len, 1, out=self.kv_len)
            self.n_seen += 1
            self.step()

    looped, eager = State(), State()
    here = [{(s, h, j): looped.cache.export(layer, s, start[s])[0][h, j].tobytes() for s in range(S) for h in range(2) for j in range(start[s])}
            for layer in range(layers)]
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        looped.step_on_device()
    n, seen = start.copy(), start.copy()
    g = gen(50)
    for t in range(60):
        for x in "qkv":
            new = randn(g, *getattr(looped, x).shape)
            getattr(looped, x).copy_(new)
            getattr(eager, x).copy_(new)
        graph.replay()
        engine.sync_status()
        n, seen = n + 1, seen + 1
        eager.kv_len.copy_(ints(n))
        eager.n_seen.copy_(ints(seen))
        eager.step()
        engine.sync_status()
        n = np.minimum(n, budget)
        assert looped.new_len.tolist() == n.tolist() and looped.n_seen.tolist() == seen.tolist()
        for name in ("out", "lse", "score", "pos"):
            assert torch.equal(getattr(looped, name), getattr(eager, name)), (t, name)
        pos = looped.pos.cpu().numpy()
        for layer in range(layers):
            for s in range(S):
                k = looped.cache.export(layer, s, n[s])[0]
                for h in range(2):
                    at = pos[layer, s, h, : n[s]]
                    assert len(set(at)) == n[s] and seen[s] - 1 in at
                    for j, p in enumerate(at):
                        if p == seen[s] - 1:
                            here[layer][s, h, p] = k[h, j].tobytes()
                        assert here[layer][s, h, p] == k[h, j].tobytes(), (t, layer, s, h, j, p)


def test_calls_under_another_device_are_refused(engine, pkg):
    """With another device current a stream (the default one above all) would be that device's.  One device is enough for this test: the
    engine is told that it belongs to the next one."""
    c, o, v = (SharedCase(engine, pkg, ("f16", [0, 0], [20], [5, 9], 16, 2)), ObserveCase(engine, pkg, ("f16", [5, 9], 1, 16, 2)),
               EvictCase(engine, pkg, "f16", [30, 20], 1, 2, 32))
    n2 = ints([0, 0])
    calls = [lambda: c.run(stream=0), lambda: o.run(stream=0), lambda: c.plan.set([0, -1], stream=0),
             lambda: v.cache.evict(v.kv_len, 30, 10, v.score, v.row_pos, v.n_seen, n2, n_sink=0, n_recent=0, stream=0)]
    engine.sync_status()
    device = ctypes.c_int.from_address(engine.h.value)  # the engine's first member
    assert device.value == 0
    try:
        device.value = 1
        for call in calls:
            refuses(engine, pkg, "device 1 must be the current", call)
    finally:
        device.value = 0
    c.check()


# q8_0 values over many magnitudes.  The weights, each times its row's scale, travel as two f16 parts in units that follow the largest
# such product of a query row so far: 2^-25 / 32 of it is the most that a part's rounding takes off a product, 8 * 2^-30 of the
# result's RMS (one of 64 columns at least is at its block's largest), and over n rows the square root of n times that: 4e-7 for 3000.
# Scores are sums of 64 products of at most 5 (the one that tells rows apart) and about 0.1 (the others), added up in f32: a few times
# 2^-24 * 5.  1e-5 of the result, which the header promises, leaves a factor of ten.
FORMS = {  # streams, own rows, prefix rows: which kernel takes the prefix
    "small row tiles": (2, 200, 512),
    "full row tiles beside long streams": (40, 3000, 512),
    "full row tiles, two groups": (20, 64, 512),
    "own rows only": (3, 1500, 0),
    "one tile": (2, 30, 30),
}


def magnitudes(engine, pkg, form, k0, v_size):
    """Rows j of n whose first K element is k0(j / n) and whose V rows are v_size(j / n) times as large; queries whose first element is 8, so
    that a row's score is k0 and something of standard deviation 1."""
    import torch
    streams, own, prefix = FORMS[form]
    c = SharedCase(engine, pkg, ("q8_0", [0 if prefix else -1] * streams, [prefix], [own, max(1, own // 3)] * (streams // 2) + [own] * (streams % 2), 16, 2),
                   junk=False)
    for i, (cache, n) in enumerate(((c.own, own), (c.prefix, prefix))):
        rows = cache.cfg.max_len
        k, v = randn(gen(3 + i), cache.cfg.n_streams, rows, 2, D), randn(gen(5 + i), cache.cfg.n_streams, rows, 2, D)
        at = (torch.arange(rows, device="cuda", dtype=torch.float64) / max(n, 1)).float()
        k[..., 0] = k0(at)[None, :, None]
        cache.append(0, k, v * v_size(at)[None, :, None, None])
    c.q[..., 0] = 8.0
    out, lse = c.run()
    engine.sync_status()
    want, want_lse = c.want()
    assert float((lse.double() - want_lse).abs().max()) < 6e-5
    error = (out.double() - want).norm(dim=-1) / want.norm(dim=-1).clamp(min=1e-30)  # of every stream and head (nothing but zeros: none)
    assert float(error.max()) < 1e-5, float(error.max())


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("size", [1e2, 1e4, 1e6])
@pytest.mark.parametrize("where", [0.0, 0.4, 0.96])
def test_a_large_row_of_no_weight_takes_nothing_off_the_others(form, size, where, engine, pkg):
    """A few V rows are far larger than the others and their keys far away (e^-40)."""
    import torch
    there = lambda at: (at >= where) & (at < where + 0.04)  # noqa: E731
    magnitudes(engine, pkg, form, lambda at: torch.where(there(at), -40.0, 0.0), lambda at: torch.where(there(at), size, 1.0))


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("rise", [6.0, 40.0, 200.0])
def test_large_rows_first_and_the_weight_behind(form, rise, engine, pkg):
    """The weight rises along the rows while their size falls: what was largest when it was met is next to nothing at the end."""
    import torch
    magnitudes(engine, pkg, form, lambda at: rise * (at - 1.0), lambda at: 10.0 ** (6.0 * (0.5 - at.clamp(max=1.0))))


@pytest.mark.parametrize("form", FORMS)
def test_rows_of_zeros_beside_others(form, engine, pkg):
    """V rows of nothing (scale 0) carry all the weight at first."""
    import torch
    magnitudes(engine, pkg, form, lambda at: torch.where(at < 0.5, 0.0, -6.0), lambda at: torch.where(at < 0.5, 0.0, 1.0))


def test_no_refusal_launches_anything(engine, pkg, monkeypatch):
    """All of test_refusals again, with a look at the launch count around every refused call."""
    seen = []

    class Counting:
        @staticmethod
        @contextlib.contextmanager
        def raises(*args, **kw):
            before = engine.launches
            with pytest.raises(*args, **kw) as err:
                yield err
            assert engine.launches == before
            seen.append(err)

    monkeypatch.setattr(cases, "pytest", Counting)
    cases.test_refusals(engine, pkg)
    assert len(seen) >= 40


# The weights themselves, to the relative error that their derivation allows (test_gpu_bounded_cache.py: 1.2e-4, whatever their size: a score's
# error does not depend on it).  From scores of 0, since beside an old score of about 1 a weight of 1 / rows could be missing and
# not be seen; 1e-30: weights below 2^-126 count as 0.

def check_weights(c, n_new=1):
    c.score.zero_()
    want, pos = c.want(n_new, 0.75)
    c.run(n_new, 0.75)
    c.engine.sync_status()
    error = (c.score.double() - want).abs() - WEIGHT * want - 1e-30
    assert float(error.max()) <= 0, float(((c.score.double() - want).abs() / want.clamp(min=1e-30)).max())
    # and beside old scores of the weights' size: one addition more, rounded once
    rows = float(np.mean([max(n, 1) for n in c.n]))
    c.score.copy_(randn(gen(1), *c.score.shape).abs() * (c.n_q * c.H / c.HK / rows))
    old = c.score.double().clone()
    both, _ = c.want(n_new, 0.75)
    c.run(n_new, 0.75)
    c.engine.sync_status()
    live = cases.cuda(np.arange(old.shape[-1])[None] < np.array(c.n)[:, None])[:, None]
    error = ((c.score.double() - both).abs() - WEIGHT * want - 2.0 ** -23 * both)[live.expand_as(both)]
    assert float(error.max()) <= 0
    assert bool((c.score.double() == old)[~live.expand_as(both)].all())


@pytest.mark.parametrize("case", OBSERVE)
def test_every_weight_to_its_relative_error(case, engine, pkg):
    check_weights(ObserveCase(engine, pkg, case), n_new=OBSERVE[case][2])


@pytest.mark.parametrize("given_lse", [True, False])
@pytest.mark.parametrize("kind,streams,rows", [("f16", 128, 4700), ("q8_0", 64, 9300), ("f16", 12, 24576), ("q8_0", 9, 26000)])
def test_every_weight_of_many_long_streams(kind, streams, rows, given_lse, engine, pkg):
    lens = [min(rows, max(0, 512 * (i % 11) + (0, 1, -1, 64, 257)[i % 5])) for i in range(streams - 2)] + [rows, rows - 1]
    check_weights(ObserveCase(engine, pkg, (kind, lens, 1, 4, 2), given_lse=given_lse))


@pytest.mark.parametrize("kind,streams,rows", [("f16", 128, 4700), ("q8_0", 64, 9300)])
@pytest.mark.parametrize("n_q", [3, 46, 49])
def test_every_weight_of_a_window_over_many_long_streams(kind, streams, rows, n_q, engine, pkg):
    lens = [min(rows, max(0, 512 * (i % 11) + (0, 1, -1, 64, 257)[i % 5])) for i in range(streams - 2)] + [rows, rows - 1]
    check_weights(ObserveCase(engine, pkg, (kind, lens, n_q, 4, 2)), n_new=2)


@pytest.mark.parametrize("kind", ["f16", "q8_0"])
@pytest.mark.parametrize("n_q,heads,kv_heads", [(13, 16, 2), (28, 16, 2), (44, 16, 2), (64, 16, 2), (43, 18, 3), (50, 4, 4)])
def test_every_weight_of_wide_windows(n_q, heads, kv_heads, kind, engine, pkg):
    check_weights(ObserveCase(engine, pkg, (kind, [4 * ((i * 37) % 97) + 1 for i in range(73)] + [2600], n_q, heads, kv_heads)), n_new=2)


@pytest.mark.parametrize("count", [97, 255, 256, 257])
def test_eviction_where_the_border_is_in_a_full_bin(count, engine, pkg):
    """As many keys in the border's bin as are ranked against one another, one more and one less."""
    c = EvictCase(engine, pkg, "f16", [700, 700], 1, 2, 704)
    w = np.zeros(c.score.shape, np.float32)
    for s in range(2):
        for h in range(2):
            w[0, s, h, :700] = scores_with_a_bin_of(count, 700, 4 * s + h)
    above = int((w[0, 0, 0] >= 1.25).sum())
    c.score.copy_(cases.cuda(w))
    c.row_pos.copy_(c.row_pos + 100)
    c.check(above + count // 2)


@pytest.mark.parametrize("kind", ["f16", "q8_0"])
@pytest.mark.parametrize("streams,prefix", [(64, 8000), (256, 8000), (40, 16000)])
def test_full_row_tiles_under_long_prefixes(kind, streams, prefix, engine, pkg):
    """The tensor core truncates a sum once every 32 keys (sums of even and of odd tiles of 64 keys apart, 16 keys a product), by less than
    2^-23 of it and half of that on average.  A CTA's share of the keys is the prefix over the CTAs of a cluster: as many as there are
    SMs for, eight at most."""
    tiles = 2 * -(-streams // 16)
    share = prefix / min(8, 148 // tiles)
    c = SharedCase(engine, pkg, (kind, [0] * streams, [prefix], [1 + s % 3 for s in range(streams)], 16, 2), junk=False)
    out, lse = c.run()
    engine.sync_status()
    want, want_lse = c.want()
    assert float((out.double() - want).norm() / want.norm()) < share / 32 * 2.0 ** -23 + 5e-7
    assert float((lse.double() - want_lse).abs().max()) < 6e-5
