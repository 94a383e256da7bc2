"""What the binding of the bounded-cache operators looks at before it hands addresses to the library.  No GPU: the library is a
recorder, the tensors lie on the CPU, and the engine stands on the "device" that such tensors name (-1)."""
import ctypes as C
import sys

import pytest
import torch

S, H, HK, ROWS, L = 3, 16, 2, 24, 2


class Recorder:
    """In the library's place: notes which entry points are called, and that all is well."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        return lambda *a: self.calls.append(name) or 0


@pytest.fixture
def rig(pkg, monkeypatch):
    binding, recorder = sys.modules[pkg.__name__ + ".binding"], Recorder()
    monkeypatch.setattr(binding, "_LIB", recorder)

    class Rig:
        calls = recorder.calls
        engine = object.__new__(pkg.Engine)
        plans = []  # kept until the end: what a plan that goes asks of the library is not counted

        def cache(self, kind=pkg.F16, streams=S):
            c = object.__new__(pkg.KVCache)
            c.engine, c.cfg, c.h, c._at, c.owned = self.engine, pkg.KVConfig(L, streams, HK, 64, ROWS, kind), C.c_void_p(64), 64, False
            return c

        def plan(self, prefixes=2):
            p = object.__new__(pkg.PrefixPlan)
            p.engine, p.h, p._at, p.n_streams, p.n_prefixes = self.engine, C.c_void_p(128), 128, S, prefixes
            self.plans.append(p)
            return p

    r = Rig()
    r.engine.h, r.engine.device, r.engine._ws, r.engine._ws_at, r.engine._outgrown = C.c_void_p(32), -1, None, (0, 0), []
    yield r
    r.engine.h = None
    for p in r.plans:
        p.h = None


def decode(rig, **kw):
    a = {"cache": rig.cache(), "layer": 0, "q": torch.zeros(S, H, 64), "kv_len": torch.ones(S, dtype=torch.int32), "kv_bound": ROWS,
         "prefix": rig.cache(streams=2), "plan": rig.plan(), "prefix_len": torch.ones(2, dtype=torch.int32), "prefix_bound": 9,
         "dst": torch.zeros(S, H, 64), "lse": torch.zeros(S, H), "k_new": torch.zeros(S, HK, 64), "v_new": torch.zeros(S, HK, 64),
         "rope_table": torch.zeros(S, 32, 2), "workspace": torch.zeros(4096, dtype=torch.uint8), "stream": 0} | kw
    return a.pop("cache").decode_shared(a.pop("layer"), a.pop("q"), a.pop("kv_len"), a.pop("kv_bound"), **a)


def observe(rig, n_q=1, **kw):
    one = n_q == 1
    a = {"cache": rig.cache(), "q": torch.zeros(S, n_q, H, 64), "kv_len": torch.ones(S, dtype=torch.int32), "kv_bound": ROWS,
         "score": torch.zeros(S, HK, ROWS), "row_pos": torch.zeros(S, HK, ROWS, dtype=torch.int32), "n_seen": torch.ones(S, dtype=torch.int32),
         "lse": torch.zeros(S, H) if one else None, "rope_table": torch.zeros(S, 32, 2) if one else None,
         "workspace": torch.zeros(4096, dtype=torch.uint8), "stream": 0} | kw
    a.pop("cache").observe(0, a.pop("q"), a.pop("kv_len"), a.pop("kv_bound"), a.pop("score"), **a)


def evict(rig, budget=8, **kw):
    a = {"cache": rig.cache(), "kv_len": torch.ones(S, dtype=torch.int32), "kv_bound": ROWS, "score": torch.zeros(L, S, HK, ROWS),
         "row_pos": torch.zeros(L, S, HK, ROWS, dtype=torch.int32), "n_seen": torch.ones(S, dtype=torch.int32),
         "new_len": torch.zeros(S, dtype=torch.int32), "kept": torch.zeros(L, S, HK, budget, dtype=torch.int32), "n_sink": 0, "n_recent": 0, "stream": 0} | kw
    a.pop("cache").evict(a.pop("kv_len"), a.pop("kv_bound"), budget, a.pop("score"), a.pop("row_pos"), a.pop("n_seen"), a.pop("new_len"), **a)


def refused(rig, pkg, reason, call, *args, **kw):
    before = len(rig.calls)
    with pytest.raises(pkg.VoxError, match=reason) as err:
        call(rig, *args, **kw)
    assert err.value.status_name == "INVALID_ARGUMENT" and len(rig.calls) == before


def test_a_call_that_fits_goes_to_the_library(rig):
    decode(rig)
    decode(rig, prefix=None, plan=None, prefix_len=None, prefix_bound=0, lse=None, k_new=None, v_new=None, rope_table=None, dst=None)
    observe(rig)
    observe(rig, n_q=5, row_pos=None, n_seen=None)
    evict(rig)
    evict(rig, n_seen=None, kept=None)
    assert rig.calls == ["vox_attn_decode_shared"] * 2 + ["vox_kv_observe"] * 2 + ["vox_kv_evict"] * 2


def test_closed_handles_are_refused(rig, pkg):
    """NULL in the place of a prefix and its plan means that there is none: a closed one must not become NULL."""
    cache, plan = rig.cache(), rig.plan()
    cache.close()
    plan.close()
    for kw in ({"prefix": cache, "plan": plan}, {"prefix": cache}, {"plan": plan}, {"cache": cache}):
        refused(rig, pkg, "closed", decode, **kw)
    refused(rig, pkg, "closed", observe, cache=cache)
    refused(rig, pkg, "closed", evict, cache=cache)


def ints(*shape):
    return torch.ones(shape, dtype=torch.int32)


def wide(x):
    """The same values, every second element of a larger tensor."""
    w = torch.zeros(*x.shape, 2, dtype=x.dtype)
    w[..., 0] = x
    return w[..., 0]


@pytest.mark.parametrize("name,bad", [
    ("q", torch.zeros(S, H, 32)), ("q", torch.zeros(S, H, 64).half()), ("q", wide(torch.zeros(S, H, 64))),
    ("kv_len", ints(S - 1)), ("kv_len", ints(S).long()), ("kv_len", ints(S).float()), ("kv_len", wide(ints(S))),
    ("prefix_len", ints(1)), ("prefix_len", ints(2).long()), ("prefix_len", wide(ints(2))),
    ("k_new", torch.zeros(S, HK, 64).half()), ("k_new", torch.zeros(S, 1, 64)), ("k_new", torch.zeros(S, HK, 65)[..., :64]),
    ("v_new", torch.zeros(S, HK, 64).double()), ("v_new", torch.zeros(S - 1, HK, 64)), ("v_new", torch.zeros(HK, S, 64).transpose(0, 1)),
    ("rope_table", torch.zeros(S, 32)), ("rope_table", torch.zeros(S, 32, 2).half()), ("rope_table", torch.zeros(S, 64, 2)[:, ::2]),
    ("lse", torch.zeros(S, H - 1)), ("lse", torch.zeros(S, H).double()), ("lse", torch.zeros(H, S).T),
    ("dst", torch.zeros(S, H, 63)), ("dst", torch.zeros(S, H, 64).half()), ("dst", torch.zeros(H, S, 64).transpose(0, 1)),
])
def test_decode_shared_looks_at_what_it_passes_on(name, bad, rig, pkg):
    refused(rig, pkg, name, decode, **{name: bad})


@pytest.mark.parametrize("name,bad", [
    ("q", torch.zeros(S, 1, H, 32)), ("q", torch.zeros(S, 1, H, 64).double()),
    ("kv_len", ints(S - 1)), ("kv_len", ints(S).long()), ("kv_len", wide(ints(S))),
    ("n_seen", ints(S).long()), ("n_seen", ints(S - 1)),
    ("lse", torch.zeros(S - 1, H)), ("lse", torch.zeros(S, H).half()), ("lse", torch.zeros(H, S).T),
    ("rope_table", torch.zeros(S, 32)), ("rope_table", torch.zeros(S, 32, 2).double()),
    ("score", torch.zeros(S, 1, ROWS)), ("score", torch.zeros(S, HK, ROWS).half()), ("score", torch.zeros(S - 1, HK, ROWS)),
    ("score", torch.zeros(S, HK, ROWS, 2)[..., 0]),
    ("row_pos", ints(S, HK, ROWS).long()), ("row_pos", ints(S, HK, ROWS + 1)), ("row_pos", ints(S, HK, ROWS + 1)[..., :ROWS]),
])
def test_observe_looks_at_what_it_passes_on(name, bad, rig, pkg):
    refused(rig, pkg, name, observe, **{name: bad})


@pytest.mark.parametrize("name,bad", [
    ("kv_len", ints(S - 1)), ("kv_len", ints(S).long()), ("n_seen", ints(S).long()), ("n_seen", wide(ints(S))),
    ("new_len", ints(S - 1)), ("new_len", ints(S).long()), ("new_len", wide(ints(S))),
    ("score", torch.zeros(L, S, HK + 1, ROWS)), ("score", torch.zeros(L, S, HK, ROWS).double()),
    ("row_pos", ints(L, S, HK, ROWS - 1)), ("row_pos", ints(L, S, HK, ROWS).float()), ("row_pos", ints(L, S, ROWS, HK).transpose(2, 3)),
    ("kept", ints(L, S, HK, 7)), ("kept", ints(L, S, HK, 9)), ("kept", ints(L - 1, S, HK, 8)), ("kept", ints(L, S, HK, 8).long()),
    ("kept", ints(L, S, HK, 9)[..., :8]),
])
def test_evict_looks_at_what_it_passes_on(name, bad, rig, pkg):
    refused(rig, pkg, name, evict, **{name: bad})


def test_scores_of_fewer_rows_than_the_bound_are_refused(rig, pkg):
    """One stream of one kv head has no stride that the library could compare with the bound."""
    refused(rig, pkg, "kv_bound 24 exceeds the 23 rows", observe, score=torch.zeros(S, HK, ROWS - 1), row_pos=None)
    refused(rig, pkg, "kv_bound 24 exceeds the 23 rows", evict, score=torch.zeros(L, S, HK, ROWS - 1), row_pos=ints(L, S, HK, ROWS - 1))


def test_larger_tensors_than_the_call_needs_are_taken(rig):
    """Lengths of more streams than are decoded, rows of more than the bound, strided queries and rows."""
    decode(rig, kv_len=ints(S + 4), prefix_len=ints(9), q=torch.zeros(S, H, 66)[..., :64], k_new=torch.zeros(S, HK, 66)[..., :64],
           v_new=torch.zeros(S, HK, 66)[..., :64])
    score, pos = torch.zeros(S, HK, ROWS + 9)[..., 2: ROWS + 3], ints(S, HK, ROWS + 9)[..., 2: ROWS + 3]
    observe(rig, score=score, row_pos=pos, n_seen=ints(S + 1), kv_len=ints(S + 1))
    evict(rig, score=torch.zeros(S, L, HK, ROWS + 1).transpose(0, 1), row_pos=ints(S, L, HK, ROWS + 1).transpose(0, 1), new_len=ints(S + 1))
    assert rig.calls == ["vox_attn_decode_shared", "vox_kv_observe", "vox_kv_evict"]


def test_tensors_of_another_device_are_refused(rig, pkg):
    rig.engine.device = 0  # the tensors are the host's
    refused(rig, pkg, "on device 0", decode)
    refused(rig, pkg, "on device 0", observe)
    refused(rig, pkg, "on device 0", evict)


@pytest.mark.parametrize("step", [1 << 10, 1 << 20, 50 << 20, 700 << 20])
def test_outgrown_workspaces_do_not_pile_up(step, rig, monkeypatch):
    """Needs that grow a little with every call: the workspaces kept for captured graphs stay in proportion to the largest."""
    class Memory:
        def __init__(self, n, **_):
            self.n = n

        def numel(self):
            return self.n

        def data_ptr(self):
            return 256
    monkeypatch.setattr(torch, "empty", Memory)
    e, largest = rig.engine, 0
    for i in range(1, 400):
        largest = i * step
        ws = e.workspace(largest)
        assert ws.numel() >= largest and e._ws_at == (256, ws.numel())
    assert e._ws.numel() <= max(2 * largest, 256)
    assert e._ws.numel() + sum(w.numel() for w in e._outgrown) <= 6 * largest
    assert len(e._outgrown) < 40


@pytest.mark.parametrize("bad", [[0, 1], [0, 1, 0, 1], [], [[0, 1, 0]], [0.5, 1, 0], [0, 1, float("nan")], torch.tensor([0, 1 << 32, 0]).numpy(), 0])
def test_assignments_that_are_not_one_whole_number_per_stream_are_refused(bad, rig, pkg):
    """The library reads as many numbers as the plan has streams."""
    plan = rig.plan()
    refused(rig, pkg, "prefix_of", lambda rig: plan.set(bad, stream=0))
    plan.set([0, 1, -1], stream=0)
    plan.set(torch.tensor([1, 1, 0]), stream=0)
    assert rig.calls == ["vox_prefix_plan_set"] * 2


def test_a_closed_plan_is_not_set(rig, pkg):
    plan = rig.plan()
    plan.close()
    refused(rig, pkg, "closed", lambda rig: plan.set([0, 1, -1], stream=0))


def test_a_workspace_that_the_device_cannot_use_is_refused(rig, pkg):
    """It is written by the kernels over its whole length."""
    for call in (decode, observe):
        refused(rig, pkg, "workspace", call, workspace=wide(torch.zeros(4096, dtype=torch.uint8)))

    class Elsewhere:
        dtype, device = torch.uint8, "elsewhere"
        get_device = staticmethod(lambda: 5)
        is_contiguous = staticmethod(lambda: True)
        data_ptr = staticmethod(lambda: 256)
        numel = staticmethod(lambda: 4096)
        stride = staticmethod(lambda: (1,))
    for call in (decode, observe):
        refused(rig, pkg, "workspace", call, workspace=Elsewhere())
