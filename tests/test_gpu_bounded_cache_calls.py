"""Calls of the bounded-cache operators that must be refused, and what the operators promise about calls in a row: beside
test_gpu_bounded_cache.py, whose cases and definitions these use."""
import pytest
from test_gpu_bounded_cache import EvictCase, ObserveCase, SharedCase, ints

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
