"""Calls of the bounded-cache operators that must be refused, and what the operators promise about calls in a row: beside
test_gpu_bounded_cache.py, whose cases and definitions these use."""
import pytest
from test_gpu_bounded_cache import SharedCase

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
