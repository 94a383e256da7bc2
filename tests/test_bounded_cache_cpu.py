"""Entry points of the bounded-cache operators without a GPU: null arguments and size queries."""
import ctypes as C

import pytest


@pytest.fixture(scope="module")
def L(pkg):
    return pkg.lib()


def test_null_arguments_are_refused(pkg, L):
    out = C.c_void_p(1)
    assert L.vox_prefix_plan_create(None, 1, 1, 16, 2, None, C.byref(out)) == 1
    assert L.vox_prefix_plan_create(None, 1, 1, 16, 2, None, None) == 1
    assert L.vox_prefix_plan_set(None, None, None) == 1
    L.vox_prefix_plan_destroy(None)
    assert L.vox_attn_decode_shared(None, None, None, 0, None) == 1
    assert L.vox_attn_decode_shared(None, C.byref(pkg.DecodeSharedArgs()), None, 0, None) == 1
    assert L.vox_kv_observe(None, None, None, 0, None) == 1
    assert L.vox_kv_observe(None, C.byref(pkg.ObserveArgs()), None, 0, None) == 1
    assert b"null argument" in L.vox_attn_last_error_string()
    assert L.vox_kv_evict(None, None, None) == 1
    assert L.vox_kv_evict(None, C.byref(pkg.EvictArgs()), None) == 1


def test_size_queries_of_nothing(pkg, L):
    assert L.vox_attn_decode_shared_workspace_bytes(None) == 0
    assert L.vox_attn_decode_shared_workspace_bytes(C.byref(pkg.DecodeSharedArgs())) == 0
    assert L.vox_kv_observe_workspace_bytes(None) == 0
    assert L.vox_kv_observe_workspace_bytes(C.byref(pkg.ObserveArgs())) == 0


@pytest.mark.parametrize("name", ["DecodeSharedArgs", "ObserveArgs", "EvictArgs"])
def test_packed_argument_blocks_are_the_structures(pkg, name):
    """The bytes that the binding packs are those of the ctypes structure with the same values."""
    cls = getattr(pkg, name)

    def fill(c, values):
        x = c()
        for field, t in c._fields_:
            if issubclass(t, C.Structure):
                setattr(x, field, fill(t, values))
            else:
                values.append(len(values) + (0.25 if t is C.c_float else 3))
                setattr(x, field, values[-1])
        return x
    values = []
    want = fill(cls, values)
    binding = __import__("sys").modules[pkg.__name__ + ".binding"]
    got = cls.from_buffer_copy(binding._packer(cls)(*values))

    def same(a, b):
        for field, t in a._fields_:
            x, y = getattr(a, field), getattr(b, field)
            same(x, y) if issubclass(t, C.Structure) else _equal(x, y)
    same(got, want)


def _equal(x, y):
    assert x == y
