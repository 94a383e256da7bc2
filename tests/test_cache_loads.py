"""How the kernels may read cache rows.  CPU only: a look at the sources."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "voxcpm.cpp_b200", "csrc")


@pytest.mark.parametrize("source", ["decode_attn.cu", "shared_decode.cu", "kv_observe.cu", "kv_observe_window.cu", "kv_evict.cu", "kv_cache.cuh"])
def test_cache_rows_are_read_coherently(source):
    """These kernels may be resident while the launch in front of them still writes rows (programmatic dependent launch), which the
    non-coherent load path (__ldg, ld.global.nc) does not allow for memory that they read."""
    text = re.sub(r"//[^\n]*|/\*.*?\*/", "", open(os.path.join(CSRC, source)).read(), flags=re.S)
    assert not re.findall(r"__ldg\s*\(|\bld\.global(?:\.\w+)*\.nc\b", text)
