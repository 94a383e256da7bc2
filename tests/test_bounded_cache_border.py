"""The border that vox_kv_evict finds, as the kernel looks for it: the keys of a bin are ranked against one another if they are no more
than the threads of its CTA (test_bounded_cache_schedule.py restates the search with a smaller limit)."""
import os
import re

import numpy as np
import pytest
from test_bounded_cache_schedule import border, keys_of

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "voxcpm.cpp_b200", "csrc")
RANKED = 256


def scores_with_a_bin_of(count, n, seed):
    """n scores of which `count` fall into one bin (a quarter of an octave: from 1 to 1.25), the others on both sides of it."""
    rng = np.random.default_rng(seed)
    w = np.concatenate([rng.uniform(1.0, 1.2499, count), rng.uniform(0.01, 0.99, (n - count) // 2), rng.uniform(1.26, 9.0, n - count - (n - count) // 2)])
    return rng.permutation(w).astype(np.float32)


def test_the_limit_is_the_kernels():
    text = open(os.path.join(CSRC, "kv_evict.cu")).read()
    assert re.search(r"kThreads\s*=\s*%d;" % RANKED, text) and re.search(r"kRanked\s*=\s*kThreads;", text)


def stays(key, budget):
    edge, last = border(key, budget, ranked=RANKED)
    i = np.arange(len(key))
    return (key > edge) | ((key == edge) & (i <= last))


def largest(key, budget):
    want = np.zeros(len(key), bool)
    want[np.lexsort((np.arange(len(key)), -key.astype(np.int64)))[:budget]] = True
    return want


@pytest.mark.parametrize("count", [1, 95, 97, 255, 256, 257, 400])
@pytest.mark.parametrize("ties", [False, True])
def test_bins_on_both_sides_of_the_limit(count, ties):
    w = scores_with_a_bin_of(count, 700, count)
    if ties:
        w = np.floor(w * 64).astype(np.float32) / 64
    key = keys_of(w.copy(), np.zeros(700, bool))
    above = int((w >= 1.25).sum())
    for budget in {above + 1, above + count // 2 or 1, above + count, max(1, above), 699}:
        assert np.array_equal(stays(key, budget), largest(key, budget))


@pytest.mark.parametrize("seed", range(60))
def test_any_scores(seed):
    rng = np.random.default_rng(seed)
    n = int(rng.integers(2, 3000))
    w = rng.random(n).astype(np.float32)
    score = [w, np.where(w < 0.7, np.float32(0), w), (1 + np.floor(w * 50) * 2.0 ** -23).astype(np.float32),
             np.exp2(w * 250 - 125).astype(np.float32)][seed % 4]
    score[rng.random(n) < 0.02] = np.nan
    safe = rng.random(n) < 0.05
    key = keys_of(score.copy(), safe)
    budget = int(rng.integers(max(1, safe.sum()), n))
    assert np.array_equal(stays(key, budget), largest(key, budget))
