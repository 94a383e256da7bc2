"""Host-side restatements of how the bounded-cache operators cut their work, with the properties the kernels rely on."""
import numpy as np
import pytest

KEYS, CTAS = 128, 148


# ------------------------------------------------------- vox_kv_observe, windows: parts of (stream, kv head) row lists

def window_parts(lens, kv_heads, n_ctas):
    """find_part of kv_observe_window.cu for every part: (stream, kv head, first tile, tiles, first slot, slots)."""
    tiles = [-(-n // KEYS) for n in lens]
    total, live, most = sum(tiles) * kv_heads, sum(t > 0 for t in tiles) * kv_heads, max(tiles, default=0)
    if total == 0:
        return []
    r = most if live >= n_ctas else -(-total // n_ctas)
    while r < most and sum(-(-t // r) for t in tiles) * kv_heads > n_ctas:
        r += 1
    parts, b = [], 0
    for s, t in enumerate(tiles):
        np_ = -(-t // r)
        for i in range(np_ * kv_heads):
            j = i % np_
            first = j * t // np_
            parts.append((s, i // np_, first, (j + 1) * t // np_ - first, b - j, np_))
            b += 1
    return parts


@pytest.mark.parametrize("seed", range(40))
def test_window_parts_cover_every_tile_once(seed):
    rng = np.random.default_rng(seed)
    S, HK = int(rng.integers(1, 300)), int(rng.integers(1, 9))
    lens = [int(x) for x in rng.integers(0, 2 ** rng.integers(1, 15), S)]
    parts = window_parts(lens, HK, CTAS)
    seen = {}
    for b, (s, h, first, n, slot, slots) in enumerate(parts):
        assert n >= 1 and slot <= b < slot + slots and parts[slot][:2] == (s, h) and parts[slot + slots - 1][:2] == (s, h)
        for t in range(first, first + n):
            assert seen.setdefault((s, h, t), b) == b
    assert len(seen) == sum(-(-n // KEYS) for n in lens) * HK
    # the statistics' workspace has a slot for each
    assert len(parts) <= max(CTAS, S * HK)
    if parts and sum(n > 0 for n in lens) * HK < CTAS:
        assert len(parts) <= CTAS


# ------------------------------------------------------- vox_attn_decode_shared: row tiles, clusters and shares of rows

def arrange(prefix_of, n_prefixes, per_tile):
    """arrange() of shared_decode.cu: tiles (prefix, streams) and their members."""
    tiles, members, first = [], [], []
    for g in range(n_prefixes):
        first.append(len(tiles))
        for left in range(sum(p == g for p in prefix_of), 0, -per_tile):
            tiles.append((g, min(left, per_tile)))
            members.append([None] * per_tile)
    come = [0] * n_prefixes
    for s, g in enumerate(prefix_of):
        if g >= 0:
            j = come[g]
            come[g] += 1
            members[first[g] + j // per_tile][j % per_tile] = s
    return tiles, members


@pytest.mark.parametrize("seed", range(40))
def test_row_tiles_hold_every_sharing_stream_once(seed):
    rng = np.random.default_rng(seed)
    S, G, gqa = int(rng.integers(1, 300)), int(rng.integers(1, 20)), int(rng.integers(1, 9))
    prefix_of = [int(x) for x in rng.integers(-1, G, S)]
    for rows in (128, 64, 32, 16):
        per_tile = rows // gqa
        tiles, members = arrange(prefix_of, G, per_tile)
        assert len(tiles) <= S // per_tile + min(S, G)  # max_tiles
        found = []
        for (g, n), m in zip(tiles, members):
            assert 1 <= n and n * gqa <= rows and None not in m[:n] and set(m[n:]) <= {None}
            assert all(prefix_of[s] == g for s in m[:n])
            found += m[:n]
        assert sorted(found) == [s for s in range(S) if prefix_of[s] >= 0]


def cluster_size(n_tiles, kv_heads, n_keys, full):
    useful = max(-(-n_keys // KEYS), 4 if full else 1)
    return max(1, min(8, CTAS // max(1, n_tiles * kv_heads), useful))


@pytest.mark.parametrize("seed", range(40))
def test_a_cluster_shares_out_keys_and_rows(seed):
    """Every key of a prefix belongs to one CTA, every row of the tile is joined by one; a share fits the memory behind the parts."""
    rng = np.random.default_rng(seed)
    rows, length = int(rng.integers(1, 129)), int(rng.integers(1, 2 ** rng.integers(1, 15)))
    bound = int(rng.integers(1, length + 300))
    for full in (False, True):
        C = cluster_size(int(rng.integers(1, 40)), int(rng.integers(1, 9)), bound, full)
        n = -(-length // KEYS)
        keys = [(r * n // C * KEYS, min(length, (r + 1) * n // C * KEYS)) for r in range(C)]
        assert keys[0][0] == 0 and keys[-1][1] == length
        assert all(a[1] == b[0] or b[0] >= length for a, b in zip(keys, keys[1:]))
        shares = [((r * rows) // C, ((r + 1) * rows) // C) for r in range(C)]
        assert shares[0][0] == 0 and shares[-1][1] == rows and all(a[1] == b[0] for a, b in zip(shares, shares[1:]))
        if C > 1:
            assert max(b - a for a, b in shares) <= 64


# ------------------------------------------------------- vox_kv_evict: the border by bins

def keys_of(score, safe):
    """ordered() of kv_evict.cu."""
    bits = (score + np.float32(0)).view(np.uint32)
    key = np.where(bits >> 31, ~bits, bits | np.uint32(0x80000000)).astype(np.uint32)
    key[np.isnan(score)] = 0
    key[safe] = 0xFFFFFFFF
    return key


def border(key, budget, ranked=96):
    """The (edge, last) of evict_kernel: keys above edge stay, and those equal to it up to index last."""
    edge, mask, need, last, shift, width = 0, 0, budget, len(key), 21, 11
    while True:
        here = (key & np.uint32(mask)) == edge
        hist = np.bincount((key[here] >> np.uint32(shift)) & np.uint32((1 << width) - 1), minlength=1 << width)
        before = 0
        for b in range((1 << width) - 1, -1, -1):
            if before + hist[b] >= need:
                break
            before += hist[b]
        edge |= b << shift
        mask |= ((1 << width) - 1) << shift
        need -= before
        inside = np.flatnonzero((key & np.uint32(mask)) == edge)
        if shift == 0:
            return edge, int(inside[need - 1]) if hist[b] > need else last
        if hist[b] <= ranked:
            order = inside[np.lexsort((inside, -key[inside].astype(np.int64)))]
            return int(key[order[need - 1]]), int(order[need - 1])
        width, shift = min(11, shift), max(0, shift - 11)


@pytest.mark.parametrize("seed", range(60))
def test_the_border_leaves_the_largest_keys(seed):
    rng = np.random.default_rng(seed)
    n = int(rng.integers(2, 3000))
    kind = seed % 4
    w = rng.random(n).astype(np.float32)
    score = [w, np.where(w < 0.7, np.float32(0), w), (1 + np.floor(w * 50) * 2.0 ** -23).astype(np.float32), np.exp2(w * 250 - 125).astype(np.float32)][kind]
    score[rng.random(n) < 0.02] = np.nan
    safe = rng.random(n) < 0.05
    key = keys_of(score.copy(), safe)
    budget = int(rng.integers(max(1, safe.sum()), n))
    edge, last = border(key, budget)
    i = np.arange(n)
    stays = (key > edge) | ((key == edge) & (i <= last))
    want = np.zeros(n, bool)
    want[np.lexsort((i, -key.astype(np.int64)))[:budget]] = True
    assert stays.sum() == budget and np.array_equal(stays, want)
    assert stays[safe].all()


# ------------------------------------------------------- vox_kv_observe, windows: score tiles of the groups of warps

def score_tiles(q8, weights, rows, key_tiles, groups=4):
    """The score tiles that each group of warps of kv_observe_window.cu takes, in order, and how many there are."""
    n_b, blocks = -(-rows // 64), -(-rows // 128)
    n_m = 4 if q8 and not weights and blocks == 3 else blocks
    per_tile = n_b if weights else 2 * n_m
    taken = [[] for _ in range(groups)]
    for t in range(key_tiles):
        u = t * per_tile
        for g in range(groups):
            if weights:
                taken[g] += [u + i for i in range((g - u) % groups, n_b, groups)]
            else:
                taken[g] += [u + 2 * mt + (g & 1) for mt in range(g >> 1, n_m, 2)]
    return taken, per_tile * key_tiles


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("weights", [False, True])
def test_a_wait_for_a_score_tile_is_never_two_uses_of_its_buffer_away(q8, weights):
    """A barrier tells even uses of a buffer from odd ones.  When a group waits for tile u, the use of its buffer before that, tile
    u - buffers, must be over: that is so if the group has taken a tile from there on."""
    buffers = 4 if q8 else 8
    for rows in range(2, 513):
        taken, total = score_tiles(q8, weights, rows, 11)
        assert sorted(u for g in taken for u in g) == list(range(total))
        for g in taken:
            for last, u in zip([-1] + g, g):
                assert u - buffers <= last, (rows, last, u)
