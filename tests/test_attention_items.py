"""The work items of attention's split tiles (on the CPU: the plan takes
lengths and a CU count): every range of every tile is one item of the launch,
with a place of its own for its partial sums, and the join finds them all."""
import ctypes
import random

import numpy as np
import pytest

import bonsai_b1

ROWS = 128  # of a tile
STAGE = {64: 64, 128: 32, 256: 32}  # keys, by head dim


@pytest.fixture(scope="module")
def items():
    """items(q lengths, key lengths, ..., join): the items of a split call and
    the rows of partial sums; None where nothing is split."""
    fn = bonsai_b1.load().b1_attention_items
    fn.restype = ctypes.c_int64

    def of(ql, kl, most, heads, kv_heads, d, causal, window, cus, join):
        q, k = np.array(ql, np.int32), np.array(kl, np.int32)
        out, rows, room = np.zeros((1 << 15, 9), np.int32), ctypes.c_int64(0), 1 << 15
        n = fn(q.ctypes.data_as(ctypes.c_void_p), k.ctypes.data_as(ctypes.c_void_p), len(ql), most, heads, kv_heads,
               d, int(causal), window, cus, int(join), out.ctypes.data_as(ctypes.c_void_p), ctypes.c_int64(room),
               ctypes.byref(rows))
        assert n <= room
        return (out[:n].tolist(), rows.value) if n else None

    return of


def stages(nq, nk, group, tile, causal, window, size):
    """The stages of `size` keys that hold what a tile's rows see, from the
    definition: token i sees keys 0 .. nk - nq + i, the last `window` of them."""
    first, last = tile * ROWS // group, (min(tile * ROWS + ROWS, nq * group) - 1) // group
    lo, hi = 0, nk - 1
    if causal:
        hi = nk - nq + last
        lo = max(0, nk - nq + first - window + 1) if window else 0
    hi = max(hi + 1, lo)
    return lo // size, -(-hi // size), hi - lo


def check(items, ql, kl, heads, kv_heads, d, causal, window, cus=256, most=None):
    """True if the call is split."""
    most = sum(kl) if most is None else most
    launched = items(ql, kl, most, heads, kv_heads, d, causal, window, cus, False)
    if launched is None:
        return False
    what = (ql, kl, heads, kv_heads, d, causal, window, cus)
    launched, rows = launched
    joined, _ = items(ql, kl, most, heads, kv_heads, d, causal, window, cus, True)
    group, size = heads // kv_heads, STAGE[d]
    tiles = {}
    for b, kvh, tile, r, ranges, t0, t1, part, apart in launched:
        if b < 0 or r >= ranges:
            continue  # such a work-group returns at once
        assert (b, kvh, tile, r) not in tiles, what
        tiles[b, kvh, tile, r] = (ranges, t0, t1, part + r * apart)
    places = [v[3] for v in tiles.values() if v[0] > 1]
    assert len(set(places)) == len(places) and all(0 <= p and (p + 1) * ROWS <= rows for p in places), what
    found = {}
    for b, kvh, tile, _, ranges, _, _, part, apart in joined:
        if b >= 0:
            assert (b, kvh, tile) not in found, what
            found[b, kvh, tile] = (ranges, part, apart)
    for b, (nq, nk) in enumerate(zip(ql, kl)):
        for tile in range(-(-nq * group // ROWS)):
            first, last, keys = stages(nq, nk, group, tile, causal, window, size)
            for kvh in range(kv_heads):
                if len(ql) == 1 and (b, kvh, tile) not in found:
                    continue  # one of the whole tiles in front of the split ones
                ranges, part, apart = found[b, kvh, tile]
                at = first
                for r in range(ranges):
                    n, t0, t1, place = tiles[b, kvh, tile, r]
                    assert n == ranges and t0 == at and (t1 > t0 or keys == 0), what
                    assert ranges == 1 or place == part + r * apart, what
                    at = t1
                assert at == max(first, last), what
    return True


@pytest.mark.parametrize("ql,kl,heads,kv_heads,d,window", [
    ([129, 129], [4096, 4096], 8, 8, 128, 2048), ([4097, 4097], [4097, 4097], 1, 1, 128, 1024),
    ([19713], [30000], 1, 1, 128, 4096), ([130, 70, 257], [5000, 3000, 9000], 4, 2, 64, 1536),
    ([65, 200], [8000, 8100], 8, 4, 256, 1023), ([129, 129], [4096, 4096], 8, 8, 128, 0)])
def test_every_range_is_one_item(items, ql, kl, heads, kv_heads, d, window):
    """Among them windows whose last tile has fewer rows, and so fewer keys,
    than the others; and more keys than an fp32 count of them holds."""
    assert check(items, ql, kl, heads, kv_heads, d, True, window)


@pytest.mark.parametrize("ql,kl", [([200], [(1 << 30) - 1]), ([200, 300], [(1 << 28) + 33, (1 << 29) + 1])])
@pytest.mark.parametrize("window", [0, (1 << 27) + 1])
def test_more_keys_than_fp32_counts(items, ql, kl, window):
    assert check(items, ql, kl, 2, 1, 64, True, window)


def test_random_calls(items):
    rng = random.Random(11)

    def spread(lo, hi):
        return int(lo * (hi / lo) ** rng.random())

    split = windowed = 0
    for _ in range(3000):
        n = rng.choice([1, 1, 2, 2, 3, 5, 9, 30, 70])
        kv_heads, group, d = rng.choice([1, 1, 2, 3, 8]), rng.choice([1, 1, 2, 3, 4, 8, 130]), rng.choice([64, 128, 256])
        ql = [0 if rng.random() < 0.1 else spread(1, 6000 // (n * group) + 200) for _ in range(n)]
        kl = [rng.choice([q + spread(1, 30000) - 1, spread(1, 9000), q]) for q in ql]
        causal = rng.random() < 0.8
        window = spread(1, 8000) if causal and rng.random() < 0.7 else 0
        most = sum(kl) + rng.choice([0, 1, 5000])
        if check(items, ql, kl, kv_heads * group, kv_heads, d, causal, window, rng.choice([256, 256, 64, 304]), most):
            split += 1
            windowed += window > 0
    assert split > 500 and windowed > 200  # the rest have too little work to split
