"""Trees of drafted tokens of which one has a key or a value that is no number (thip_lm_tree_attention): rows on whose path it is not have what they had, and those on
whose path it is have what the definition says, element by element."""
import numpy as np
import pytest

import torq_compiler_amd as thip
from oracle import attention as ref
from test_cache_attention import Batch, Built
from test_tree import plant

STREAM, TILES = "tree_attention_stream<", "tree_attention_tiles<"
CASES = [
    (STREAM, False, dict(sequences=[(16, 80), (5, 200)], D=64, H=4, KVH=1)),
    (STREAM, True, dict(sequences=[(16, 80), (5, 200)], D=96, H=4, KVH=2)),
    (STREAM, False, dict(sequences=[(33, 90)], D=256, H=4, KVH=1)),
    (STREAM, True, dict(sequences=[(33, 90)], D=256, H=4, KVH=1)),
    (STREAM, False, dict(sequences=[(20, 1100)], D=128, H=2, KVH=1)),  # cut into parts
    (TILES, False, dict(sequences=[(90, 120), (45, 60)], D=64, H=64, KVH=8)),
    (TILES, True, dict(sequences=[(90, 120), (45, 60)], D=64, H=64, KVH=8)),
    (TILES, False, dict(sequences=[(70, 90)], D=112, H=120, KVH=8)),
    (TILES, True, dict(sequences=[(70, 90)], D=128, H=120, KVH=8)),
    (TILES, False, dict(sequences=[(60, 80)], D=256, H=72, KVH=8)),
    (TILES, True, dict(sequences=[(130, 150)], D=256, H=128, KVH=8)),
    (TILES, False, dict(sequences=[(66, 1100)], D=64, H=128, KVH=2)),  # cut into parts
]
BAD = dict(nan=(0x7FC0, np.nan), inf=(0x7F80, np.inf), minus=(0xFF80, -np.inf))


def seen(b, parents, row):
    """Positions that a row of the first sequence sees."""
    base = int(b.lengths[0]) - int(b.starts[1])
    path = [row]
    while 0 <= parents[path[-1]] < path[-1]:
        path.append(int(parents[path[-1]]))
    return list(range(base)) + sorted(base + r for r in path)


def expected(b, parents, place, at, clean):
    """(result, bound).  clean: those of the batch without the bad numbers, which rows have that do not see them.  Where the position's score is minus infinity its
    weight is 0, so the bound is that of the row without it."""
    result, bound = clean[0].copy(), clean[1].copy()
    cache, q = b.cache(), ref.from_bf16(b.query)
    key = np.repeat(cache.row(0, 0, place), b.H // b.KVH, axis=0)
    for row in np.flatnonzero(reaches(b, parents, at)):
        with_it = seen(b, parents, row)
        keys, values = (np.stack([cache.row(which, 0, j) for j in with_it], axis=1) for which in (0, 1))
        result[row], bound[row] = ref._weighed(q[row], keys, values, b.scale, False, False)
        gone = (q[row] * key).sum(axis=-1) == -np.inf
        if gone.any():
            others = [i for i, j in enumerate(with_it) if j != place]
            without = ref._weighed(q[row], keys[:, others], values[:, others], b.scale, False, False)
            result[row][gone], bound[row][gone] = without[0][gone], without[1][gone]
    return result, bound


def reaches(b, parents, at):
    """Rows of the first sequence on whose path its row `at` is."""
    hit = np.zeros(b.T, dtype=bool)
    for i in range(int(b.starts[1])):
        hit[i] = i == at or (0 <= parents[i] < i and hit[parents[i]])
    return hit


def agree(got, result, bound):
    """NaN and infinities in the same places, and every number within its bound, which is one."""
    assert np.array_equal(np.isnan(got), np.isnan(result))
    inf = np.isinf(result)
    assert np.array_equal(got[inf], result[inf]) and np.isfinite(got[np.isfinite(result)]).all()
    number = np.isfinite(result)
    assert np.isfinite(bound[number]).all()
    assert (np.abs(got - result)[number] <= bound[number]).all(), np.max((np.abs(got - result) / bound)[number])


def spoil(b, place, what, bad, element):
    """The batch with a number that is none at a position of its first sequence."""
    which = 0 if what == "key" else 1
    b.caches, b.scales = [x.copy() for x in b.caches], [None if x is None else x.copy() for x in b.scales]
    page, slot = b.pages[0, place // b.page], place % b.page
    if b.quantised:
        b.scales[which][page, :, slot] = BAD[bad][1]
    else:
        b.caches[which][page, :, slot, slice(None) if element is None else element] = BAD[bad][0]


@pytest.mark.gpu
@pytest.mark.parametrize("kernel,quantised,case", CASES, ids=lambda v: "-".join(str(x) for x in list(v.values())[1:]) if isinstance(v, dict) else str(v).strip("<"))
def test_gpu_numbers_that_are_none(device, kernel, quantised, case):
    """A NaN or an infinity in one element of a row, or in all of them; of int8 in its scale (of a key a NaN: times an infinite scale, elements of both signs make a NaN
    of a score that has a sign once they are summed, so the order would decide)."""
    b = Batch(quantised=quantised, page=8, **case)
    parents, at = plant(b, "pairs"), 2
    place = int(b.lengths[0]) - int(b.starts[1]) + at
    clean = ref.tree_attention(b.query, b.starts, b.lengths, parents, b.cache(), b.scale)
    hit, caches, scales = reaches(b, parents, at), b.caches, b.scales
    assert hit.any() and not hit.all()
    built = Built()
    q = built.bind("query", b.query)
    cache, more = built.cache(b)
    starts, lengths = built.rows(b)
    built.program.tree_attention(q, *cache, starts, lengths, built.bind("parents", parents), init=built.bind("out", b.query), scale=b.scale, **more)
    exe = thip.Executable(device, built.program.serialize())
    names = exe.op_kernels()
    exe.close()
    assert names[0].startswith(kernel), names
    for what, bad, element in [(w, x, e) for w in ("key", "value") for x in BAD for e in ((5, None) if not quantised else (None,)) if not (quantised and w == "key" and x != "nan")]:
        b.caches, b.scales = caches, scales
        spoil(b, place, what, bad, element)
        now = dict(key_cache=b.caches[0], value_cache=b.caches[1], key_scales=b.scales[0], value_scales=b.scales[1])
        built.arrays = [(name, now.get(name, x)) for name, x in built.arrays]
        with np.errstate(all="ignore"):
            result, bound = expected(b, parents, place, at, clean)
            assert not np.isfinite(result[hit]).all()
            try:
                agree(ref.from_bf16(built.run(device)["out"]), result, bound)
            except AssertionError as e:
                raise AssertionError("%s %s element %s: %s" % (what, bad, element, e))


def test_expectation_of_a_score_of_minus_infinity():
    """It is the definition's: what the reference gives where such a key is seen is what it gives without the position."""
    b = Batch(**CASES[0][2])
    parents, at = plant(b, "pairs"), 2
    place = int(b.lengths[0]) - int(b.starts[1]) + at
    args = b.query, b.starts, b.lengths, parents
    clean = ref.tree_attention(*args, b.cache(), b.scale)
    spoil(b, place, "key", "inf", 5)
    hit = reaches(b, parents, at)
    with np.errstate(all="ignore"):
        defined, its_bound = ref.tree_attention(*args, b.cache(), b.scale)
        result, bound = expected(b, parents, place, at, clean)
    both = hit[:, None, None] & np.isfinite(result)
    assert both.any() and np.allclose(defined[both], result[both], rtol=1e-12, atol=1e-15) and np.isfinite(bound[both]).all()
    assert np.array_equal(np.isnan(defined), np.isnan(result)) and np.array_equal(defined[~hit], result[~hit]) and np.array_equal(its_bound[~hit], bound[~hit])
