"""Trees of drafted tokens over a paged cache (thip_lm_tree_attention, thip_lm_cache_keep): records and refusals on the CPU, results on the GPU against the
64-bit definition (oracle/attention.py, which derives the bound that is held), and a decoder's layers that check a tree and keep its accepted path."""
import ctypes
import os
import shutil
import struct
import subprocess

import numpy as np
import pytest

import desc_interp
import torq_compiler_amd as thip
from helpers import host_check
from oracle import attention as ref
from oracle import layer
from test_cache_attention import Batch, Built, _operands, _serialize_error, check_attention
from torq_compiler_amd import runtime as rt
from torq_compiler_amd import workloads as w

U16, I32 = np.uint16, np.int32
KIND_TREE, KIND_KEEP = 20, 21


def _id(case):
    return "-".join(str(v) if not isinstance(v, list) else "%dseq" % len(v) for v in case.values()).replace(" ", "")


def plant(b, kind="bushy"):
    """parents of a batch's rows."""
    out = np.full(b.T, 7, I32)  # what rows of no sequence have is nobody's
    for s, (n, _) in enumerate(b.sequences):
        for i in range(n):
            out[b.starts[s] + i] = dict(chain=i - 1, star=-1 if i == 0 else 0, roots=-1, pairs=(i - 1) // 2,
                                        bushy=int(b.rng.integers(-1, i)) if i else -1, comb=i - 1 if i % 3 else i - 3)[kind]
    return out


def attend_tree(b, parents, window=0, sinks=0, constant=False):
    built = Built()
    out = b.normal(b.T, b.H, b.D)
    q = built.bind("query", b.query)
    cache, scales = built.cache(b)
    starts, lengths = built.rows(b)
    see = dict(scale=b.scale, window=window, sinks=sinks)
    built.program.tree_attention(q, *cache, starts, lengths, parents if constant else built.bind("parents", parents), init=built.bind("out", out), **see, **scales)
    return built, out, ref.tree_attention(b.query, b.starts, b.lengths, parents, b.cache(), **see)


TREES = [
    dict(sequences=[(1, 1)], D=16, H=1, page=1),
    dict(sequences=[(1, 7), (5, 64), (2, 65), (3, 3), (0, 9), (1, 200)], D=64, H=4, page=16, tail=2),
    dict(sequences=[(16, 129), (7, 31)], D=128, H=8, KVH=2, page=7),
    dict(sequences=[(16, 700)], D=256, H=4, KVH=1, page=16),
    dict(sequences=[(9, 33)] * 9, D=80, H=16, KVH=1, page=24),
    dict(sequences=[(40, 50), (4, 4), (33, 100)], D=96, H=5, KVH=5, page=32),
    dict(sequences=[(5, 3), (9, 9), (12, 300)], D=128, H=32, KVH=2, page=64, spare_entries=3),  # the first rows of one have places below 0
    dict(sequences=[(64, 200), (1, 90), (40, 41)], D=64, H=4, KVH=2, page=24, tail=4),
    dict(sequences=[(100, 333)], D=256, H=2, KVH=1, page=128),
    dict(sequences=[(3, 40)] * 130, D=32, H=2, KVH=1, page=8),
    dict(sequences=[(200, 900), (1, 2000), (2, 700), (130, 131)], D=64, H=8, KVH=2, page=24, tail=3),
]
SEEN = [dict(), dict(window=1), dict(window=3, sinks=1), dict(window=65, sinks=4), dict(window=40, sinks=100)]


@pytest.mark.gpu
@pytest.mark.parametrize("quantised", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("see", SEEN, ids=_id)
@pytest.mark.parametrize("case", TREES, ids=_id)
def test_gpu_trees(device, case, see, quantised):
    """Every shape of batch under every window, bushy trees; twice, as the second dispatch finds what the first left."""
    b = Batch(quantised=quantised, **case)
    built, before, want = attend_tree(b, plant(b), **see)
    first = built.run(device)["out"]
    check_attention(b, first, before, want)
    assert np.array_equal(built.run(device, dispatches=2)["out"], first)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["chain", "star", "roots", "pairs", "comb"])
@pytest.mark.parametrize("case", [TREES[2], TREES[7], dict(sequences=[(300, 420), (31, 90)], D=128, H=8, KVH=2, page=16)], ids=_id)
def test_gpu_shapes_of_trees(device, case, kind):
    """Chains, stars, rows that all follow the text, complete trees, combs; a chain is what attention over the cache gives its rows."""
    for see in (dict(), dict(window=20, sinks=2)):
        b = Batch(quantised=True, **case)
        parents = plant(b, kind)
        built, before, want = attend_tree(b, parents, **see)
        got = built.run(device)["out"]
        check_attention(b, got, before, want, kind)
        if kind == "chain":
            want = ref.attention(b.query, b.starts, b.scale, cache=b.cache(), lengths=b.lengths, **see)
            check_attention(b, got, before, want, "as a chunk")


@pytest.mark.gpu
@pytest.mark.parametrize("D,H,KVH", [(64, 2, 2), (128, 4, 1), (256, 4, 1)])
@pytest.mark.parametrize("n", [511, 512, 513, 700])
def test_gpu_largest_trees(device, n, D, H, KVH):
    """Up to 512 rows; those behind see nothing, and nobody sees them, also where parents say so."""
    b = Batch([(n, n + 90), (3, 50)], D=D, H=H, KVH=KVH, page=16, quantised=D == 128)
    for kind, see in (("bushy", dict()), ("chain", dict(window=30, sinks=95))):
        built, before, want = attend_tree(b, plant(b, kind), **see)
        check_attention(b, built.run(device)["out"], before, want, kind)


@pytest.mark.gpu
@pytest.mark.parametrize("quantised", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("D,H,KVH", [(64, 16, 4), (128, 16, 2)])
@pytest.mark.parametrize("kind", ["chain", "comb", "bushy"])
def test_gpu_windows_over_trees_of_all_sizes(device, kind, D, H, KVH, quantised):
    """Sequences whose windows are cut into different numbers of parts, and paths that leave a window inside the tree, at and next to a word's end."""
    b = Batch([(300, 1300), (3, 1300), (40, 700), (129, 131), (96, 97), (0, 50), (17, 1100)], D=D, H=H, KVH=KVH, page=24, quantised=quantised, tail=3)
    parents = plant(b, kind)
    for see in (dict(window=600, sinks=40), dict(window=33, sinks=1050), dict(window=32, sinks=2 ** 31 - 1)):
        built, before, want = attend_tree(b, parents, **see)
        check_attention(b, built.run(device)["out"], before, want, str(see))


@pytest.mark.gpu
@pytest.mark.parametrize("quantised", [False, True], ids=["bf16", "int8"])
def test_gpu_parents_of_every_kind(device, quantised):
    """Parents that are the row itself, come behind it, or are no rows at all count as none; as constants, and by host pointers too."""
    b = Batch([(20, 60), (40, 300)], D=64, H=4, KVH=2, quantised=quantised)
    parents = plant(b)
    parents[[1, 5, 7, 9, 30, 41, 50, 59]] = [1, 6, 2 ** 31 - 1, -2 ** 31, 39, -7, 40, 39]
    for constant in (False, True):
        built, before, want = attend_tree(b, parents, constant=constant)
        check_attention(b, built.run(device)["out"], before, want)
        check_attention(b, built.run(device, "host")["out"], before, want)


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [0x7FC0, 0x7F80, 0xFF80], ids=["nan", "inf", "-inf"])
@pytest.mark.parametrize("case", [dict(sequences=[(16, 80), (5, 300)], D=64, H=4, KVH=1), dict(sequences=[(90, 300), (2, 40)], D=128, H=4, KVH=2),
                                  dict(sequences=[(33, 90)], D=256, H=4, KVH=1)], ids=_id)
def test_gpu_numbers_that_are_none_on_other_branches(device, case, bad):
    """Keys and values of one drafted row are no numbers: rows on whose path it is not have what they had."""
    for what in (0, 1):
        b = Batch(**case)
        parents = plant(b, "pairs")
        at = 2  # of the first sequence
        place = int(b.lengths[0]) - int(b.starts[1]) + at
        b.caches[what][b.pages[0, place // b.page], :, place % b.page] = bad
        built, before, want = attend_tree(b, parents)
        got = built.run(device)["out"]
        hit = np.zeros(b.T, dtype=bool)
        for i in range(int(b.starts[1])):
            hit[i] = i == at or (parents[i] >= 0 and hit[parents[i]])
        assert hit.any() and not hit.all()
        check_attention(b, np.where(hit[:, None, None], before, got), np.where(hit[:, None, None], before, before), (np.where(hit[:, None, None], ref.from_bf16(before), want[0]), want[1]))
        # and those on whose path it is do not keep it from themselves: they see what the definition does
        bad_there = ~np.isfinite(want[0]) & hit[:, None, None]
        if bad == 0x7FC0:
            assert np.isnan(ref.from_bf16(got)[bad_there]).all()


@pytest.mark.gpu
def test_gpu_pages_that_are_none_in_a_tree(device):
    """A drafted row whose page is none is seen by nobody, its own row keeps the rest of its path."""
    for quantised in (False, True):
        for D, H in ((64, 4), (128, 16)):
            b = Batch([(30, 100), (50, 400)], D=D, H=H, KVH=2, page=8, quantised=quantised)
            b.pages[0, 80 // 8] = -1
            b.pages[1, 360 // 8] = 2 ** 30
            b.pages[1, 3] = -5
            built, before, want = attend_tree(b, plant(b))
            check_attention(b, built.run(device)["out"], before, want)


@pytest.mark.gpu
@pytest.mark.parametrize("starts", [[0, 9, 4, 12], [5, 5, 5, 5], [-3, 2, 40, 7], [2 ** 31 - 1, 0, 3, -2 ** 31]])
def test_gpu_starts_that_do_not_ascend(device, starts):
    """Rows stay inside their tensors whatever row_starts holds, and an ordinary dispatch behind that is right (counters and workspace are as they were)."""
    b = Batch([(4, 2000), (4, 3000), (4, 500)], D=128, H=8, KVH=2, page=16)
    built, before, want = attend_tree(b, plant(b))
    rows = np.array(starts, I32)
    exe = thip.Executable(device, built.program.serialize())
    try:
        ptrs = [device.upload(a) for _, a in built.arrays]
        sizes = [a.nbytes for _, a in built.arrays]
        at = [n for n, _ in built.arrays].index("row_starts")
        odd = device.upload(rows)
        exe.run_device([odd if i == at else p for i, p in enumerate(ptrs)], sizes)
        exe.run_device(ptrs, sizes)
        where = [n for n, _ in built.arrays].index("out")
        got = device.download(ptrs[where], before.shape, before.dtype)
        for p in ptrs + [odd]:
            device.free(p)
    finally:
        exe.close()
    check_attention(b, got, before, want)  # no row is of no sequence


@pytest.mark.gpu
def test_gpu_many_sequences_of_trees(device):
    """More sequences than a wave looks through at once, of very different lengths, their runs cut into parts."""
    b = Batch([(3, 40 + 7 * i % 300) for i in range(150)] + [(60, 5000)], D=64, H=4, KVH=1, page=16, quantised=True)
    for see in (dict(), dict(window=100, sinks=2)):
        built, before, want = attend_tree(b, plant(b), **see)
        check_attention(b, built.run(device)["out"], before, want)


@pytest.mark.gpu
@pytest.mark.parametrize("quantised", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("rows,D", [(1, 64), (3, 128), (60, 64), (60, 128), (60, 256), (600, 128)])
def test_gpu_last_positions_of_32_bits(device, rows, D, quantised):
    """Tables of 2^31 - 8 positions (all of their entries the same page) with trees that end there, or behind; the reference has the same rows a whole number of
    pages further down."""
    page, P = 8 * 127 * 113, 3 * 5 * 29 * 43
    assert page * P == 2 ** 31 - 8
    b = Batch([(rows, 16)], D=D, H=4, KVH=1, page=16, quantised=quantised, garbage=False)
    shape = (1, 1, page, D)
    if quantised:
        b.caches = [b.rng.integers(-127, 128, size=shape, dtype=np.int8) for _ in range(2)]
        b.scales = [(b.rng.uniform(0.5, 1.5, size=shape[:3]) / 73).astype(np.float32) for _ in range(2)]
        b.scales[1][0, 0, page - 25] = np.nan  # a row that sees it is done again
    else:
        b.caches = [b.normal(*shape) for _ in range(2)]
        b.caches[1][0, 0, page - 25] = 0x7FC0
    parents = plant(b)
    for length in (2 ** 31 - 8, 2 ** 31 - 1, 2 ** 31 - 37):
        see = dict(window=16, sinks=3 if length % 2 else 0)
        b.page, b.pages, b.lengths = page, np.zeros((1, 1), dtype=I32), np.array([length - (P - 1) * page], dtype=I32)
        near = ref.tree_attention(b.query, b.starts, b.lengths, parents, b.cache(), b.scale, **see)
        b.pages, b.lengths = np.zeros((1, P), dtype=I32), np.array([length], dtype=I32)
        built, out = Built(), b.normal(b.T, b.H, b.D)
        q = built.bind("query", b.query)
        cache, scales = built.cache(b)
        starts, lengths = built.rows(b)
        built.program.tree_attention(q, *cache, starts, lengths, built.bind("parents", parents), init=built.bind("out", out), scale=b.scale, **see, **scales)
        check_attention(b, built.run(device)["out"], out, near, str(length))


@pytest.mark.gpu
@pytest.mark.parametrize("quantised", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("case", [TREES[2], TREES[3], TREES[10], dict(sequences=[(120, 3000)] * 3, D=128, H=32, KVH=4, page=16)], ids=_id)
def test_gpu_results_over_the_queries(device, case, quantised):
    """init is the query's own bytes, also where runs are cut into parts."""
    b = Batch(quantised=quantised, **case)
    parents = plant(b)
    built = Built()
    q = built.bind("query", b.query)
    cache, scales = built.cache(b)
    starts, lengths = built.rows(b)
    built.program.tree_attention(q, *cache, starts, lengths, built.bind("parents", parents), init=q, scale=b.scale, **scales)
    check_attention(b, built.run(device)["query"], b.query, ref.tree_attention(b.query, b.starts, b.lengths, parents, b.cache(), b.scale))


@pytest.mark.gpu
def test_gpu_two_programs_at_once(device):
    """Two executables dispatched from a thread each, their runs cut into parts: each has its own workspace, and the results are those of one alone."""
    import threading
    batches = [Batch([(16, 3000 + 100 * i), (40, 900)], D=128, H=8, KVH=2, page=16, quantised=i == 1, seed=i) for i in range(2)]
    made = [attend_tree(b, plant(b)) for b in batches]
    alone = [m[0].run(device)["out"] for m in made]
    together = [None, None]

    def work(i):
        together[i] = made[i][0].run(device, dispatches=40)["out"]

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for i in range(2):
        check_attention(batches[i], alone[i], made[i][1], made[i][2])
        assert np.array_equal(alone[i], together[i])


def test_the_bound_tells_trees_apart():
    """A row that took a neighbour's path would be seen."""
    b = Batch([(12, 40)], D=64, H=2, KVH=1)
    parents = plant(b, "pairs")
    want, bound = ref.tree_attention(b.query, b.starts, b.lengths, parents, b.cache(), b.scale)
    other, _ = ref.tree_attention(b.query, b.starts, b.lengths, np.roll(parents, 1), b.cache(), b.scale)
    assert (np.abs(want - other) > bound).any(axis=(1, 2))[2:].mean() > 0.6
    # a chain is attention of a chunk
    chain = ref.tree_attention(b.query, b.starts, b.lengths, plant(b, "chain"), b.cache(), b.scale, window=9, sinks=2)[0]
    assert np.allclose(chain, ref.attention(b.query, b.starts, b.scale, 9, 2, cache=b.cache(), lengths=b.lengths)[0], rtol=1e-12, atol=1e-14)


@pytest.mark.parametrize("seed", [1, 2])
def test_shares_of_a_launch(tmp_path, seed):
    """The parts of a run that is cut have all of its blocks, whatever the trees, their windows and the text before them are (tests/host/tree_plan.cpp)."""
    run = subprocess.run([host_check("tree_plan", tmp_path), str(seed)], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=300)
    assert run.returncode == 0 and int(run.stdout) > 1000, run.stdout[-2000:]


# ---- what is kept -------------------------------------------------------------------------------------------------------

KEPT = [
    dict(sequences=[(1, 1)], D=16, KVH=1, page=1),
    dict(sequences=[(5, 9), (0, 5), (1, 0), (16, 40)], D=64, KVH=2, page=16, tail=2),
    dict(sequences=[(40, 100), (5, 5), (0, 3), (33, 100)], D=80, KVH=3, page=24, spare_entries=2),
    dict(sequences=[(7, 3), (9, 4), (100, 1000)], D=96, KVH=1, page=7),  # rows at places below 0
    dict(sequences=[(300, 700), (64, 64)], D=128, KVH=8, page=64),
    dict(sequences=[(16, 300)] * 40 + [(2, 9)], D=256, KVH=1, page=16),
    dict(sequences=[(5, 9)] * 1100, D=16, KVH=1, page=4),
]


def _accept(b, K, kind, rng):
    out = np.full((len(b.sequences), K), -1, I32)
    for s, (n, _) in enumerate(b.sequences):
        take = min(n, K)
        if kind == "all":
            path = np.arange(take)
        elif kind == "last":
            path = np.arange(n - take, n)
        else:
            path = np.sort(rng.choice(n, int(rng.integers(0, take + 1)), replace=False)) if n else []
        out[s, :len(path)] = path
        if kind == "odd" and take:  # what follows the end of a list is not looked at
            end = int(rng.integers(0, take))
            out[s, end] = rng.choice([-1, n, 2 ** 31 - 1, -2 ** 31] + ([out[s, end - 1], 0] if end else []))
            out[s, end + 1:] = rng.integers(0, max(n, 1), K - end - 1)
    return out


def keep(b, accepted, constant=False):
    built = Built()
    cache, scales = built.cache(b)
    starts, lengths = built.rows(b)
    built.program.cache_keep(*cache, starts, lengths, accepted if constant else built.bind("accepted", accepted), **scales)
    return built


def check_kept(b, got, accepted):
    for name, x in zip(("key_cache", "value_cache", "key_scales", "value_scales"), ref.cache_keep(b.cache(), accepted, b.starts, b.lengths)):
        if x is not None:
            bits = np.uint32 if x.dtype == np.float32 else x.dtype
            assert np.array_equal(got[name].view(bits), x.view(bits)), name


@pytest.mark.gpu
@pytest.mark.parametrize("quantised", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("kind", ["some", "all", "last", "odd"])
@pytest.mark.parametrize("case", KEPT, ids=_id)
def test_gpu_keep(device, case, kind, quantised):
    """Equals the definition bit for bit, everything else in the cache stays as it was; short lists and ones of more entries than a wave has lanes."""
    for K in (1, 6, 130):
        b = Batch(quantised=quantised, seed=K, **case)
        accepted = _accept(b, K, kind, b.rng)
        check_kept(b, keep(b, accepted).run(device), accepted)
    check_kept(b, keep(b, accepted, constant=True).run(device, "host"), accepted)


@pytest.mark.gpu
@pytest.mark.parametrize("quantised", [False, True], ids=["bf16", "int8"])
def test_gpu_keep_without_places(device, quantised):
    """Entries of which one place has no page move nothing; the others of the list do."""
    b = Batch([(40, 100), (30, 64)], D=64, KVH=2, page=8, quantised=quantised)
    b.pages[0, 9] = -1
    b.pages[1, 5] = 10 ** 6
    accepted = np.array([[1, 5, 9, 14, 15, 20, 30, 39, -1], [0, 2, 3, 4, 8, 9, 20, 28, 29]], I32)
    check_kept(b, keep(b, accepted).run(device), accepted)


def test_keep_reference():
    """The rows of the path are behind one another, in their order."""
    b = Batch([(9, 30)], D=16, KVH=1, page=4)
    accepted = np.array([[0, 3, 4, 8, -1]], I32)
    key = ref.cache_keep(b.cache(), accepted, b.starts, b.lengths)[0]
    after = ref.Cache(key, b.caches[1], b.pages)
    for k, r in enumerate([0, 3, 4, 8]):
        assert np.array_equal(after.row(0, 0, 21 + k), b.cache().row(0, 0, 21 + r))


# ---- records and refusals -----------------------------------------------------------------------------------------------

def _tree(p, v, scales=False, parents=None, **see):
    see.setdefault("scale", 0.125)
    s = dict(key_scales=v["key_scales"], value_scales=v["value_scales"]) if scales else {}
    p.tree_attention(v["query"], v["key_cache"], v["value_cache"], v["pages"], v["row_starts"], v["lengths"],
                     p.binding(20, (v["query"].shape[0],), I32) if parents is None else parents, init=v["out"], **see, **s)


def _keep(p, v, scales=False, accepted=None):
    s = dict(key_scales=v["key_scales"], value_scales=v["value_scales"]) if scales else {}
    p.cache_keep(v["key_cache"], v["value_cache"], v["pages"], v["row_starts"], v["lengths"], p.binding(20, (2, 5), I32) if accepted is None else accepted, **s)


def test_records_and_bindings():
    b = Batch([(2, 5), (3, 20)], quantised=True)
    built = Built()
    cache, scales = built.cache(b)
    starts, lengths = built.rows(b)
    p = built.program
    y = p.tree_attention(built.bind("query", b.query), *cache, starts, lengths, built.bind("parents", plant(b)), scale=0.125, **scales)
    assert y.shape == b.query.shape
    p.cache_keep(*cache, starts, lengths, built.bind("accepted", np.zeros((2, 3), I32)), **scales)
    blob = p.serialize()
    assert [int(o["kind"]) for o in desc_interp.Descriptor(blob).ops] == [KIND_TREE, KIND_KEEP]
    _, bindings, _ = rt.describe_blob(blob)
    modes = {name: (bool(x["is_read_only"]), bool(x["is_write_only"])) for (name, _), x in zip(built.arrays, bindings)}
    assert modes == {name: (name not in ("key_cache", "value_cache", "key_scales", "value_scales"), False) for name in modes}


@pytest.mark.parametrize("shapes,code,text", [
    (dict(D=72), rt.UNIMPLEMENTED, "multiples of 16"),
    (dict(H=3), rt.INVALID_ARGUMENT, "query heads"),
    (dict(dtype=np.int8), rt.INVALID_ARGUMENT, "key_scales"),
    (dict(pages=((3, 4), I32)), rt.INVALID_ARGUMENT, "sequences"),
    (dict(out=((5, 4, 32), U16)), rt.INVALID_ARGUMENT, "expected [5, 4, 64]"),
], ids=["D", "H", "int8", "pages", "out"])
def test_refused_shapes(shapes, code, text):
    got, message = _serialize_error(lambda p: _tree(p, _operands(p, **shapes)))
    assert got == code and text in message, (got, message)


def test_refused_operands():
    def parents(shape, dtype=I32):
        def call(p):
            v = _operands(p)
            _tree(p, v, parents=p.binding(20, shape, dtype))
        return call

    def accepted(shape, dtype=I32):
        def call(p):
            v = _operands(p)
            _keep(p, v, accepted=p.binding(20, shape, dtype))
        return call

    def computed(p):
        v = _operands(p)
        _tree(p, v, parents=p.tensor((5,), I32))

    def written_over(p):
        v = _operands(p)
        _tree(p, v, parents=p.view(p.binding(1, (5 * 4 * 32,), I32), (5,)))

    def accepted_in_the_scales(p):
        v = _operands(p, dtype=np.int8)
        _keep(p, v, scales=True, accepted=p.view(p.binding(9, (9 * 2 * 16,), I32), (2, 5)))

    def over_rows(p):
        v = _operands(p)
        op = rt.LmTreeAttention(v["out"].index, v["query"].index, v["key"].index, v["value"].index, -1, -1, -1, v["row_starts"].index, -1,
                                p.binding(20, (5,), I32).index, 0.125, 0, 0)
        rt.check(rt.lib().thip_lm_tree_attention(p._h, ctypes.byref(op)))

    def cache_of_a_program(p):
        v = _operands(p)
        v["key_cache"] = p.tensor((9, 2, 16, 64), U16)
        _keep(p, v)

    def scales_of_bf16(p):
        _keep(p, _operands(p), scales=True)

    for make in (parents((4,)), parents((5, 1)), parents((5,), np.int16), accepted((3, 5)), accepted((10,)), accepted((2, 5), np.float32), computed, written_over,
                 accepted_in_the_scales, over_rows, cache_of_a_program, scales_of_bf16):
        assert _serialize_error(make)[0] == rt.INVALID_ARGUMENT, make
    for see in (dict(window=-1), dict(sinks=-1), dict(scale=0.0), dict(window=2 ** 31)):
        assert _serialize_error(lambda p: _tree(p, _operands(p), **see))[0] == rt.INVALID_ARGUMENT
    for fn in (rt.lib().thip_lm_tree_attention, rt.lib().thip_lm_cache_keep):
        assert fn(None, None) == rt.INVALID_ARGUMENT


def test_changed_records_are_refused_or_stay_inside():
    """Every 32-bit word of the records and of their further operands set to other values: a status each time; every extent that they name, larger, is refused."""
    p = thip.Program()
    v = _operands(p, dtype=np.int8)
    _tree(p, v, scales=True, window=9)
    _keep(p, v, scales=True, accepted=p.binding(21, (2, 5), I32))
    blob = bytearray(p.serialize())
    d = desc_interp.Descriptor(bytes(blob))
    size = d.ops.dtype.itemsize

    def status(b):
        words = (ctypes.c_uint64 * (len(b) // 8 + 1))()  # 8-byte aligned
        ctypes.memmove(words, bytes(b), len(b))
        return rt.lib().thip_descriptor_validate(words, len(b))

    assert status(blob) == rt.OK
    at = bytes(blob).index(d.ops[0].tobytes())
    for op in range(2):
        for word in range(size // 4):
            o = at + op * size + 4 * word
            old = bytes(blob[o:o + 4])
            for value in (0, 1, 3, 0x7FFFFFFF, 0x80000000, 0xFFFFFFFF, struct.unpack("<I", old)[0] + 1):
                blob[o:o + 4] = struct.pack("<I", value & 0xFFFFFFFF)
                assert status(blob) in (rt.OK, rt.INVALID_ARGUMENT)
            blob[o:o + 4] = old
        for field in ("M", "N", "W", "OH", "KW", "H") if op == 0 else ("N", "W", "OH", "KW", "K"):
            o = at + op * size + d.ops.dtype.fields[field][1]
            old = bytes(blob[o:o + 4])
            blob[o:o + 4] = struct.pack("<i", 2 * int(d.ops[op][field]) + 1)
            assert status(blob) == rt.INVALID_ARGUMENT, field
            blob[o:o + 4] = old
    for o in range(int(d.header["data_offset"]), len(blob) - 3, 4):
        old = bytes(blob[o:o + 4])
        for value in (1, 7, 0x7FFFFFFF, 0xFFFFFFFF):
            blob[o:o + 4] = struct.pack("<I", value)
            assert status(blob) in (rt.OK, rt.INVALID_ARGUMENT)
        blob[o:o + 4] = old


# ---- a decoder's layers that check a tree -------------------------------------------------------------------------------

def _layers(b, hidden, caches, parents, accepted, expose, layers=2):
    """Layers in one program: the norm before the block, grouped linears (int8 weights in blocks), norms of the heads, rotary positions of two axes, the cache's write,
    attention of the tree, the linear behind, and its norm with the residual and the next layer's norm; at the end what was accepted moves together in every
    layer's cache.  expose: what each op gives is a binding, else the program's own."""
    rng = np.random.default_rng(19)
    built = Built()
    p, M = built.program, b.T
    bf16 = lambda *shape: ref.to_bf16(rng.standard_normal(shape).astype(np.float32))  # noqa: E731
    zero, noclamp = np.zeros(1, np.float32), dict(output_zp=0, output_min=w.NO_CLAMP[0], output_max=w.NO_CLAMP[1])

    def linear(src, N, init):
        wq, scale, qbias = w._block_quantized(rng, src.shape[1], N, 128, 1.0)
        return p.matmul(src, p.expand_weights(wq, scale, qbias, block_size=128, output_min=w.NO_CLAMP[0], output_max=w.NO_CLAMP[1]), zero, init=init, shift=0, **noclamp)

    def place(name, shape, dtype=U16):
        return built.bind(name, np.zeros(shape, dtype)) if expose else p.tensor(shape, dtype)

    positions = rng.integers(0, 10 ** 5, size=(2, M)).astype(I32)
    frequencies = (10000.0 ** (-np.arange(b.D // 2) / (b.D // 2))).astype(np.float32)
    axes = (np.arange(b.D // 2) // 3 % 2).astype(I32)
    held = dict(positions=positions, frequencies=frequencies, axes=axes, norms=[])
    stream = built.bind("stream", rng.standard_normal((M, hidden)).astype(np.float32))  # the residual, in 32 bits
    x = built.bind("x", bf16(M, hidden))
    starts, lengths = built.rows(b)
    pages, up = built.bind("pages", b.pages), built.bind("parents", parents)
    turned = built.bind("positions", positions)
    kept = []
    for i in range(layers):
        weights = [bf16(n) for n in (b.D, b.D, hidden, hidden)]
        held["norms"].append(weights)
        q, k, v = (linear(x, h * b.D, place("%s%d" % (n, i), (M, h * b.D))) for n, h in zip(("q", "k", "v"), (b.H, b.KVH, b.KVH)))
        q, k, v = (p.view(t, (M, h, b.D)) for t, h in zip((q, k, v), (b.H, b.KVH, b.KVH)))
        q = p.norm(q, weights[0], eps=1e-6, init=place("qn%d" % i, (M, b.H, b.D)))
        k = p.norm(k, weights[1], eps=1e-6, init=place("kn%d" % i, (M, b.KVH, b.D)))
        q, k = p.rotary(q, k, turned, frequencies, axes=axes, query_out=place("qr%d" % i, (M, b.H, b.D)) if expose else q,
                        key_out=place("kr%d" % i, (M, b.KVH, b.D)) if expose else k)
        cache = built.bind("key_cache%d" % i, caches[i][0]), built.bind("value_cache%d" % i, caches[i][1]), pages
        scales = dict(key_scales=built.bind("key_scales%d" % i, caches[i][2]), value_scales=built.bind("value_scales%d" % i, caches[i][3]))
        kept.append((cache, scales))
        p.cache_write(k, v, *cache, starts, lengths, **scales)
        y = p.tree_attention(q, *cache, starts, lengths, up, scale=b.scale, window=90, sinks=2, init=p.view(place("y%d" % i, (M, b.H * b.D)), (M, b.H, b.D)), **scales)
        o = linear(p.view(y, (M, b.H * b.D)), hidden, place("o%d" % i, (M, hidden)))
        after = place("stream%d" % i, (M, hidden), np.float32) if expose else stream
        x = p.norm(o, weights[3], eps=1e-6, weight_offset=1.0, post_weight=weights[2], residual=stream, residual_out=after, residual_scale=0.5,
                   init=built.bind("out", np.zeros((M, hidden), U16)) if i == layers - 1 else place("x%d" % i, (M, hidden)))
        stream = after
    if accepted is not None:
        rows = built.bind("accepted", accepted)
        for cache, scales in kept:
            p.cache_keep(*cache, starts, lengths, rows, **scales)
    return built, held


LAYERS = [dict(sequences=[(1, 9), (5, 30), (3, 90)], D=64, H=4, KVH=1, page=16), dict(sequences=[(8, 40), (16, 200)], D=128, H=4, KVH=2, page=16, tail=2),
          dict(sequences=[(13, 130), (1, 1)], D=256, H=4, KVH=1, page=32)]


def test_a_layer_s_records():
    b = Batch(**LAYERS[0])
    caches = [b.caches + [None, None]] * 2
    built, _ = _layers(b, 256, caches, plant(b), np.zeros((3, 2), I32), False)
    assert [int(o["kind"]) for o in desc_interp.Descriptor(built.program.serialize()).ops] == [15, 23, 23, 22, 17, KIND_TREE, 15, 23] * 2 + [KIND_KEEP] * 2


@pytest.mark.gpu
@pytest.mark.parametrize("quantised", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("case", LAYERS, ids=_id)
def test_gpu_layers_that_check_a_tree(device, case, quantised):
    """Each op of the run is checked on what the ops before it gave; the program with intermediates of its own, some of them written in place, gives the same."""
    b, hidden = Batch(quantised=quantised, **case), 256
    other = Batch(quantised=quantised, seed=5, garbage=False, **case)  # the second layer's has the first one's pages
    caches = [c.caches + list(c.scales) for c in (b, other)]
    parents = plant(b)
    built, held = _layers(b, hidden, caches, parents, None, True)
    got = built.run(device)

    def near(name, want):
        result, bound = want
        have = layer.wide(got[name]).reshape(result.shape)
        assert (np.abs(have - result) <= bound).all(), name

    stream = dict(built.arrays)["stream"]
    for i, start in enumerate((b, other)):
        qw, kw, post, pre = held["norms"][i]
        for n, weight in (("q", qw), ("k", kw)):
            near("%sn%d" % (n, i), layer.norm(got["%s%d" % (n, i)].reshape(-1, b.D), weight, eps=1e-6)[0])
            near("%sr%d" % (n, i), layer.rotary(got["%sn%d" % (n, i)].reshape(b.T, -1, b.D), held["positions"], held["frequencies"], held["axes"]))
        cache = ref.Cache(start.caches[0], start.caches[1], b.pages, *start.scales)
        written = ref.cache_write(cache, got["kr%d" % i].reshape(b.T, -1, b.D), got["v%d" % i].reshape(b.T, -1, b.D), b.starts, b.lengths)
        for name, x in zip(("key_cache", "value_cache", "key_scales", "value_scales"), written):
            if x is not None:
                assert np.array_equal(got["%s%d" % (name, i)], x, equal_nan=x.dtype == np.float32), (name, i)
        cache = ref.Cache(written[0], written[1], b.pages, *written[2:])
        y = got["y%d" % i].reshape(b.T, b.H, b.D)
        check_attention(b, y, y, ref.tree_attention(got["qr%d" % i].reshape(b.T, -1, b.D), b.starts, b.lengths, parents, cache, b.scale, 90, 2, fine=True), "layer %d" % i)
        out = "out" if i else "x0"
        normed, sums = layer.norm(got["o%d" % i], pre, eps=1e-6, weight_offset=1.0, post_weight=post, residual=stream, residual_scale=0.5, sum_dtype=np.float32)
        near(out, normed)
        near("stream%d" % i, sums)
        stream = got["stream%d" % i]
    inside, _ = _layers(b, hidden, caches, parents, None, False)
    assert np.array_equal(inside.run(device)["out"], got["out"])
    # and with what was accepted moved behind: the caches are those of the rows' own order
    accepted = _accept(b, 6, "some", b.rng)
    moved = _layers(b, hidden, caches, parents, accepted, False)[0].run(device)
    assert np.array_equal(moved["out"], got["out"])
    for i in range(2):
        cache = ref.Cache(got["key_cache%d" % i], got["value_cache%d" % i], b.pages, got.get("key_scales%d" % i), got.get("value_scales%d" % i))
        for name, x in zip(("key_cache", "value_cache", "key_scales", "value_scales"), ref.cache_keep(cache, accepted, b.starts, b.lengths)):
            if x is not None:
                assert np.array_equal(moved["%s%d" % (name, i)], x, equal_nan=x.dtype == np.float32), (name, i)


@pytest.mark.gpu
def test_gpu_layers_without_an_allocation(device):
    """The same program enqueued kernel by kernel, without a graph and without an allocation, and replayed: the bits of each dispatch on fresh buffers."""
    b = Batch(**LAYERS[1])
    caches = [b.caches + [None, None], [x.copy() for x in b.caches] + [None, None]]
    built, _ = _layers(b, 256, caches, plant(b), _accept(b, 4, "some", b.rng), False)
    first = built.run(device)
    again = built.run(device, "noalloc")
    for name in ("out", "key_cache0", "value_cache1", "stream"):
        assert np.array_equal(first[name], again[name]), name


def test_programs_and_records_under_sanitizers(tmp_path):
    """Random programs of these ops, and mutated copies of their descriptors, through the emitter and the validation built with the sanitizers."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    csrc, exe = os.path.join(root, "torq-compiler_amd", "csrc"), str(tmp_path / "layer_host")
    built = subprocess.run([shutil.which("g++"), "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined", "-static-libasan", "-fno-sanitize-recover=undefined", "-w",
                            "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", "-I" + csrc, os.path.join(root, "tests", "fuzz", "layer_host.cpp")] +
                           [os.path.join(csrc, s) for s in ("thip_emitter.cpp", "thip_validate.cpp", "thip_status.cpp")] + ["-o", exe], stdout=subprocess.PIPE,
                           stderr=subprocess.STDOUT, text=True)
    assert built.returncode == 0, built.stdout[-3000:]
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=1:abort_on_error=0:verify_asan_link_order=0", UBSAN_OPTIONS="print_stacktrace=1")
    done = subprocess.run([exe, "400", "1"], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, env=env, timeout=300)
    assert done.returncode == 0 and "runtime error" not in done.stdout and "AddressSanitizer" not in done.stdout, done.stdout[-4000:]
