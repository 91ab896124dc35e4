"""Trees of drafted tokens whose rows go by tiles of 128 (thip_lm_tree_attention): what a key head's rows are so many for, or what there is so much text in front of, that
the launch takes tree_attention_tiles.  Every test makes sure of that by the kernel's name."""
import subprocess

import numpy as np
import pytest

import torq_compiler_amd as thip
from helpers import host_check
from oracle import attention as ref
from test_cache_attention import Batch, Built, check_attention
from test_tree import attend_tree, plant

U16, I32 = np.uint16, np.int32
BOTH = pytest.mark.parametrize("quantised", [False, True], ids=["bf16", "int8"])


def _id(case):
    return "-".join(str(v) if not isinstance(v, list) else "%dseq" % len(v) for v in case.values()).replace(" ", "")


def run(device, built, dispatches=1, via="device", kernel="tree_attention_tiles"):
    """The arrays behind the dispatches of a program whose only kernel is this one."""
    exe = thip.Executable(device, built.program.serialize())
    try:
        names = exe.op_kernels()
    finally:
        exe.close()
    assert len(names) == 1 and names[0].startswith(kernel + "<"), names
    return built.run(device, via, dispatches)


# So many rows that there are 64 tiles of 128 and more (of heads above 128 half as many, of int8 there twice).
MANY = [
    dict(sequences=[(130, 400), (100, 300), (1, 50), (0, 9), (3, 2)], D=64, H=40, KVH=8, page=16, tail=2),
    dict(sequences=[(70, 500)], D=128, H=128, KVH=16, page=24),
    dict(sequences=[(40, 200), (33, 40), (40, 33), (40, 200), (64, 64), (1, 300), (40, 64), (5, 200)], D=80, H=32, KVH=8, page=32),
    dict(sequences=[(60, 90), (40, 200)], D=96, H=96, KVH=3, page=7),
    dict(sequences=[(300, 700), (3, 90)], D=256, H=56, KVH=4, page=64),
    dict(sequences=[(150, 155)] * 2, D=176, H=55, KVH=11, page=16),
    dict(sequences=[(9, 20)] * 60, D=16, H=16, KVH=2, page=8),
]
SEEN = [dict(), dict(window=1), dict(window=20, sinks=3), dict(window=65, sinks=4), dict(window=40, sinks=100), dict(window=290, sinks=2 ** 31 - 1)]


# each shape without a window and under two of them
MANY_SEEN = [(c, see) for i, c in enumerate(MANY) for see in (SEEN[0], SEEN[1 + i % 5], SEEN[1 + (i + 2) % 5])]


@pytest.mark.gpu
@BOTH
@pytest.mark.parametrize("case,see", MANY_SEEN, ids=_id)
def test_gpu_many_rows(device, case, see, quantised):
    """Heads as long as their kernel's and shorter, sequences of one row and of none among long ones, places below 0."""
    b = Batch(quantised=quantised, **case)
    assert b.T * b.H >= (16384 if quantised and b.D > 128 else 8192)
    built, before, want = attend_tree(b, plant(b), **see)
    first = run(device, built)["out"]
    check_attention(b, first, before, want)
    assert np.array_equal(built.run(device, dispatches=3)["out"], first)


# Fewer rows, but tables for so much text that its reading counts: one or two tiles in place of many streams.  Weights meet their values in two parts here.
FEW = [
    dict(sequences=[(25, 60), (35, 100), (15, 300)], D=64, H=32, KVH=8, page=16),
    dict(sequences=[(40, 50), (30, 100)], D=80, H=15, KVH=5, page=32),
    dict(sequences=[(12, 900), (1, 40), (20, 20), (16, 3)], D=128, H=32, KVH=4, page=24, tail=1),
    dict(sequences=[(200, 900), (1, 2000), (2, 700), (130, 131)], D=64, H=8, KVH=2, page=24, tail=3),
    dict(sequences=[(50, 333)], D=96, H=2, KVH=1, page=128),
    dict(sequences=[(30, 250), (22, 900)], D=32, H=64, KVH=16, page=8),
]
FEW_OF_256 = [
    dict(sequences=[(25, 300), (26, 40)], D=256, H=16, KVH=4, page=16),
    dict(sequences=[(30, 1300)], D=208, H=3, KVH=1, page=24),
    dict(sequences=[(100, 110), (2, 500), (99, 600)], D=256, H=4, KVH=2, page=32, tail=2),
]


def with_room(case, quantised, **more):
    """The batch with so many entries in its table (none of which is a page) that tiles spare more reading than they cost."""
    S, KVH, T = len(case["sequences"]), case["KVH"], sum(n for n, _ in case["sequences"]) + case.get("tail", 0)
    tiles = ((T * case["H"] // KVH - 1) // S + 128) // 128
    blocks = (16384 if quantised else 2048) // (tiles * S * KVH) + 2
    return Batch(quantised=quantised, spare_entries=32 * blocks // case["page"] + 1, **case, **more)


@pytest.mark.gpu
@pytest.mark.parametrize("case,quantised", [(c, q) for q in (False, True) for c in FEW] + [(c, False) for c in FEW_OF_256], ids=lambda v: _id(v) if isinstance(v, dict) else "int8" if v else "bf16")
def test_gpu_few_rows_over_much_room(device, case, quantised):
    """Within the bound of weights in two parts, which is that of the result's own rounding and little more."""
    b = with_room(case, quantised)
    assert b.T * b.H < 8192
    for kind in ("bushy", "comb"):
        parents = plant(b, kind)
        built, before, _ = attend_tree(b, parents)
        first = run(device, built)["out"]
        check_attention(b, first, before, ref.tree_attention(b.query, b.starts, b.lengths, parents, b.cache(), b.scale, fine=True), kind)
    assert np.array_equal(built.run(device, "noalloc", dispatches=3)["out"], first)


@BOTH
@pytest.mark.parametrize("case", [FEW[0], FEW[4], FEW_OF_256[0]], ids=_id)
def test_the_bound_tells_weights_rounded_once(case, quantised):
    """Keys so small that weights are alike: results are sums of a few values, some next to nothing."""
    b = Batch(quantised=quantised, **dict(case, sequences=[(3, 3), (4, 6)]))
    b.caches[0] = (b.caches[0] // 40).astype(np.int8) if quantised else ref.to_bf16((ref.from_bf16(b.caches[0]) / 40).astype(np.float32))
    args = b.query, b.starts, b.lengths, plant(b, "chain"), b.cache(), b.scale
    exact, bound = ref.tree_attention(*args, fine=True)
    once = ref.from_bf16(ref.to_bf16(ref.tree_attention(*args, rounded=True)[0].astype(np.float32)))
    plain = ref.from_bf16(ref.to_bf16(exact.astype(np.float32)))
    assert (np.abs(once - exact) > bound).any() and (np.abs(plain - exact) <= bound).all()


@pytest.mark.gpu
@BOTH
@pytest.mark.parametrize("case,see", [
    (dict(sequences=[(60, 3100), (40, 1500), (30, 700)], D=64, H=64, KVH=16, page=24), dict(window=1000, sinks=5)),
    (dict(sequences=[(70, 2500), (68, 640)], D=128, H=64, KVH=8, page=16), dict(window=1900)),
    (dict(sequences=[(127, 1300), (2, 900)], D=256, H=128, KVH=8, page=32), dict(window=700, sinks=40)),
    (dict(sequences=[(64, 2600), (64, 900), (64, 70)], D=80, H=48, KVH=3, page=24), dict()),
], ids=["64", "128", "256", "80"])
def test_gpu_long_runs(device, case, see, quantised):
    """Runs that are cut into parts, of trees of different lengths; chains and bushes."""
    b = Batch(quantised=quantised, **case)
    for kind in ("chain", "bushy") if b.D < 256 else ("bushy",):
        built, before, want = attend_tree(b, plant(b, kind), **see)
        check_attention(b, run(device, built)["out"], before, want, kind)


@pytest.mark.gpu
@BOTH
@pytest.mark.parametrize("n,D,H,KVH", [(511, 64, 16, 4), (512, 64, 16, 4), (513, 64, 16, 2), (700, 64, 12, 4), (700, 128, 12, 1), (513, 256, 32, 2)])
def test_gpu_largest_trees(device, n, D, H, KVH, quantised):
    """Up to 512 rows; those behind see nothing, and nobody sees them, also where parents say so."""
    b = Batch([(n, n + 90), (3, 50)], D=D, H=H, KVH=KVH, page=16, quantised=quantised)
    for kind, see in (("bushy", dict()), ("chain", dict(window=30, sinks=95))):
        built, before, want = attend_tree(b, plant(b, kind), **see)
        check_attention(b, run(device, built)["out"], before, want, kind)


@pytest.mark.gpu
@BOTH
@pytest.mark.parametrize("D", [64, 128, 256])
def test_gpu_pages_that_are_none(device, D, quantised):
    """Text and drafted rows whose page is none are seen by nobody, such a row itself keeps the rest of its path; pages of eight positions and of odd lengths."""
    for page in (8, 7):
        b = Batch([(60, 200), (70, 400)], D=D, H=128, KVH=8, page=page, quantised=quantised)
        b.pages[0, 150 // page] = -1
        b.pages[0, 12 // page] = 2 ** 31 - 1
        b.pages[1, 360 // page] = 2 ** 30
        b.pages[1, 3] = -5
        for see in (dict(), dict(window=100, sinks=9)):
            built, before, want = attend_tree(b, plant(b), **see)
            check_attention(b, run(device, built)["out"], before, want)


@pytest.mark.gpu
@BOTH
@pytest.mark.parametrize("starts", [[0, 90, 40, 120], [50, 50, 50, 50], [-3, 20, 400, 7], [2 ** 31 - 1, 0, 3, -2 ** 31], [0, 120, 0, 120]])
def test_gpu_starts_that_do_not_ascend(device, starts, quantised):
    """Rows stay inside their tensors whatever row_starts holds, and an ordinary dispatch behind that is right (counters and workspace are as they were)."""
    b = Batch([(40, 1000), (40, 1500), (40, 500)], D=128, H=72, KVH=8, page=16, quantised=quantised)
    built, before, want = attend_tree(b, plant(b))
    exe = thip.Executable(device, built.program.serialize())
    try:
        assert exe.op_kernels()[0].startswith("tree_attention_tiles<")
        ptrs = [device.upload(a) for _, a in built.arrays]
        sizes = [a.nbytes for _, a in built.arrays]
        names = [n for n, _ in built.arrays]
        odd = device.upload(np.array(starts, I32))
        exe.run_device([odd if n == "row_starts" else p for n, p in zip(names, ptrs)], sizes)
        exe.run_device(ptrs, sizes)
        got = device.download(ptrs[names.index("out")], before.shape, before.dtype)
        for p in ptrs + [odd]:
            device.free(p)
    finally:
        exe.close()
    check_attention(b, got, before, want)  # no row is of no sequence


@pytest.mark.gpu
@BOTH
def test_gpu_many_sequences(device, quantised):
    """More sequences than a wave looks through at once, some of one row, and one whose run is cut into parts."""
    b = Batch([(1 + i % 23, 30 + 7 * i % 300) for i in range(90)] + [(60, 3000)], D=64, H=16, KVH=2, page=16, quantised=quantised)
    for see in (dict(), dict(window=100, sinks=2)):
        built, before, want = attend_tree(b, plant(b), **see)
        check_attention(b, run(device, built)["out"], before, want)


@pytest.mark.gpu
@BOTH
@pytest.mark.parametrize("case", [MANY[1], MANY[4], dict(sequences=[(40, 2000)] * 3, D=128, H=72, KVH=4, page=16)], ids=_id)
def test_gpu_results_over_the_queries(device, case, quantised):
    """init is the query's own bytes, also where runs are cut into parts."""
    b = Batch(quantised=quantised, **case)
    parents = plant(b)
    built = Built()
    q = built.bind("query", b.query)
    cache, scales = built.cache(b)
    starts, lengths = built.rows(b)
    built.program.tree_attention(q, *cache, starts, lengths, built.bind("parents", parents), init=q, scale=b.scale, **scales)
    check_attention(b, run(device, built)["query"], b.query, ref.tree_attention(b.query, b.starts, b.lengths, parents, b.cache(), b.scale))


@pytest.mark.gpu
@BOTH
@pytest.mark.parametrize("D,H", [(64, 16), (128, 16), (256, 32)])
def test_gpu_last_positions_of_32_bits(device, D, H, quantised):
    """Tables of 2^31 - 8 positions (all of their entries the same page) with trees that end there, or behind; the reference has the same rows a whole number of
    pages further down."""
    page, P = 8 * 127 * 113, 3 * 5 * 29 * 43
    assert page * P == 2 ** 31 - 8
    b = Batch([(520, 16)], D=D, H=H, KVH=1, page=16, quantised=quantised, garbage=False)
    shape = (1, 1, page, D)
    if quantised:
        b.caches = [b.rng.integers(-127, 128, size=shape, dtype=np.int8) for _ in range(2)]
        b.scales = [(b.rng.uniform(0.5, 1.5, size=shape[:3]) / 73).astype(np.float32) for _ in range(2)]
        b.scales[1][0, 0, page - 25] = np.nan  # a row that sees it is done again
    else:
        b.caches = [b.normal(*shape) for _ in range(2)]
        b.caches[1][0, 0, page - 25] = 0x7FC0
    parents = plant(b)
    for length in (2 ** 31 - 8, 2 ** 31 - 1, 2 ** 31 - 37)[:3 if D == 64 else 1]:
        see = dict(window=16, sinks=3 if length % 2 else 0)
        b.page, b.pages, b.lengths = page, np.zeros((1, 1), dtype=I32), np.array([length - (P - 1) * page], dtype=I32)
        near = ref.tree_attention(b.query, b.starts, b.lengths, parents, b.cache(), b.scale, **see)
        b.pages, b.lengths = np.zeros((1, P), dtype=I32), np.array([length], dtype=I32)
        built, out = Built(), b.normal(b.T, b.H, b.D)
        q = built.bind("query", b.query)
        cache, scales = built.cache(b)
        starts, lengths = built.rows(b)
        built.program.tree_attention(q, *cache, starts, lengths, built.bind("parents", parents), init=built.bind("out", out), scale=b.scale, **see, **scales)
        check_attention(b, run(device, built)["out"], out, near, str(length))


@pytest.mark.parametrize("seed", [1, 2, 3])
def test_blocks_of_a_tile(tmp_path, seed):
    """By the kernels' own arithmetic: a tile reads every position that its rows can see, and the parts of a run that is cut have all of its blocks
    (tests/host/tree_blocks.cpp); a count that were one block short is found."""
    exe = host_check("tree_blocks", tmp_path)
    run = subprocess.run([exe, str(seed)], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=300)
    assert run.returncode == 0 and int(run.stdout) > 1000, run.stdout[-2000:]
    short = subprocess.run([exe, str(seed), "short"], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=300)
    assert short.returncode == 1 and "FAIL" in short.stdout and "blocks, the sequence counts" in short.stdout, short.stdout[-2000:]


def test_streams_or_tiles(tmp_path):
    """The plan's choice next to what both sides took (tests/host/tree_rule.cpp)."""
    done = subprocess.run([host_check("tree_rule", tmp_path)], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=60)
    assert done.returncode == 0, done.stdout
