"""Attention and its cache (thip_lm_*) where a row's result hangs on what is easily lost: numbers that are none, values next to the largest,
positions at the ends of what 32 bits hold, batches of very unequal sequences, and the programs around the ops."""
import ctypes
import os
import shutil
import subprocess

import numpy as np
import pytest

import desc_interp
import torq_compiler_amd as thip
from helpers import host_check
from oracle import attention as ref
from oracle import programs as prog
from test_cache_attention import Batch, Built, attend, check_attention
from torq_compiler_amd import runtime as rt
from torq_compiler_amd import workloads as w

U16 = np.uint16


def _along(b, low, high, at):
    """Queries all the same vector of +1 and -1, keys so that a row scores `high` everywhere and `low` at the positions `at` of each sequence (before
    the maximum is taken off; both within a rounding of the cache)."""
    sign = np.where(b.rng.random(b.D) < 0.5, -1.0, 1.0)
    b.query[:] = ref.to_bf16(sign.astype(np.float32))
    unit = 1.0 / (b.D * b.scale)  # of a key along the sign, for a score of 1
    def put(where, score):
        if b.quantised:
            b.caches[0][where] = (127 * np.sign(score) * sign).astype(np.int8)
            b.scales[0][where] = abs(score) * unit / 127
        else:
            b.caches[0][where] = ref.to_bf16((score * unit * sign).astype(np.float32))
    for s, (_, length) in enumerate(b.sequences):
        for p in range(length):
            put((b.pages[s, p // b.page], slice(None), p % b.page), low if p in at else high)


FORMS = [
    dict(sequences=[(1, 90), (2, 50)], D=64, H=4, KVH=2),                                # streams
    dict(sequences=[(1, 900), (3, 700)], D=128, H=4, KVH=1),                             # cut
    dict(sequences=[(1, 800)], D=256, H=4, KVH=1),
    dict(sequences=[(70, 130), (40, 60)], D=64, H=4, KVH=2),                             # tiles
    dict(sequences=[(60, 1500), (1, 700), (2, 90)], D=128, H=8, KVH=2),                  # cut, with streams among them
    dict(sequences=[(130, 300), (1, 90)], D=256, H=16, KVH=1),
    dict(sequences=[(300, 400), (1, 80)], D=80, H=32, KVH=2),                            # weights rounded once
]


def _id(case):
    return "-".join("%dseq" % len(v) if isinstance(v, list) else str(v) for v in case.values())


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [np.nan, np.inf], ids=["nan", "inf"])
@pytest.mark.parametrize("case", FORMS, ids=_id)
def test_gpu_scales_that_are_no_number(device, case, bad):
    """The scale of a value that a row sees makes the row's result no number where the value's weight is nothing in 32 bits (0 times the scale, by the
    definition), and has no influence where a mask hides the position."""
    b = Batch(quantised=True, page=16, **case)
    low = {21, 47}
    _along(b, -4000.0, 0.0, low)
    for s, (_, length) in enumerate(b.sequences):
        for p in low & set(range(length)):
            b.scales[1][b.pages[s, p // b.page], :, p % b.page] = bad
    for see in (dict(), dict(window=8), dict(window=40, sinks=30)):
        built, before, want = attend(b, True, **see)
        if not see:
            assert np.isnan(want[0][:b.starts[-1]]).any()
        check_attention(b, built.run(device)["out"], before, want, str(see))


@pytest.mark.gpu
@pytest.mark.parametrize("case", FORMS, ids=_id)
def test_gpu_infinite_scales(device, case):
    """A value that is infinite makes infinities, of its codes' signs, and NaN where the code is 0."""
    b = Batch(quantised=True, page=16, **case)
    for s in range(len(b.sequences)):
        b.scales[1][b.pages[s, 1], :, 5] = np.inf
        b.caches[1][b.pages[s, 1], :, 5, ::7] = 0
    for see in (dict(), dict(window=8)):
        built, before, want = attend(b, True, **see)
        if not see:
            assert np.isinf(want[0][:b.starts[-1]]).any()
        check_attention(b, built.run(device)["out"], before, want, str(see))


@pytest.mark.gpu
@pytest.mark.parametrize("quantised", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("case", FORMS, ids=_id)
def test_gpu_values_next_to_the_largest(device, case, quantised):
    """Values of about 2^121, with weights that grow by 2^7.6 along a run: their sums pass what 32 bits hold only where weights pass 1."""
    b = Batch(quantised=quantised, page=16, garbage=False, **case)
    _along(b, 0.0, 5.3, set(range(40)) | set(range(70, 120)) | set(range(200, 680)))
    if quantised:
        b.scales[1][:] = b.scales[1] * np.float32(2.0 ** 121)
    else:
        b.caches[1][:] = ref.to_bf16((ref.from_bf16(b.caches[1]) * 2.0 ** 121).astype(np.float32))
    built, before, want = attend(b, True)
    with np.errstate(invalid="ignore"):
        assert np.nanmax(np.abs(want[0])) < 2.0 ** 126
    check_attention(b, built.run(device)["out"], before, want)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128, 256])
def test_gpu_prompts_of_values_next_to_the_largest(device, D):
    b = Batch([(90, 90), (3, 3), (200, 200)], D=D, H=4, KVH=2, tail=1)
    sign = np.where(b.rng.random(D) < 0.5, -1.0, 1.0)
    b.query[:] = ref.to_bf16(sign.astype(np.float32))
    score = np.zeros(b.T)
    for s, (n, _) in enumerate(b.sequences):
        score[b.starts[s] + 40:b.starts[s] + n] = 5.3
    b.key[:] = ref.to_bf16((score[:, None, None] / (D * b.scale) * sign).astype(np.float32))
    b.value[:] = ref.to_bf16((ref.from_bf16(b.value) * 2.0 ** 121).astype(np.float32))
    built, before, want = attend(b, False)
    check_attention(b, built.run(device)["out"], before, want)


# ---- programs around the ops ------------------------------------------------------------------------------------------

def _transposed_cache(between, quantised=False):
    """query times the transposed pages of a key cache, with `between` (an op, or none) where the transpose has been and the product has not; returns the
    program, the batch and its bindings."""
    b = Batch([(2, 20), (1, 9)], D=64, H=4, KVH=1, page=16, quantised=quantised, garbage=False)
    built = Built()
    pages = b.caches[0].shape[0]
    k, v = built.bind("key", b.key), built.bind("value", b.value)
    cache, scales = built.cache(b)
    starts, lengths = built.rows(b)
    x = b.normal(pages, 3, b.D)
    a, query = built.bind("x", x), built.bind("query", b.query)
    p = built.program
    turned = p.transpose(p.view(cache[0], (pages, b.page, b.D)), (0, 2, 1))
    if between == "write":
        p.cache_write(k, v, *cache, starts, lengths, **scales)
    elif between == "read":  # into the first rows of the key cache
        other = built.bind("other_keys", b.caches[0].copy()), built.bind("other_values", b.caches[1].copy())
        p.cache_read(*other, cache[2], starts, lengths, key=p.view(cache[0], (b.T, 1, b.D)), value=v, **scales)
    elif between == "attention":
        p.attention(query, k, v, starts, scale=b.scale, init=p.view(cache[0], (b.T, b.H, b.D)))
    elif between == "elsewhere":  # what is written are other bindings
        p.cache_read(*cache, starts, lengths, key=p.view(a, (b.T, 1, b.D)), value=v, **scales)
    out = built.bind("product", np.zeros((pages, 3, b.page), U16))
    p.matmul(built.values["x"], turned, np.array([0.0], np.float32), init=out, output_zp=0, output_min=w.NO_CLAMP[0], output_max=w.NO_CLAMP[1], shift=0)
    if between == "behind":
        p.cache_write(k, v, *cache, starts, lengths, **scales)
    return built, b, x


def _kinds(blob):
    return [int(o["kind"]) for o in desc_interp.Descriptor(blob).ops]


TRANSPOSE, DEC_MATMUL, WRITE, READ, ATTENTION = 1, 16, 17, 18, 19


@pytest.mark.parametrize("between,record", [("write", WRITE), ("read", READ), ("attention", ATTENTION)])
def test_transposes_stay_in_front_of_what_overwrites_their_input(between, record):
    built, _, _ = _transposed_cache(between)
    kinds = _kinds(built.program.serialize())
    assert kinds[0] == TRANSPOSE and record in kinds[1:] and DEC_MATMUL not in kinds, kinds


@pytest.mark.parametrize("between,kinds", [(None, [DEC_MATMUL]), ("behind", [DEC_MATMUL, WRITE]), ("elsewhere", [READ, DEC_MATMUL])])
def test_transposes_of_what_stays_are_read_in_place(between, kinds):
    built, _, _ = _transposed_cache(between)
    assert _kinds(built.program.serialize()) == kinds


@pytest.mark.gpu
@pytest.mark.parametrize("between", [None, "write", "read", "attention", "behind"])
def test_gpu_products_see_the_cache_as_it_was(device, between):
    built, b, x = _transposed_cache(between)
    got = built.run(device)["product"]
    turned = np.ascontiguousarray(b.caches[0].reshape(-1, b.page, b.D).transpose(0, 2, 1))
    want = prog.orc.matmul_bf16(x, turned, np.array([0.0], np.float32))
    mag = np.abs(ref.from_bf16(x)) @ np.abs(ref.from_bf16(turned))
    prog.assert_bf16_close(got, want, str(between), magnitude=mag)


def _over_an_intermediate(op, query_too=False):
    """An intermediate (rows that a transpose made) that attention, or a read of the cache, writes for the sequences' rows, then turned back into a
    binding."""
    b = Batch([(3, 20), (0, 5), (2, 9)], D=64, H=4, KVH=4, page=16, tail=4)
    built = Built()
    k, v = built.bind("key", b.key), built.bind("value", b.value)
    cache, scales = built.cache(b)
    starts, lengths = built.rows(b)
    p = built.program
    first = b.normal(b.T, b.H, b.D)
    rows = p.transpose(built.bind("first", np.ascontiguousarray(first.transpose(0, 2, 1))), (0, 2, 1))
    if op == "read":
        p.cache_read(*cache, starts, lengths, key=rows, value=v, **scales)
    else:
        p.paged_attention(rows if query_too else built.bind("query", b.query), *cache, starts, lengths, scale=b.scale, init=rows, **scales)
    p.transpose(rows, (0, 2, 1), init=built.bind("out", np.zeros((b.T, b.D, b.H), U16)))
    return built, b, first


@pytest.mark.parametrize("op,query_too", [("read", False), ("attention", False), ("attention", True)])
def test_intermediates_are_written_in_place(op, query_too):
    built, _, _ = _over_an_intermediate(op, query_too)
    made, record, back = desc_interp.Descriptor(built.program.serialize()).ops
    assert made["out"] == record["out"] and record["out"] == back["in0"]


@pytest.mark.gpu
@pytest.mark.parametrize("op,query_too", [("read", False), ("attention", False), ("attention", True)])
def test_gpu_rows_of_no_sequence_stay_in_intermediates(device, op, query_too):
    built, b, first = _over_an_intermediate(op, query_too)
    got = np.ascontiguousarray(built.run(device, dispatches=3)["out"].transpose(0, 2, 1))
    if op == "read":
        assert np.array_equal(got, ref.cache_read(b.cache(), first, b.value, b.starts, b.lengths)[0])
        assert np.array_equal(got[-4:], first[-4:])
    else:
        want = ref.attention(first if query_too else b.query, b.starts, b.scale, cache=b.cache(), lengths=b.lengths)
        check_attention(b, got, first, want)


def test_a_transposed_intermediate_that_attention_writes_is_no_operand_in_place():
    """The product behind it reads what attention left there, not what the transpose was made of."""
    b = Batch([(3, 3)], D=64, H=64, KVH=64)
    built = Built()
    p = built.program
    turned = p.transpose(built.bind("first", b.normal(b.T, b.D, b.H)), (0, 2, 1))
    p.attention(built.bind("query", b.query), built.bind("key", b.key), built.bind("value", b.value), built.bind("row_starts", b.starts), scale=b.scale,
                init=turned)
    p.matmul(built.bind("x", b.normal(b.T, 2, b.H)), turned, np.array([0.0], np.float32), init=built.bind("out", b.normal(b.T, 2, b.D)), output_zp=0,
             output_min=w.NO_CLAMP[0], output_max=w.NO_CLAMP[1], shift=0)
    kinds = _kinds(p.serialize())
    assert kinds[:2] == [TRANSPOSE, ATTENTION] and DEC_MATMUL not in kinds, kinds


# ---- the ends of 32 bits ------------------------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("quantised", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 3])
@pytest.mark.parametrize("case", [dict(sequences=[(5, 2), (9, 4), (8, 5), (3, 300)], D=64, H=4, KVH=2), dict(sequences=[(60, 20), (70, 69), (40, 90)], D=128, H=4, KVH=2),
                                  dict(sequences=[(9, 4)], D=256, H=4, KVH=1)], ids=_id)
def test_gpu_longest_windows(device, case, window, quantised):
    """A window that takes in everything, where the first rows of a sequence stand before its position 0."""
    b = Batch(quantised=quantised, page=16, **case)
    for sinks in (0, 3):
        built, before, want = attend(b, True, window=window, sinks=sinks)
        plain = ref.attention(b.query, b.starts, b.scale, cache=b.cache(), lengths=b.lengths)[0]
        assert np.array_equal(want[0], plain, equal_nan=True)
        check_attention(b, built.run(device)["out"], before, want)


@pytest.mark.gpu
@pytest.mark.parametrize("quantised", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("rows", [1, 3, 60])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_gpu_last_positions_of_32_bits(device, D, rows, quantised):
    """Tables of 2^31 - 8 positions (all of their entries the same page) with sequences that end there, or behind.  The reference has the same rows
    a whole number of pages further down."""
    page, P = 8 * 127 * 113, 3 * 5 * 29 * 43
    assert page * P == 2 ** 31 - 8
    rng = np.random.default_rng(D + rows)
    b = Batch([(rows, 16)], D=D, H=4, KVH=1, page=16, quantised=quantised, garbage=False)
    shape = (1, 1, page, D)
    if quantised:
        b.caches = [rng.integers(-127, 128, size=shape, dtype=np.int8) for _ in range(2)]
        b.scales = [(rng.uniform(0.5, 1.5, size=shape[:3]) / 73).astype(np.float32) for _ in range(2)]
        b.scales[1][0, 0, page - 25] = np.nan  # a row that sees it is done again
    else:
        b.caches = [b.normal(*shape) for _ in range(2)]
        b.caches[1][0, 0, page - 25] = 0x7FC0
    b.page, b.pages = page, np.zeros((1, P), dtype=np.int32)
    for length in (2 ** 31 - 8, 2 ** 31 - 1, 2 ** 31 - 37):
        for sinks in (0, 3):
            b.pages, b.lengths = np.zeros((1, 1), dtype=np.int32), np.array([length - (P - 1) * page], dtype=np.int32)
            near = ref.attention(b.query, b.starts, b.scale, window=16, sinks=sinks, cache=b.cache(), lengths=b.lengths)
            b.pages, b.lengths = np.zeros((1, P), dtype=np.int32), np.array([length], dtype=np.int32)
            built, out = Built(), b.normal(b.T, b.H, b.D)
            q = built.bind("query", b.query)
            cache, scales = built.cache(b)
            starts, lengths = built.rows(b)
            built.program.paged_attention(q, *cache, starts, lengths, init=built.bind("out", out), scale=b.scale, window=16, sinks=sinks, **scales)
            check_attention(b, built.run(device)["out"], out, near, "%d %d" % (length, sinks))


@pytest.mark.parametrize("see", [dict(window=2 ** 32), dict(window=2 ** 32 + 5), dict(sinks=2 ** 31), dict(window=-2 ** 32), dict(window=1.5)], ids=str)
@pytest.mark.parametrize("cached", [False, True], ids=["rows", "cache"])
def test_windows_that_a_field_would_not_hold_are_refused(see, cached):
    with pytest.raises(thip.ThipError) as e:
        attend(Batch([(2, 2)]), cached, **see)
    assert e.value.code == rt.INVALID_ARGUMENT and "32 bits" in e.value.message


# ---- batches of very unequal sequences ----------------------------------------------------------------------------------

@pytest.mark.parametrize("seed", [1, 2])
def test_shares_of_a_launch(tmp_path, seed):
    done = subprocess.run([host_check("attention_plan", tmp_path), str(seed)], stdout=subprocess.PIPE, text=True, timeout=120)
    assert done.returncode == 0 and int(done.stdout) > 500, done.stdout


SKEWED = [
    dict(sequences=[(1, 30)] * 40 + [(1, 3000)] + [(1, 50)] * 70 + [(0, 9)], D=16, H=8, KVH=8, page=16),              # streams, a long run in the first 64
    dict(sequences=[(1, 3)] * 290 + [(2, 2500)] + [(0, 4)] * 10 + [(1, 9)] * 20, D=16, H=2, KVH=2, page=32, tail=2),      # more than 256
    dict(sequences=[(1, 1 + i % 3) for i in range(4200)] + [(1, 500)] + [(1, 2)] * 3, D=16, H=1, KVH=1, page=8),          # groups of more than 64
    dict(sequences=[(1, 40)] * 66 + [(300, 2600)] + [(3, 1200)] + [(40, 50)] * 12, D=32, H=8, KVH=2, page=24, tail=1),    # tiles, streams among them
    dict(sequences=[(17, 100)] * 20 + [(17, 4100)] + [(17, 90)] * 50, D=16, H=16, KVH=8, page=16),                       # more than 384 tiles
]


@pytest.mark.gpu
@pytest.mark.parametrize("quantised", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("case", SKEWED, ids=_id)
def test_gpu_one_long_sequence_among_many(device, case, quantised):
    b = Batch(quantised=quantised, garbage=False, **case)
    for see in (dict(), dict(window=1500, sinks=3)):
        built, before, want = attend(b, True, **see)
        first = built.run(device)["out"]
        check_attention(b, first, before, want)
        assert np.array_equal(built.run(device, dispatches=3)["out"], first)


@pytest.mark.gpu
@pytest.mark.parametrize("case", SKEWED[:4], ids=_id)
def test_gpu_after_many_starts_that_do_not_ascend(device, case):
    """Starts that claim far more rows than there are, in batches of many sequences, leave nothing behind for the next dispatch."""
    b = Batch(garbage=False, **case)
    built, before, want = attend(b, True)
    exe = thip.Executable(device, built.program.serialize())
    ptrs = [device.upload(x) for _, x in built.arrays]
    try:
        names = [name for name, _ in built.arrays]
        starts, out = ptrs[names.index("row_starts")], ptrs[names.index("out")]
        odd = np.where(np.arange(len(b.starts)) % 2, b.T, 0).astype(np.int32)
        for x in (odd, b.starts, b.starts[::-1].copy(), odd[::-1].copy(), b.starts):
            for where, data in ((starts, x), (out, before)):  # the others claim rows behind the last sequence too
                rt.check(rt.lib().thip_device_h2d(device.handle, ctypes.c_void_p(where), data.ctypes.data_as(ctypes.c_void_p), data.nbytes))
            exe.run_device(ptrs, [a.nbytes for _, a in built.arrays])
        check_attention(b, device.download(out, before.shape, before.dtype), before, want)
    finally:
        for p in ptrs:
            device.free(p)
        exe.close()


def _two_attentions(quantised=False):
    """A program of attentions of other sizes, two of which are cut into parts (tiles of heads of 128, then streams of heads of 64 with more parts), and the first
    once more behind the others."""
    big = Batch([(300, 3000), (1, 900)], D=128, H=4, KVH=1, page=64, quantised=quantised, seed=1)
    few = Batch([(1, 2500), (2, 1900), (1, 30)], D=64, H=8, KVH=4, page=16, quantised=quantised, seed=2)
    none = Batch([(9, 40)], D=64, H=2, KVH=1, page=16, quantised=quantised, seed=3)
    built, wants = Built(), []
    for i, b in enumerate((big, few, none, big)):
        q, out = built.bind("query%d" % i, b.query), b.normal(b.T, b.H, b.D)
        k, v = built.bind("k%d" % i, b.caches[0]), built.bind("v%d" % i, b.caches[1])
        scales = dict(key_scales=built.bind("ks%d" % i, b.scales[0]), value_scales=built.bind("vs%d" % i, b.scales[1]))
        built.program.paged_attention(q, k, v, built.bind("p%d" % i, b.pages), built.bind("s%d" % i, b.starts), built.bind("l%d" % i, b.lengths), scale=b.scale,
                                      init=built.bind("out%d" % i, out), **scales)
        wants.append((b, out))
    return built, wants


def test_attentions_of_a_program_have_one_workspace():
    built, _ = _two_attentions()
    d = desc_interp.Descriptor(built.program.serialize())
    refs = [tuple(o["in1"].tolist()) for o in d.ops]
    assert refs[0] == refs[1] == refs[3] and refs[0][0] == 2 and refs[2][0] == 0 and len(d.temps) == 1
    alone = [Built(), Built()]
    sizes = []
    for built, case in zip(alone, (dict(sequences=[(300, 3000), (1, 900)], D=128, H=4, KVH=1, page=64), dict(sequences=[(1, 2500), (2, 1900), (1, 30)], D=64, H=8, KVH=4))):
        sizes.append(int(desc_interp.Descriptor(attend(Batch(**case), True)[0].program.serialize()).temps["size"][0]))
    assert int(d.temps["size"][0]) == max(sizes)


@pytest.mark.gpu
@pytest.mark.parametrize("quantised", [False, True], ids=["bf16", "int8"])
def test_gpu_attentions_one_after_another_in_one_workspace(device, quantised):
    built, wants = _two_attentions(quantised)
    first = built.run(device)
    for i, (b, out) in enumerate(wants):
        check_attention(b, first["out%d" % i], out, ref.attention(b.query, b.starts, b.scale, cache=b.cache(), lengths=b.lengths), str(i))
    again = built.run(device, dispatches=4)  # replayed as a graph from the second on
    for name in first:
        assert np.array_equal(first[name], again[name], equal_nan=first[name].dtype == np.float32), name


# ---- weights in two parts -----------------------------------------------------------------------------------------------

FINE = [
    dict(sequences=[(1, 3), (2, 5), (1, 9), (3, 40), (1, 2)], D=64, H=8, KVH=2, page=16),     # streams
    dict(sequences=[(1, 6), (2, 4), (4, 700)], D=128, H=8, KVH=2, page=16),
    dict(sequences=[(1, 7), (3, 3)], D=256, H=16, KVH=4, page=16),
    dict(sequences=[(70, 75), (40, 40)], D=64, H=4, KVH=2, page=16),                          # tiles of few rows
    dict(sequences=[(50, 55), (1, 5), (60, 900)], D=128, H=8, KVH=2, page=16),
    dict(sequences=[(140, 140)], D=256, H=16, KVH=1, page=16),
    dict(sequences=[(300, 300), (1, 4), (250, 300)], D=64, H=16, KVH=8, page=16),             # as one, but for the sequence of one row
]


def _few_keys(b):
    """Keys so small that the first rows' weights are alike: results there are sums of a few values, some next to nothing."""
    b.caches[0] = (b.caches[0] // 40).astype(np.int8) if b.quantised else ref.to_bf16((ref.from_bf16(b.caches[0]) / 40).astype(np.float32))
    b.key = ref.to_bf16((ref.from_bf16(b.key) / 40).astype(np.float32))


def _is_fine(b, cached):
    """Rows whose weights meet the values in two parts, as the header says."""
    G = b.H // b.KVH
    once = b.T * b.H >= 8192 and b.T * G > 32 * len(b.sequences)
    fine = np.ones(b.T, dtype=bool)
    for s, (n, _) in enumerate(b.sequences):
        fine[b.starts[s]:b.starts[s + 1]] = not once or (cached and n * G <= 16 and b.D <= 128)
    return fine


@pytest.mark.parametrize("quantised", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("case", FINE[:6], ids=_id)
def test_the_bound_tells_weights_rounded_once(case, quantised):
    b = Batch(quantised=quantised, **case)
    _few_keys(b)
    over = dict(cache=b.cache(), lengths=b.lengths)
    exact, bound = ref.attention(b.query, b.starts, b.scale, fine=True, **over)
    once = ref.from_bf16(ref.to_bf16(ref.attention(b.query, b.starts, b.scale, rounded=True, **over)[0].astype(np.float32)))
    plain = ref.from_bf16(ref.to_bf16(exact.astype(np.float32)))
    assert (np.abs(once - exact) > bound).any() and (np.abs(plain - exact) <= bound).all()


@pytest.mark.gpu
@pytest.mark.parametrize("keys", ["rows", "bf16", "int8"])
@pytest.mark.parametrize("case", FINE, ids=_id)
def test_gpu_weights_in_two_parts(device, case, keys):
    b = Batch(quantised=keys == "int8", **case)
    if keys == "rows":
        b.lengths = np.array([n for n, _ in b.sequences], dtype=np.int32)
    _few_keys(b)
    built, before, (result, coarse) = attend(b, keys != "rows")
    over = dict(cache=b.cache(), lengths=b.lengths) if keys != "rows" else dict(key=b.key, value=b.value)
    bound = ref.attention(b.query, b.starts, b.scale, fine=True, **over)[1]
    fine = _is_fine(b, keys != "rows")
    assert fine.any() or (keys == "rows" and case is FINE[-1])  # without a cache nothing goes as a stream among tiles
    check_attention(b, built.run(device)["out"], before, (result, np.where(fine[:, None, None], bound, coarse)))


# ---- a decoder's layers -------------------------------------------------------------------------------------------------

def _layers(b, hidden, caches, expose, layers=2):
    """Layers of grouped linears (int8 weights in blocks), a write into each layer's cache, attention over it, and the linear behind with the residual sum, in
    one program; expose: queries, keys, values and what attention gave are bindings, else the program's own."""
    rng = np.random.default_rng(17)
    built = Built()
    p, M = built.program, b.T
    x = built.bind("x", ref.to_bf16(rng.standard_normal((M, hidden)).astype(np.float32)))
    starts, lengths = built.rows(b)
    pages = built.bind("pages", b.pages)
    zero, noclamp = np.zeros(1, np.float32), dict(output_zp=0, output_min=w.NO_CLAMP[0], output_max=w.NO_CLAMP[1])
    half = ref.to_bf16(np.array([0.70703125, 0.70703125], dtype=np.float32))

    def linear(src, N, gain, init):
        K = src.shape[1]
        wq, scale, qbias = w._block_quantized(rng, K, N, 128, gain)
        return p.matmul(src, p.expand_weights(wq, scale, qbias, block_size=128, output_min=w.NO_CLAMP[0], output_max=w.NO_CLAMP[1]), zero, init=init, shift=0, **noclamp)

    def place(name, shape):
        return built.bind(name, np.zeros(shape, U16)) if expose else p.tensor(shape, U16)

    for i in range(layers):
        names = ["%s%d" % (n, i) for n in ("query", "key", "value", "attended")]
        q, k, v = (linear(x, h * b.D, 1.0, place(n, (M, h * b.D))) for n, h in zip(names, (b.H, b.KVH, b.KVH)))
        q, k, v = (p.view(t, (M, h, b.D)) for t, h in zip((q, k, v), (b.H, b.KVH, b.KVH)))
        cache = built.bind("key_cache%d" % i, caches[i][0]), built.bind("value_cache%d" % i, caches[i][1]), pages
        scales = dict(key_scales=built.bind("key_scales%d" % i, caches[i][2]), value_scales=built.bind("value_scales%d" % i, caches[i][3]))
        p.cache_write(k, v, *cache, starts, lengths, **scales)
        y = p.paged_attention(q, *cache, starts, lengths, scale=b.scale, window=90, sinks=2, init=p.view(place(names[3], (M, b.H * b.D)), (M, b.H, b.D)), **scales)
        o = linear(p.view(y, (M, b.H * b.D)), hidden, 1.0, p.tensor((M, hidden), U16))
        last = i == layers - 1
        x = p.add(x, o, half, zero, init=built.bind("out", np.zeros((M, hidden), U16)) if last else p.tensor((M, hidden), U16), shift_factor=0, **noclamp)
    return built


LAYERS = [dict(sequences=[(1, 1 + 13 * i) for i in range(7)], D=64, H=4, KVH=1, page=16), dict(sequences=[(1, 40 + 7 * i) for i in range(24)], D=128, H=4, KVH=2, page=16),
          dict(sequences=[(3, 30), (1, 200), (2, 2)], D=256, H=4, KVH=1, page=32)]


def test_a_layer_is_four_records():
    b = Batch(**LAYERS[0])
    caches = [b.caches + [None, None]] * 2
    assert _kinds(_layers(b, 256, caches, False).program.serialize()) == [15, WRITE, ATTENTION, 15] * 2


@pytest.mark.gpu
@pytest.mark.parametrize("quantised", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("case", LAYERS, ids=_id)
def test_gpu_layers_of_a_decoder(device, case, quantised):
    """Each attention of the run is checked on the queries, keys and values that the linears gave it, each cache on what was written; the program with
    intermediates of its own gives the same."""
    b, hidden = Batch(quantised=quantised, **case), 256
    other = Batch(quantised=quantised, seed=5, garbage=False, **case)  # the second layer's has the first one's pages
    caches = [c.caches + list(c.scales) for c in (b, other)]
    exposed = _layers(b, hidden, caches, True).run(device)
    for i, start in enumerate((b, other)):
        q, k, v, got = (exposed["%s%d" % (n, i)].reshape(b.T, -1, b.D) for n in ("query", "key", "value", "attended"))
        cache = ref.Cache(start.caches[0], start.caches[1], b.pages, *start.scales)
        written = ref.cache_write(cache, k, v, b.starts, b.lengths)
        for name, x in zip(("key_cache", "value_cache", "key_scales", "value_scales"), written):
            if x is not None:
                assert np.array_equal(exposed["%s%d" % (name, i)], x, equal_nan=x.dtype == np.float32), (name, i)
        cache = ref.Cache(written[0], written[1], b.pages, *written[2:])
        want = ref.attention(q, b.starts, b.scale, window=90, sinks=2, cache=cache, lengths=b.lengths, fine=True)
        check_attention(b, got, got, want, "layer %d" % i)
    inside = _layers(b, hidden, caches, False).run(device, dispatches=3)
    assert np.isfinite(ref.from_bf16(inside["out"])).all() and np.array_equal(inside["out"], exposed["out"])


def test_programs_and_records_under_sanitizers(tmp_path):
    """Random programs around a cache, and mutated copies of their descriptors, through the emitter and the validation built with the sanitizers."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    csrc, exe = os.path.join(root, "torq-compiler_amd", "csrc"), str(tmp_path / "attention_host")
    built = subprocess.run([shutil.which("g++"), "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined", "-static-libasan", "-fno-sanitize-recover=undefined", "-w",
                            "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", "-I" + csrc, os.path.join(root, "tests", "fuzz", "attention_host.cpp")] +
                           [os.path.join(csrc, s) for s in ("thip_emitter.cpp", "thip_validate.cpp", "thip_status.cpp")] + ["-o", exe], stdout=subprocess.PIPE,
                           stderr=subprocess.STDOUT, text=True)
    assert built.returncode == 0, built.stdout[-3000:]
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=1:abort_on_error=0:verify_asan_link_order=0", UBSAN_OPTIONS="print_stacktrace=1")
    done = subprocess.run([exe, "300", "1"], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, env=env, timeout=300)
    assert done.returncode == 0 and "runtime error" not in done.stdout and "AddressSanitizer" not in done.stdout, done.stdout[-4000:]


@pytest.mark.gpu
@pytest.mark.parametrize("quantised", [False, True], ids=["bf16", "int8"])
def test_gpu_tables_that_are_constants(device, quantised):
    """Starts, lengths and pages that a program carries itself, and tables that are parts of one binding."""
    b = Batch([(1, 700), (40, 90), (0, 3), (2, 2)], D=64, H=4, KVH=2, page=16, quantised=quantised, tail=1)
    want = ref.attention(b.query, b.starts, b.scale, cache=b.cache(), lengths=b.lengths)
    S, P = b.pages.shape
    for carried in (True, False):
        built, out = Built(), b.normal(b.T, b.H, b.D)
        q, p = built.bind("query", b.query), built.program
        k, v = built.bind("key_cache", b.caches[0]), built.bind("value_cache", b.caches[1])
        scales = dict(key_scales=built.bind("key_scales", b.scales[0]), value_scales=built.bind("value_scales", b.scales[1]))
        if carried:
            tables = b.pages, b.starts, b.lengths
        else:
            whole = built.bind("tables", np.concatenate([b.lengths, b.starts, b.pages.reshape(-1)]).astype(np.int32))
            tables = p.view(whole, (S, P), 2 * S + 1), p.view(whole, (S + 1,), S), p.view(whole, (S,), 0)
        p.paged_attention(q, k, v, *tables, scale=b.scale, init=built.bind("out", out), **scales)
        for via in ("device", "host"):
            check_attention(b, built.run(device, via)["out"], out, want, "%s %s" % (carried, via))


@pytest.mark.gpu
@pytest.mark.parametrize("keys", ["rows", "bf16", "int8"])
@pytest.mark.parametrize("case", [dict(sequences=[(300, 300)], D=64, H=4, KVH=2), dict(sequences=[(90, 90), (5, 5)], D=256, H=2, KVH=1),
                                  dict(sequences=[(60, 1500), (1, 900)], D=128, H=8, KVH=2)], ids=_id)
def test_gpu_rows_of_nothing_but_nan(device, case, keys):
    """Whole rows of NaN in keys or values, which every later row sees."""
    if keys == "rows":  # prompts have no positions before their first row
        case = dict(case, sequences=[(n, n) for n, _ in case["sequences"]])
    for which in (0, 1):
        b = Batch(quantised=keys == "int8", page=16, **case)
        for s, (n, length) in enumerate(b.sequences):
            for p in {2, 33, length - 2} & set(range(length)):
                if keys == "rows":
                    (b.key, b.value)[which][b.starts[s] + p] = 0x7FC0
                elif keys == "int8":
                    b.scales[which][b.pages[s, p // 16], :, p % 16] = np.nan
                else:
                    b.caches[which][b.pages[s, p // 16], :, p % 16] = 0x7FC0
        for see in (dict(), dict(window=30, sinks=1)):
            built, before, want = attend(b, keys != "rows", **see)
            assert np.isnan(want[0]).any()
            check_attention(b, built.run(device)["out"], before, want, "%d %s" % (which, see))


@pytest.mark.gpu
@pytest.mark.parametrize("later", [False, True], ids=["all", "first"])
def test_gpu_values_behind_scores_of_minus_infinity(device, later):
    """Keys that give scores of minus infinity, all of a row's or the first 100, one of them with a value of NaN: zeros where no weight is above 0, else NaN."""
    b = Batch([(1, 200), (90, 120), (120, 120)], D=64, H=2, KVH=1, page=16)
    b.query[:, :, 0] = 0x3F80
    for s, (_, length) in enumerate(b.sequences):
        for p in range(100 if later else length):
            b.caches[0][b.pages[s, p // 16], 0, p % 16, 0] = 0xFF80
        b.caches[1][b.pages[s, 2], 0, 3] = 0x7FC0
    built, before, want = attend(b, True)
    assert (want[0][b.starts[2] + 90] == 0).all() and (np.isnan(want[0][0]).all() if later else (want[0][0] == 0).all())
    check_attention(b, built.run(device)["out"], before, want)


def _product_over_its_operand():
    """x times a transposed binding, into the bytes of that binding."""
    rng = np.random.default_rng(3)
    x, keys = (ref.to_bf16(rng.standard_normal(shape).astype(np.float32)) for shape in ((3, 4, 64), (3, 64, 64)))
    built = Built()
    a, whole = built.bind("x", x), built.bind("keys", keys)
    p = built.program
    p.matmul(a, p.transpose(whole, (0, 2, 1)), np.array([0.0], np.float32), init=p.view(whole, (3, 4, 64), 64), output_zp=0, output_min=w.NO_CLAMP[0],
             output_max=w.NO_CLAMP[1], shift=0)
    return built, x, keys


def test_a_product_does_not_read_in_place_what_it_overwrites():
    kinds = _kinds(_product_over_its_operand()[0].program.serialize())
    assert TRANSPOSE in kinds and DEC_MATMUL not in kinds, kinds


@pytest.mark.gpu
def test_gpu_product_over_its_operand(device):
    built, x, keys = _product_over_its_operand()
    got = built.run(device)["keys"].reshape(-1)
    turned = np.ascontiguousarray(keys.transpose(0, 2, 1))
    want = prog.orc.matmul_bf16(x, turned, np.array([0.0], np.float32))
    prog.assert_bf16_close(got[64:64 + 768].reshape(3, 4, 64), want, "over its operand", magnitude=np.abs(ref.from_bf16(x)) @ np.abs(ref.from_bf16(turned)))
    rest = np.ones(got.size, dtype=bool)
    rest[64:64 + 768] = False
    assert np.array_equal(got[rest], keys.reshape(-1)[rest])
