"""Attention of packed rows, over themselves and over a paged cache, and the cache's writes and reads (thip_lm_*): records and refusals on the
CPU, results on the GPU against the 64-bit definition (oracle/attention.py, which derives the bound that is held)."""
import ctypes
import struct

import numpy as np
import pytest

import desc_interp
import torq_compiler_amd as thip
from oracle import attention as ref
from torq_compiler_amd import runtime as rt

U16 = np.uint16
KIND_WRITE, KIND_READ, KIND_ATTENTION = 17, 18, 19


class Batch:
    """Sequences of (rows, length) with queries, keys and values, a cache with contents and their tables, from a seed."""

    def __init__(self, sequences, H=4, KVH=1, D=64, page=16, quantised=False, tail=0, seed=0, spare_entries=0, garbage=True):
        rng = self.rng = np.random.default_rng(seed)
        self.sequences, self.H, self.KVH, self.D, self.page, self.quantised = sequences, H, KVH, D, page, quantised
        self.starts = np.concatenate([[0], np.cumsum([n for n, _ in sequences])]).astype(np.int32)
        self.lengths = np.array([length for _, length in sequences], dtype=np.int32)
        self.T = T = max(int(self.starts[-1]) + tail, 1)
        S = len(sequences)
        P = max(1, -(-int(max(self.lengths.max(), 1)) // page)) + spare_entries
        NP = S * P + 3
        self.pages = rng.permutation(NP)[:S * P].reshape(S, P).astype(np.int32)
        for s in range(S):  # no page behind a sequence's last
            self.pages[s, -(-int(self.lengths[s]) // page):] = rng.choice([-1, NP, 2 ** 31 - 1, -2 ** 31], size=P - -(-int(self.lengths[s]) // page))
        shape = (NP, KVH, page, D)
        self.scales = (None, None)
        if quantised:
            self.caches = [rng.integers(-127, 128, size=shape, dtype=np.int8) for _ in range(2)]
            self.scales = [(rng.uniform(0.5, 1.5, size=shape[:3]) / 73).astype(np.float32) for _ in range(2)]
        else:
            self.caches = [self.normal(*shape) for _ in range(2)]
        if garbage:  # what no sequence has holds NaN and infinities
            mine = np.zeros((NP, page), dtype=bool)
            for s, (_, length) in enumerate(sequences):
                for p in range(length):
                    mine[self.pages[s, p // page], p % page] = True
            for k in range(2):
                if quantised:
                    self.scales[k][np.broadcast_to(~mine[:, None], shape[:3])] = np.nan if k else np.inf
                else:
                    self.caches[k][np.broadcast_to(~mine[:, None, :, None], shape)] = 0x7FC0 if k else 0xFF80
        self.query, self.key, self.value = self.normal(T, H, D), self.normal(T, KVH, D), self.normal(T, KVH, D)
        self.scale = float(np.float32(1 / np.sqrt(D)))

    def normal(self, *shape):
        return ref.to_bf16(self.rng.standard_normal(shape).astype(np.float32))

    def cache(self):
        return ref.Cache(self.caches[0], self.caches[1], self.pages, *self.scales)


class Built:
    """A program whose bindings are named arrays."""

    def __init__(self):
        self.program, self.arrays, self.values = thip.Program(), [], {}

    def bind(self, name, array):
        if array is None:
            return None
        v = self.program.binding(len(self.arrays), array.shape, array.dtype)
        self.arrays.append((name, array))
        self.values[name] = v
        return v

    def cache(self, b):
        """Bindings of a batch's cache; returns the operands (key_cache, value_cache, pages) and the scales."""
        k, v = self.bind("key_cache", b.caches[0]), self.bind("value_cache", b.caches[1])
        pages = self.bind("pages", b.pages)
        return (k, v, pages), dict(key_scales=self.bind("key_scales", b.scales[0]), value_scales=self.bind("value_scales", b.scales[1]))

    def rows(self, b):
        return self.bind("row_starts", b.starts), self.bind("lengths", b.lengths)

    def run(self, device, via="device", dispatches=1):
        """The arrays after the last dispatch, by name."""
        exe = thip.Executable(device, self.program.serialize())
        try:
            if via == "host":
                arrays = [a.copy() for _, a in self.arrays]
                for _ in range(dispatches):
                    exe.run_host(arrays)
                return {name: a for (name, _), a in zip(self.arrays, arrays)}
            ptrs = [device.upload(a) for _, a in self.arrays]
            sizes = [a.nbytes for _, a in self.arrays]
            try:
                for _ in range(dispatches):
                    if via == "noalloc":
                        exe.enqueue_device_noalloc(ptrs, sizes)
                        exe.wait()
                    else:
                        exe.run_device(ptrs, sizes)
                return {name: device.download(p, a.shape, a.dtype) for p, (name, a) in zip(ptrs, self.arrays)}
            finally:
                for p in ptrs:
                    device.free(p)
        finally:
            exe.close()


def attend(b, cached, window=0, sinks=0):
    """A program of one attention over the batch, what it starts `out` with, and the reference (result, bound)."""
    built = Built()
    out = b.normal(b.T, b.H, b.D)
    q = built.bind("query", b.query)
    see = dict(scale=b.scale, window=window, sinks=sinks)
    if cached:
        cache, scales = built.cache(b)
        starts, lengths = built.rows(b)
        built.program.paged_attention(q, *cache, starts, lengths, init=built.bind("out", out), **see, **scales)
        want = ref.attention(b.query, b.starts, cache=b.cache(), lengths=b.lengths, **see)
    else:
        k, v = built.bind("key", b.key), built.bind("value", b.value)
        built.program.attention(q, k, v, built.bind("row_starts", b.starts), init=built.bind("out", out), **see)
        want = ref.attention(b.query, b.starts, key=b.key, value=b.value, **see)
    return built, out, want


def check_attention(b, got, before, want, what=""):
    result, bound = want
    mine = np.zeros(b.T, dtype=bool)
    for row, _, _ in ref.places(b.starts, b.lengths, b.T):
        mine[row] = True
    assert np.array_equal(got[~mine], before[~mine]), "rows of no sequence were written " + what
    far = np.abs(ref.from_bf16(got[mine]) - result[mine])
    nan = np.isnan(result[mine])
    assert np.array_equal(np.isnan(ref.from_bf16(got[mine])), nan), "NaN in other places " + what
    with np.errstate(invalid="ignore"):
        over = ~nan & ~(far <= bound[mine]) & ~(ref.from_bf16(got[mine]) == result[mine])
    assert not over.any(), "%s: %d values off, by up to %g times what is allowed" % (what, over.sum(), np.max((far / bound[mine])[over]))


# ---- CPU: records -----------------------------------------------------------------------------------------------------

def test_records_and_bindings():
    """One record for each op; what is written in place is an input of the dispatch too, the tables are read only."""
    b = Batch([(2, 5), (3, 20)], quantised=True)
    built = Built()
    q, k, v = built.bind("query", b.query), built.bind("key", b.key), built.bind("value", b.value)
    cache, scales = built.cache(b)
    starts, lengths = built.rows(b)
    p = built.program
    p.cache_write(k, v, *cache, starts, lengths, **scales)
    y = p.paged_attention(q, *cache, starts, lengths, scale=0.125, **scales)
    z = p.attention(p.view(y, (b.T, b.H, b.D)), k, v, starts, scale=0.125, init=built.bind("out", b.query))
    assert z is built.values["out"]
    p.cache_read(*cache, starts, lengths, key=built.bind("rk", b.key), value=built.bind("rv", b.key), **scales)
    blob = p.serialize()
    kinds = [int(o["kind"]) for o in desc_interp.Descriptor(blob).ops]
    assert kinds == [KIND_WRITE, KIND_ATTENTION, KIND_ATTENTION, KIND_READ]
    _, bindings, _ = rt.describe_blob(blob)
    modes = {name: (bool(x["is_read_only"]), bool(x["is_write_only"])) for (name, _), x in zip(built.arrays, bindings)}
    both = ("key_cache", "value_cache", "key_scales", "value_scales", "out", "rk", "rv")
    assert modes == {name: (name not in both, False) for name in modes}


def _serialize_error(make):
    with pytest.raises(thip.ThipError) as e:
        p = thip.Program()
        make(p)
        p.serialize()
    return e.value.code, e.value.message


def _operands(p, T=5, H=4, KVH=2, D=64, S=2, P=4, NP=9, PS=16, dtype=U16, **other):
    """Bindings of one attention over a cache; `other` replaces shapes by name."""
    shapes = dict(query=((T, H, D), U16), out=((T, H, D), U16), key=((T, KVH, D), U16), value=((T, KVH, D), U16), key_cache=((NP, KVH, PS, D), dtype),
                  value_cache=((NP, KVH, PS, D), dtype), pages=((S, P), np.int32), row_starts=((S + 1,), np.int32), lengths=((S,), np.int32),
                  key_scales=((NP, KVH, PS), np.float32), value_scales=((NP, KVH, PS), np.float32))
    shapes.update(other)
    return {name: p.binding(i, *spec) for i, (name, spec) in enumerate(shapes.items())}


def _paged(p, v, scales=False, **see):
    see.setdefault("scale", 0.125)
    s = dict(key_scales=v["key_scales"], value_scales=v["value_scales"]) if scales else {}
    p.paged_attention(v["query"], v["key_cache"], v["value_cache"], v["pages"], v["row_starts"], v["lengths"], init=v["out"], **see, **s)


REFUSED = [
    (dict(D=72), rt.UNIMPLEMENTED, "multiples of 16"),
    (dict(D=272), rt.UNIMPLEMENTED, "multiples of 16"),
    (dict(H=3), rt.INVALID_ARGUMENT, "query heads"),
    (dict(out=((5, 4, 32), U16)), rt.INVALID_ARGUMENT, "expected [5, 4, 64]"),
    (dict(out=((5, 4, 64), np.int16)), rt.INVALID_ARGUMENT, "bf16"),
    (dict(query=((20, 64), U16)), rt.INVALID_ARGUMENT, "rank"),
    (dict(value_cache=((9, 2, 16, 32), U16)), rt.INVALID_ARGUMENT, "differ in dimension 3"),
    (dict(value_cache=((9, 2, 16, 64), np.int8)), rt.INVALID_ARGUMENT, "element type"),
    (dict(dtype=np.int16), rt.UNIMPLEMENTED, "int8 or bf16"),
    (dict(dtype=np.int8), rt.INVALID_ARGUMENT, "key_scales"),
    (dict(pages=((3, 4), np.int32)), rt.INVALID_ARGUMENT, "sequences"),
    (dict(pages=((8,), np.int32)), rt.INVALID_ARGUMENT, "rank"),
    (dict(lengths=((3,), np.int32)), rt.INVALID_ARGUMENT, "sequences"),
    (dict(lengths=((2,), np.int16)), rt.INVALID_ARGUMENT, "element type"),
    (dict(row_starts=((1,), np.int32)), rt.INVALID_ARGUMENT, "row_starts"),
    (dict(pages=((2, 1 << 28), np.int32)), rt.UNIMPLEMENTED, "positions"),
    (dict(key_cache=((1 << 29, 2, 16, 64), U16), value_cache=((1 << 29, 2, 16, 64), U16)), rt.UNIMPLEMENTED, "2^31"),
]


@pytest.mark.parametrize("shapes,code,text", REFUSED, ids=[t[2] + str(i) for i, t in enumerate(REFUSED)])
def test_refused_shapes(shapes, code, text):
    got, message = _serialize_error(lambda p: _paged(p, _operands(p, **shapes)))
    assert got == code and text in message, (got, message)


@pytest.mark.parametrize("see", [dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(window=-1), dict(sinks=-1)])
def test_refused_attributes(see):
    assert _serialize_error(lambda p: _paged(p, _operands(p), **see))[0] == rt.INVALID_ARGUMENT


@pytest.mark.parametrize("scale,taken", [(2.5e38, False), (1.9e38, True)])
def test_scales_that_are_no_number_in_powers_of_two(scale, taken):
    """Exponents are taken to base 2: the scale times log2(e) has to be a number, or a score of 0 were none."""
    if taken:
        p = thip.Program()
        _paged(p, _operands(p), scale=scale)
        p.serialize()
    else:
        assert _serialize_error(lambda p: _paged(p, _operands(p), scale=scale))[0] == rt.INVALID_ARGUMENT


def test_refused_operands():
    def scales_of_bf16(p):
        _paged(p, _operands(p), scales=True)

    def wrong_scales(p):
        _paged(p, _operands(p, dtype=np.int8, value_scales=((9, 2, 8), np.float32)), scales=True)

    def cache_of_a_program(p):
        v = _operands(p)
        v["key_cache"] = p.tensor((9, 2, 16, 64), U16)
        _paged(p, v)

    def shared(p):
        v = _operands(p)
        v["out"] = p.view(v["key_cache"], (5, 4, 64))
        _paged(p, v)

    def shifted(p):
        v = _operands(p, query=((6, 4, 64), U16))
        v["out"], v["query"] = p.view(v["query"], (5, 4, 64), offset=256), p.view(v["query"], (5, 4, 64))
        _paged(p, v)

    def one_cache_for_both(p):
        v = _operands(p)
        p.cache_write(v["key"], v["value"], v["key_cache"], v["key_cache"], v["pages"], v["row_starts"], v["lengths"])

    def rows_in_the_cache(p):
        v = _operands(p)
        p.cache_write(p.view(v["key_cache"], (5, 2, 64)), v["value"], v["key_cache"], v["value_cache"], v["pages"], v["row_starts"], v["lengths"])

    def same_rows(p):
        v = _operands(p)
        p.cache_read(v["key_cache"], v["value_cache"], v["pages"], v["row_starts"], v["lengths"], key=v["key"], value=v["key"])

    def pages_alone(p):
        v = _operands(p)
        op = rt.LmAttention(v["out"].index, v["query"].index, v["key_cache"].index, v["value_cache"].index, -1, -1, v["pages"].index,
                            v["row_starts"].index, -1, 0.125, 0, 0)
        rt.check(rt.lib().thip_lm_attention(p._h, ctypes.byref(op)))

    for make in (scales_of_bf16, wrong_scales, cache_of_a_program, shared, shifted, one_cache_for_both, rows_in_the_cache, same_rows, pages_alone):
        assert _serialize_error(make)[0] == rt.INVALID_ARGUMENT, make.__name__

    def odd_view(p):
        v = _operands(p, query=((6, 4, 64), U16))
        v["query"] = p.view(v["query"], (5, 4, 64), offset=4)
        _paged(p, v)

    assert _serialize_error(odd_view)[0] == rt.UNIMPLEMENTED
    with pytest.raises(thip.ThipError):
        p = thip.Program()
        v = _operands(p)
        p.cache_read(v["key_cache"], v["value_cache"], v["pages"], v["row_starts"], v["lengths"])
    lib = rt.lib()
    for fn in (lib.thip_lm_cache_write, lib.thip_lm_cache_read, lib.thip_lm_attention):
        assert fn(None, None) == rt.INVALID_ARGUMENT


def test_changed_records_are_refused_or_stay_inside():
    """Every 32-bit word of the records and of the cache's operands set to other values: a status each time, and what passes still asks for
    no more than its buffers have (every extent that the record names, larger, is refused)."""
    p = thip.Program()
    v = _operands(p, dtype=np.int8)
    s = dict(key_scales=v["key_scales"], value_scales=v["value_scales"])
    cache = (v["key_cache"], v["value_cache"], v["pages"], v["row_starts"], v["lengths"])
    p.cache_write(v["key"], v["value"], *cache, **s)
    p.paged_attention(v["query"], *cache, scale=0.125, init=v["out"], **s)
    p.cache_read(*cache, key=v["key"], value=v["value"], **s)
    blob = bytearray(p.serialize())
    d = desc_interp.Descriptor(bytes(blob))
    size = d.ops.dtype.itemsize
    lib = rt.lib()

    def status(b):
        words = (ctypes.c_uint64 * (len(b) // 8 + 1))()  # 8-byte aligned
        ctypes.memmove(words, bytes(b), len(b))
        return lib.thip_descriptor_validate(words, len(b))

    assert status(blob) == rt.OK
    at = bytes(blob).index(d.ops[0].tobytes())
    for op in range(3):
        for word in range(size // 4):
            o = at + op * size + 4 * word
            old = bytes(blob[o:o + 4])
            for value in (0, 1, 3, 0x7FFFFFFF, 0x80000000, 0xFFFFFFFF, struct.unpack("<I", old)[0] + 1):
                blob[o:o + 4] = struct.pack("<I", value & 0xFFFFFFFF)
                assert status(blob) in (rt.OK, rt.INVALID_ARGUMENT)
            blob[o:o + 4] = old
        for field in ("M", "N", "W", "OH", "KW", "H"):
            if int(d.ops[op][field]) == 0:
                continue
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


def test_reference_against_differences():
    """The reference itself: its result is the mean under the softmax (checked by the derivative of the log of the sum with respect to a shift of
    the scores along the values), a window as long as the prompt is none, and all of a row's weight on one key gives that key's value."""
    b = Batch([(7, 7)], D=16, H=2, KVH=2)
    plain, _ = ref.attention(b.query, b.starts, b.scale, key=b.key, value=b.value)
    wide, _ = ref.attention(b.query, b.starts, b.scale, window=7, key=b.key, value=b.value)
    assert np.allclose(plain, wide, rtol=0, atol=0)
    q, k, v = (ref.from_bf16(x) for x in (b.query, b.key, b.value))
    for h in range(2):
        for row in range(7):
            x = k[:row + 1, h] @ q[row, h] * b.scale
            f = lambda t: np.log(np.sum(np.exp(x + t * v[:row + 1, h, 3])))  # noqa: E731
            assert abs((f(1e-5) - f(-1e-5)) / 2e-5 - plain[row, h, 3]) < 1e-8
    alone, _ = ref.attention(b.query, b.starts, b.scale, window=1, key=b.key, value=b.value)
    assert np.allclose(alone, v, rtol=1e-15)


# ---- GPU: the cache's rows ------------------------------------------------------------------------------------------

ROWS = [
    dict(sequences=[(1, 1)], D=16, KVH=1, page=1),
    dict(sequences=[(1, 9), (0, 5), (1, 0), (3, 40)], D=64, KVH=2, page=16, tail=2),
    dict(sequences=[(0, 0), (5, 5), (0, 3), (33, 100), (0, 7)], D=80, KVH=3, page=24, tail=5, spare_entries=2),
    dict(sequences=[(2, 1), (7, 3), (4, 4)], D=96, KVH=1, page=7),
    dict(sequences=[(130, 200), (1, 1), (64, 64)], D=128, KVH=8, page=64),
    dict(sequences=[(1, 300)] * 40 + [(0, 2)] * 5 + [(2, 9)], D=256, KVH=1, page=16),
    dict(sequences=[(9, 9), (50, 61)], D=208, KVH=2, page=128, tail=1),
    dict(sequences=[(1, 5)] * 1100, D=16, KVH=1, page=4, tail=3),  # more sequences than LDS holds starts of
]


def _id(case):
    return "-".join(str(v) if not isinstance(v, list) else "%dseq" % len(v) for v in case.values()).replace(" ", "")


@pytest.mark.gpu
@pytest.mark.parametrize("quantised", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("case", ROWS, ids=_id)
def test_gpu_cache_write_and_read(device, case, quantised):
    """Writing equals the definition bit for bit, everything else in the cache and in the rows stays as it was, and so does reading back."""
    b = Batch(quantised=quantised, **case)
    grow = np.exp(3 * b.rng.standard_normal((b.T, b.KVH, 1)))
    b.key, b.value = (ref.to_bf16((ref.from_bf16(x) * grow).astype(np.float32)) for x in (b.key, b.value))
    written = Built()
    k, v = written.bind("key", b.key), written.bind("value", b.value)
    cache, scales = written.cache(b)
    written.program.cache_write(k, v, *cache, *written.rows(b), **scales)
    want = ref.cache_write(b.cache(), b.key, b.value, b.starts, b.lengths)
    for via in ("device", "host"):
        got = written.run(device, via)
        for name, x in zip(("key_cache", "value_cache", "key_scales", "value_scales"), want):
            if x is not None:
                bits = np.uint32 if x.dtype == np.float32 else x.dtype
                assert np.array_equal(got[name].view(bits), x.view(bits)), (name, via)
    read = Built()
    b.caches, b.scales = want[:2], want[2:]
    cache, scales = read.cache(b)
    before = b.normal(b.T, b.KVH, b.D), b.normal(b.T, b.KVH, b.D)
    read.program.cache_read(*cache, *read.rows(b), key=read.bind("key", before[0]), value=read.bind("value", before[1]), **scales)
    back = ref.cache_read(b.cache(), *before, b.starts, b.lengths)
    for via in ("device", "host"):
        got = read.run(device, via)
        for name, x in zip(("key", "value"), back):
            assert np.array_equal(got[name], x), (name, via)


@pytest.mark.gpu
def test_gpu_quantised_rows_of_every_kind(device):
    """Zeros, the smallest and largest magnitudes, one element alone, values between two codes, infinities and NaN."""
    b = Batch([(64, 64)], D=64, KVH=1, page=16, quantised=True)
    x = ref.from_bf16(b.key)[:, 0].astype(np.float32)
    x[0] = 0
    x[1] = np.float32(1e-40)
    x[2] = np.float32(3.38e38)
    x[3] = 0
    x[3, 17] = -5
    x[4] = np.arange(64) * 0.5  # the largest is 31.5: 127 / 31.5 is no whole number
    x[5] = np.concatenate([[127.0], np.arange(63) + 0.5])  # ties
    x[6, 3] = np.inf
    x[7, 9] = -np.inf
    x[8, 0] = np.nan
    x[9] = np.float32(2.0 ** -101)
    x[10] = np.float32(2.0 ** -99)
    with np.errstate(invalid="ignore"):
        b.key = ref.to_bf16(x)[:, None]
    b.value = b.key[::-1].copy()
    built = Built()
    k, v = built.bind("key", b.key), built.bind("value", b.value)
    cache, scales = built.cache(b)
    rows = built.rows(b)
    built.program.cache_write(k, v, *cache, *rows, **scales)
    built.program.cache_read(*cache, *rows, key=built.bind("rk", b.key), value=built.bind("rv", b.key), **scales)
    got = built.run(device)
    want = ref.cache_write(b.cache(), b.key, b.value, b.starts, b.lengths)
    for name, w in zip(("key_cache", "value_cache"), want[:2]):
        assert np.array_equal(got[name], w)
    for name, w in zip(("key_scales", "value_scales"), want[2:]):
        assert np.array_equal(got[name], w, equal_nan=True)
    back = ref.from_bf16(got["rk"])[:, 0]
    assert np.isnan(back[6:9]).all() and np.isfinite(np.delete(back, [6, 7, 8], axis=0)).all()
    # a value comes back within half a code and the two roundings of 32 and 16 bits
    fine = np.isfinite(x).all(axis=1)
    unit = np.maximum(np.abs(x[fine]).max(axis=1, keepdims=True).astype(np.float64), 2.0 ** -100) / 127
    far = np.abs(back[fine] - ref.from_bf16(b.key)[fine, 0])
    assert (far <= unit * (0.5 + 127 * 2.0 ** -22) + 2.0 ** -8 * np.abs(back[fine])).all()


# ---- GPU: attention ---------------------------------------------------------------------------------------------------

PROMPTS = [
    dict(sequences=[(1, 1)], D=16, H=1),
    dict(sequences=[(1, 1), (0, 0), (2, 2), (31, 31), (32, 32), (33, 33)], D=64, H=4, tail=3),
    dict(sequences=[(64, 64), (65, 65), (127, 127), (129, 129)], D=128, H=4, KVH=2),
    dict(sequences=[(200, 200)], D=256, H=4, KVH=1),
    dict(sequences=[(17, 17), (90, 90)], D=80, H=6, KVH=2, tail=1),
    dict(sequences=[(70, 70)], D=96, H=3, KVH=3),
    dict(sequences=[(40, 40), (150, 150)], D=192, H=8, KVH=1),
    dict(sequences=[(3, 3)] * 70, D=64, H=8, KVH=8),
    dict(sequences=[(300, 300)], D=64, H=2, KVH=2),
]
SEEN = [dict(), dict(window=1), dict(window=16, sinks=1), dict(window=65, sinks=4), dict(window=33), dict(window=40, sinks=100), dict(window=100000, sinks=3)]


@pytest.mark.gpu
@pytest.mark.parametrize("see", SEEN, ids=_id)
@pytest.mark.parametrize("case", PROMPTS, ids=_id)
def test_gpu_prompts(device, case, see):
    b = Batch(**case)
    built, before, want = attend(b, False, **see)
    check_attention(b, built.run(device)["out"], before, want)


CHUNKS = [
    dict(sequences=[(1, 1)], D=16, H=1, page=1),
    dict(sequences=[(1, 7), (1, 64), (1, 65), (1, 0), (0, 9), (1, 200)], D=64, H=4, page=16, tail=2),
    dict(sequences=[(1, 129), (1, 31)], D=128, H=8, KVH=2, page=7),
    dict(sequences=[(1, 700)], D=256, H=4, KVH=1, page=16),
    dict(sequences=[(1, 33)] * 9, D=80, H=16, KVH=1, page=24),
    dict(sequences=[(2, 50), (4, 4), (3, 100)], D=96, H=5, KVH=5, page=32),
    dict(sequences=[(5, 3), (9, 9), (3, 300)], D=128, H=32, KVH=2, page=64, spare_entries=3),  # the first rows of one stand before its position 0
    dict(sequences=[(64, 200), (1, 90), (40, 41)], D=64, H=4, KVH=2, page=24, tail=4),
    dict(sequences=[(100, 333)], D=256, H=2, KVH=1, page=128),
    dict(sequences=[(33, 150), (1, 260)], D=192, H=4, KVH=2, page=5),
    dict(sequences=[(1, 40)] * 130, D=32, H=2, KVH=1, page=8),
]


@pytest.mark.gpu
@pytest.mark.parametrize("quantised", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("see", [SEEN[0], SEEN[1], SEEN[2], SEEN[3], SEEN[5]], ids=_id)
@pytest.mark.parametrize("case", CHUNKS, ids=_id)
def test_gpu_chunks(device, case, see, quantised):
    b = Batch(quantised=quantised, **case)
    built, before, want = attend(b, True, **see)
    check_attention(b, built.run(device)["out"], before, want)


MIXED = [
    dict(sequences=[(300, 900), (1, 2000), (2, 700), (1, 1), (0, 50), (4, 300), (5, 333), (1, 130)], D=64, H=8, KVH=2, page=24, tail=3),
    dict(sequences=[(1, 1500), (260, 260), (3, 90), (1, 0)], D=80, H=4, KVH=1, page=7),
    dict(sequences=[(40, 5000), (1, 4100), (170, 600)], D=128, H=4, KVH=1, page=64),
    dict(sequences=[(1, 800), (200, 1300), (4, 500), (9, 20)], D=256, H=16, KVH=1, page=16, tail=1),
    dict(sequences=[(1, 400)] * 70 + [(500, 1100)] + [(1, 300)] * 5, D=32, H=16, KVH=1, page=40),
    dict(sequences=[(1, 600)] * 100, D=64, H=2, KVH=1, page=16),
]


@pytest.mark.gpu
@pytest.mark.parametrize("quantised", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("see", [dict(), dict(window=200, sinks=3), dict(window=1000, sinks=70)], ids=_id)
@pytest.mark.parametrize("case", MIXED, ids=_id)
def test_gpu_single_tokens_among_prompts(device, case, see, quantised):
    """Sequences of few rows and of many in one batch, their runs of keys cut into parts; twice, as the second run finds what the first left."""
    b = Batch(quantised=quantised, **case)
    built, before, want = attend(b, True, **see)
    first = built.run(device)["out"]
    check_attention(b, first, before, want)
    assert np.array_equal(built.run(device, dispatches=3)["out"], first)


@pytest.mark.gpu
@pytest.mark.parametrize("keys", ["rows", "bf16", "int8"])
@pytest.mark.parametrize("D", [48, 128, 256])
def test_gpu_many_rows(device, D, keys):
    """So many rows (T times heads) that tiles round the weights once."""
    b = Batch([(700, 1100), (1, 900), (0, 3), (400, 400), (17, 60)], D=D, H=8, KVH=2, page=16, quantised=keys == "int8", tail=2)
    assert b.T * b.H >= 8192
    b.query[::50, 1] = ref.to_bf16(np.float32(np.nan) * np.ones(D, dtype=np.float32))  # rows that are done again
    built, before, want = attend(b, keys != "rows", window=300, sinks=5)
    check_attention(b, built.run(device)["out"], before, want)


@pytest.mark.gpu
@pytest.mark.parametrize("quantised", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_gpu_holes_in_long_tables(device, D, quantised):
    """Entries in the middle of a sequence that are no page, in tiles; two sequences with the same pages."""
    b = Batch([(150, 700), (90, 300), (1, 650), (140, 700)], D=D, H=16, KVH=1, page=16, quantised=quantised)
    b.pages[3] = b.pages[0]
    for s, entries in ((0, (0, 5, 6, 20, 42)), (1, (18,)), (2, (3, 30)), (3, (5, 41))):
        for e in entries:
            b.pages[s, e] = (-1, b.caches[0].shape[0], 2 ** 31 - 1)[e % 3]
    for see in (dict(), dict(window=100, sinks=20)):
        built, before, want = attend(b, True, **see)
        check_attention(b, built.run(device)["out"], before, want)


@pytest.mark.gpu
@pytest.mark.parametrize("quantised", [False, True], ids=["bf16", "int8"])
def test_gpu_tables_that_name_no_page(device, quantised):
    """Entries that are no page, lengths beyond the table or below zero: such positions are not there."""
    b = Batch([(3, 70), (1, 40), (20, 64), (2, 30)], D=64, H=4, KVH=2, page=16, quantised=quantised, tail=1)
    b.pages[0, 1], b.pages[0, 3], b.pages[1, 0], b.pages[2, :] = -1, b.caches[0].shape[0], 2 ** 31 - 1, -5
    b.lengths[1], b.lengths[3] = 10 ** 6, -7
    for see in (dict(), dict(window=20, sinks=2)):
        built, before, want = attend(b, True, **see)
        check_attention(b, built.run(device)["out"], before, want)
    built = Built()
    k, v = built.bind("key", b.key), built.bind("value", b.value)
    cache, scales = built.cache(b)
    rows = built.rows(b)
    built.program.cache_write(k, v, *cache, *rows, **scales)
    got = built.run(device)
    for name, x in zip(("key_cache", "value_cache"), ref.cache_write(b.cache(), b.key, b.value, b.starts, b.lengths)):
        assert np.array_equal(got[name], x)
    built = Built()
    cache, scales = built.cache(b)
    before = b.normal(b.T, b.KVH, b.D), b.normal(b.T, b.KVH, b.D)
    built.program.cache_read(*cache, *built.rows(b), key=built.bind("key", before[0]), value=built.bind("value", before[1]), **scales)
    got = built.run(device)
    for name, x in zip(("key", "value"), ref.cache_read(b.cache(), *before, b.starts, b.lengths)):
        assert np.array_equal(got[name], x)


@pytest.mark.gpu
def test_gpu_starts_that_reach_outside(device):
    """row_starts below zero and beyond the rows are taken as the nearest row."""
    b = Batch([(4, 30), (6, 50), (5, 9)], D=64, H=2, page=16)
    b.starts = np.array([-3, 4, 10, 99], dtype=np.int32)
    built, before, want = attend(b, True)
    check_attention(b, built.run(device)["out"], before, want)
    b.starts = np.array([0, 0, 0, 0], dtype=np.int32)
    built, before, _ = attend(b, True)
    assert np.array_equal(built.run(device)["out"], before)


@pytest.mark.gpu
@pytest.mark.parametrize("sequences", [[(60, 2500), (50, 2000), (40, 2000), (1, 900)], [(1, 2500)] * 5 + [(2, 1500)]], ids=["tiles", "streams"])
def test_gpu_after_starts_that_do_not_ascend(device, sequences):
    """What a dispatch leaves does not touch the next one's results, even where the first one's starts were not ascending."""
    b = Batch(sequences, D=64, H=8, KVH=2, page=16)
    built, before, want = attend(b, True)
    exe = thip.Executable(device, built.program.serialize())
    ptrs = [device.upload(x) for _, x in built.arrays]
    try:
        names = [name for name, _ in built.arrays]
        starts, out = ptrs[names.index("row_starts")], ptrs[names.index("out")]
        odd = np.where(np.arange(len(b.starts)) % 2, b.T, 0).astype(np.int32)
        for x in (odd, b.starts, odd[::-1].copy(), b.starts):
            rt.check(rt.lib().thip_device_h2d(device._h, ctypes.c_void_p(starts), x.ctypes.data_as(ctypes.c_void_p), x.nbytes))
            exe.run_device(ptrs, [a.nbytes for _, a in built.arrays])
        check_attention(b, device.download(out, before.shape, before.dtype), before, want)
    finally:
        for p in ptrs:
            device.free(p)
        exe.close()


@pytest.mark.gpu
@pytest.mark.parametrize("case", [dict(sequences=[(50, 50), (70, 70)], D=64, H=4, KVH=2), dict(sequences=[(130, 130)], D=128, H=2, KVH=1),
                                  dict(sequences=[(90, 90)], D=256, H=4, KVH=1)], ids=_id)
@pytest.mark.parametrize("cached", [False, True], ids=["rows", "cache"])
def test_gpu_infinities_and_nan_in_masked_places(device, case, cached):
    """A key or value that holds NaN or an infinity changes only the rows that see it."""
    b = Batch(**case)
    for bits, p, which in ((0x7FC0, 20, 0), (0x7F80, 31, 1), (0xFF80, 40, 1), (0x7FC0, 47, 1)):
        for s in range(len(b.sequences)):
            if cached:
                b.caches[which][b.pages[s, p // b.page], :, p % b.page, 5::11] = bits
            else:
                (b.key, b.value)[which][b.starts[s] + p, :, 5::11] = bits
    for see in (dict(), dict(window=8), dict(window=5, sinks=2)):
        built, before, want = attend(b, cached, **see)
        result = want[0]
        assert np.isfinite(result[:20]).all() and not np.isfinite(result[47]).all()
        check_attention(b, built.run(device)["out"], before, want, str(see))


@pytest.mark.gpu
def test_gpu_scores_of_every_size(device):
    """Scores from far below to far above what an exponential holds, equal scores, and a key far ahead of the others, late and early."""
    b = Batch([(150, 150)], D=64, H=2, KVH=2)
    k = ref.from_bf16(b.key)
    k[:, 0] *= np.linspace(0.01, 60, 150)[:, None]
    k[:75, 1] = k[0, 1]
    k[100, 1] *= 200
    b.key = ref.to_bf16(k.astype(np.float32))
    built, before, want = attend(b, False)
    check_attention(b, built.run(device)["out"], before, want)


@pytest.mark.gpu
@pytest.mark.parametrize("cached", [False, True], ids=["rows", "cache"])
def test_gpu_result_in_place_of_the_query(device, cached):
    b = Batch([(1, 900), (40, 300), (1, 3)] if cached else [(90, 90), (1, 1)], D=128, H=4, KVH=2, tail=2)
    built = Built()
    q = built.bind("query", b.query)
    if cached:
        cache, scales = built.cache(b)
        built.program.paged_attention(q, *cache, *built.rows(b), scale=b.scale, init=q)
        want = ref.attention(b.query, b.starts, b.scale, cache=b.cache(), lengths=b.lengths)
    else:
        built.program.attention(q, built.bind("key", b.key), built.bind("value", b.value), built.bind("row_starts", b.starts), scale=b.scale, init=q)
        want = ref.attention(b.query, b.starts, b.scale, key=b.key, value=b.value)
    for via in ("device", "host", "noalloc"):
        check_attention(b, built.run(device, via)["query"], b.query, want, via)


# ---- GPU: a run of them -----------------------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("quantised", [False, True], ids=["bf16", "int8"])
def test_gpu_conversation(device, quantised):
    """Prompts of three conversations over rows and into the cache, then steps of one and of two tokens, one program a shape, the lengths going
    up from dispatch to dispatch; at the end all of it is read back."""
    D, H, KVH, page, P, S = 128, 8, 2, 16, 8, 3
    rng = np.random.default_rng(11)
    b = Batch([(P * page, P * page)] * S, D=D, H=H, KVH=KVH, page=page, quantised=quantised)
    bufs = {"key_cache": b.caches[0], "value_cache": b.caches[1], "pages": b.pages}
    if quantised:
        bufs.update(key_scales=b.scales[0], value_scales=b.scales[1])
    on = {name: (device.upload(x), x.nbytes) for name, x in bufs.items()}
    exes, length = {}, np.zeros(S, dtype=np.int64)

    def step(n):
        """n[s] new rows each; returns what attention over the cache gave, having checked it."""
        starts = np.concatenate([[0], np.cumsum(n)]).astype(np.int32)
        T = int(starts[-1])
        length[:] += n
        q, k, v = (ref.to_bf16(rng.standard_normal((T, h, D)).astype(np.float32)) for h in (H, KVH, KVH))
        if T not in exes:
            built = Built()
            vals = [built.bind(name, x) for name, x in (("query", q), ("key", k), ("value", v))]
            cache, scales = built.cache(b)
            rows = built.bind("row_starts", starts), built.bind("lengths", length.astype(np.int32))
            built.program.cache_write(vals[1], vals[2], *cache, *rows, **scales)
            out = built.bind("out", q), built.bind("prompt", q)
            built.program.paged_attention(vals[0], *cache, *rows, scale=b.scale, window=50, sinks=3, init=out[0], **scales)
            built.program.attention(*vals, rows[0], scale=b.scale, init=out[1])
            built.program.cache_read(*cache, *rows, key=built.bind("rk", k), value=built.bind("rv", k), **scales)
            exes[T] = built, thip.Executable(device, built.program.serialize()), {}
        built, exe, mine = exes[T]
        data = dict(query=q, key=k, value=v, row_starts=starts, lengths=length.astype(np.int32), out=np.zeros_like(q), prompt=np.zeros_like(q),
                    rk=np.zeros_like(k), rv=np.zeros_like(k))
        if not mine:
            mine.update({name: (device.alloc(x.nbytes), x.nbytes) for name, x in data.items()})
        for name, x in data.items():
            rt.check(rt.lib().thip_device_h2d(device.handle, ctypes.c_void_p(mine[name][0]), x.ctypes.data_as(ctypes.c_void_p), x.nbytes))
        where = [on.get(name) or mine[name] for name, _ in built.arrays]
        exe.run_device([p for p, _ in where], [size for _, size in where])
        b.caches[0], b.caches[1], *after = ref.cache_write(b.cache(), k, v, starts, length)
        b.scales = after
        got = {name: device.download(mine[name][0], data[name].shape, U16) for name in ("out", "prompt", "rk", "rv")}
        b.starts, b.lengths, b.T = starts, length.astype(np.int32), T
        see = dict(scale=b.scale, window=50, sinks=3)
        check_attention(b, got["out"], data["out"], ref.attention(q, starts, cache=b.cache(), lengths=length, **see))
        check_attention(b, got["prompt"], data["prompt"], ref.attention(q, starts, b.scale, key=k, value=v))
        back = ref.cache_read(b.cache(), data["rk"], data["rv"], starts, length)
        assert np.array_equal(got["rk"], back[0]) and np.array_equal(got["rv"], back[1])

    try:
        step(np.array([40, 7, 65]))
        for _ in range(6):  # the program's four launches are replayed as a graph from the second on
            step(np.array([1, 1, 1]))
        for _ in range(3):
            step(np.array([2, 0, 3]))
    finally:
        for built, exe, mine in exes.values():
            exe.close()
            for p, _ in mine.values():
                device.free(p)
        for p, _ in on.values():
            device.free(p)


@pytest.mark.gpu
def test_gpu_two_at_once_and_again(device):
    """Two executables on streams of their own enqueued in turn, many times: each dispatch gives the same bits."""
    made = []
    for seed, case in ((1, dict(sequences=[(1, 1500), (1, 1300)], D=128, H=8, KVH=2)), (2, dict(sequences=[(1, 2000)], D=256, H=4, KVH=1, quantised=True))):
        b = Batch(seed=seed, **case)
        built, before, want = attend(b, True)
        exe = thip.Executable(device, built.program.serialize())
        made.append((b, built, before, want, exe, [device.upload(a) for _, a in built.arrays], [a.nbytes for _, a in built.arrays]))
    try:
        seen = [None, None]
        for _ in range(10):
            for *_, exe, ptrs, sizes in made:
                for _ in range(3):
                    exe.enqueue_device(ptrs, sizes)
            for i, (b, built, before, want, exe, ptrs, sizes) in enumerate(made):
                exe.wait()
                at = [name for name, _ in built.arrays].index("out")
                got = device.download(ptrs[at], before.shape, U16)
                if seen[i] is None:
                    check_attention(b, got, before, want)
                    seen[i] = got
                assert np.array_equal(got, seen[i])
    finally:
        for *_, exe, ptrs, _ in made:
            exe.close()
            for p in ptrs:
                device.free(p)


@pytest.mark.gpu
@pytest.mark.parametrize("quantised", [False, True], ids=["bf16", "int8"])
def test_gpu_cache_beyond_four_gigabytes(device, quantised):
    """Pages at both ends of a cache of more than 2^32 bytes."""
    D, KVH, page = 256, 1, 128
    elem = 1 if quantised else 2
    NP = (1 << 32) // (page * D * elem) + 5
    b = Batch([(3, 300), (1, 250)], D=D, H=4, KVH=KVH, page=page, quantised=quantised, garbage=False)
    near = b.pages.copy()
    far = np.where(near >= 0, np.where(near % 2 == 0, NP - 1 - near, near), -1).astype(np.int32)
    far[:, -1] = np.where(near[:, -1] < b.caches[0].shape[0], far[:, -1], -1)
    built, before, want = attend(b, True)
    p = thip.Program()
    order = [name for name, _ in built.arrays]
    v = {}
    for i, (name, a) in enumerate(built.arrays):
        shape = (NP,) + a.shape[1:] if "cache" in name or "scales" in name else a.shape
        v[name] = p.binding(i, shape, a.dtype)
    scales = dict(key_scales=v.get("key_scales"), value_scales=v.get("value_scales"))
    cache = v["key_cache"], v["value_cache"], v["pages"]
    p.paged_attention(v["query"], *cache, v["row_starts"], v["lengths"], scale=b.scale, init=v["out"], **scales)
    p.cache_read(*cache, v["row_starts"], v["lengths"], key=p.binding(len(order), b.key.shape, U16), value=p.binding(len(order) + 1, b.key.shape, U16), **scales)
    exe = thip.Executable(device, p.serialize())
    ptrs, sizes = [], []
    try:
        for name, a in built.arrays:
            if "cache" in name or "scales" in name:
                one = a[0].nbytes
                ptr = device.alloc(NP * one)
                for s in range(2):
                    for e in range(near.shape[1]):
                        if 0 <= near[s, e] < a.shape[0]:
                            x = np.ascontiguousarray(a[near[s, e]])
                            rt.check(rt.lib().thip_device_h2d(device.handle, ctypes.c_void_p(ptr + int(far[s, e]) * one), x.ctypes.data_as(ctypes.c_void_p), one))
                ptrs.append(ptr)
                sizes.append(NP * one)
            else:
                ptrs.append(device.upload(far if name == "pages" else a))
                sizes.append(a.nbytes)
        for _ in range(2):
            ptrs.append(device.upload(b.key))
            sizes.append(b.key.nbytes)
        exe.run_device(ptrs, sizes)
        check_attention(b, device.download(ptrs[order.index("out")], before.shape, U16), before, want)
        back = ref.cache_read(b.cache(), b.key, b.key, b.starts, b.lengths)
        for i in range(2):
            assert np.array_equal(device.download(ptrs[len(order) + i], b.key.shape, U16), back[i])
    finally:
        exe.close()
        for ptr in ptrs:
            device.free(ptr)


@pytest.mark.gpu
def test_gpu_logs_and_dumps(device, tmp_path):
    """Under an event log and buffer dumps the ops run record by record, with the same results."""
    b = Batch([(3, 30), (1, 50)], D=64, H=4, KVH=2, quantised=True)
    built, before, want = attend(b, True)
    device.set_event_log(str(tmp_path / "log.csv"))
    device.set_dump_dirs(None, str(tmp_path))
    try:
        got = built.run(device)["out"]
    finally:
        device.set_event_log(None)
        device.set_dump_dirs(None, None)
    check_attention(b, got, before, want)
    dumped = np.load(str(tmp_path / "thip_dispatch" / "action0" / ("bufferbinding%d.npy" % [n for n, _ in built.arrays].index("out"))))
    assert np.array_equal(dumped, got) and "attention" in (tmp_path / "log.csv").read_text()
