"""Transposes whose result lies in memory as their input does take no record: the result is the input's own bytes.  Where an op writes over either of the
two, they have to be apart: records on the CPU, results on the GPU.  No record writes to a constant."""
import ctypes

import numpy as np
import pytest

import desc_interp
import torq_compiler_amd as thip
from oracle import layer as ref
from test_cache_attention import Built
from torq_compiler_amd import runtime as rt

U16, I32 = np.uint16, np.int32
KIND_TRANSPOSE, KIND_READ, KIND_ROTARY, KIND_NORM = 1, 18, 22, 23
SHAPE, TO, TURNED = (2, 4, 64, 1), (0, 3, 1, 2), (2, 1, 4, 64)  # rows, columns, channels: one channel, so the bytes stay


def rows(seed, *shape):
    return ref.to_bf16(np.random.default_rng(seed).standard_normal(shape).astype(np.float32))


def normed(x, weight):
    """The norm's result and its bound, of rows of 64."""
    return ref.norm(x.reshape(-1, 64), weight, eps=1e-6)[0]


def near(got, want):
    result, bound = want
    return (np.abs(ref.wide(got).reshape(result.shape) - result) <= bound).all()


def over(source, how):
    """A program that turns `source` round and writes over the result; then what was there and what is there now go out.  Named arrays with what each is then."""
    built = Built()
    p = built.program
    x, weight = rows(1, *SHAPE), rows(2, 64)
    w = built.bind("weight", weight)
    if source == "binding":
        src = built.bind("x", x)
    elif source == "part":
        whole = rows(3, 3 * x.size)
        x = whole[x.size:2 * x.size].reshape(SHAPE)
        src = p.view(built.bind("x", whole), SHAPE, offset=x.size)
    elif source == "constant":
        src = p.constant(x)
    else:
        given = rows(4, *SHAPE)
        ones = np.full(1, 0x3F80, U16)
        src = p.norm(built.bind("given", given), p.constant(ones), eps=1.0)  # rows of one element: x / sqrt(x^2 + 1)
        y = ref.wide(given)
        x = y / np.sqrt(y * y + 1)
    t = p.transpose(src, TO, init=p.tensor(TURNED, U16))
    other = rows(5, 8, 64)
    if how == "norm":
        p.norm(t, w, eps=1e-6, init=t)
    elif how == "sum":
        p.norm(p.view(built.bind("other", other), TURNED), None, eps=1e-6, residual=t, residual_out=t)
    elif how == "view":
        p.norm(built.bind("other", other), w, eps=1e-6, init=p.view(t, (8, 64)))
    else:
        p.rotary(p.view(built.bind("other", other), (8, 1, 64)), None, np.zeros((1, 8), I32), np.zeros(32, np.float32), query_out=p.view(t, (8, 1, 64)))
    # what the source holds behind that, and the result
    last = p.norm(src, p.constant(np.full(1, 0x3F80, U16)), eps=1.0, init=built.bind("source", np.zeros(SHAPE, U16)))
    p.norm(p.view(t, (8, 64)), w, eps=1e-6, init=built.bind("out", np.zeros((8, 64), U16)))
    assert last.shape == SHAPE
    return built, x, other, weight


SOURCES, WAYS = ["binding", "part", "constant", "intermediate"], ["norm", "sum", "view", "rotary"]


@pytest.mark.parametrize("how", WAYS)
@pytest.mark.parametrize("source", SOURCES)
def test_a_result_that_is_written_over_has_bytes_of_its_own(source, how):
    built, _, _, _ = over(source, how)
    blob = built.program.serialize()
    d = desc_interp.Descriptor(blob)
    kinds = [int(o["kind"]) for o in d.ops]
    at = kinds.index(KIND_TRANSPOSE)  # it is a record
    write = d.ops[at + 1]
    field = "table" if how == "sum" else "out"
    assert int(write[field]["space"]) == 2 and int(write[field]["index"]) == int(d.ops[at]["out"]["index"])
    assert bytes(d.ops[at]["in0"].tobytes()) != bytes(write[field].tobytes())
    _, bindings, _ = rt.describe_blob(blob)
    modes = {name: bool(b["is_read_only"]) for (name, _), b in zip(built.arrays, bindings)}
    assert modes == {name: name not in ("out", "source") for name in modes}


@pytest.mark.gpu
@pytest.mark.parametrize("how", WAYS)
@pytest.mark.parametrize("source", SOURCES)
def test_gpu_a_result_that_is_written_over(device, source, how):
    """The source is what it was in every dispatch, the constant among them, by host and by device pointers."""
    built, x, other, weight = over(source, how)
    # where the source is computed: its own rounding, then the root's, then that of the result; the derivative of x / sqrt(x^2 + 1) is at most 1
    y = ref.wide(x) if x.dtype == U16 else x
    was = y / np.sqrt(y * y + 1), (np.abs(y) * (2.0 ** -8 if x.dtype != U16 else 0) + 2.0 ** -8 * np.abs(y / np.sqrt(y * y + 1))) * 1.01
    for via, dispatches in (("device", 1), ("device", 3), ("host", 1), ("host", 2)):
        got = built.run(device, via, dispatches)
        assert near(got["source"], was), (via, dispatches)
        for name, a in built.arrays:
            if name not in ("out", "source"):
                assert np.array_equal(got[name], a), name
        if (how, source) != ("sum", "intermediate"):  # a sum may be much smaller than what is known of its parts
            first = dict(norm=lambda: normed(x if x.dtype == U16 else ref.to_bf16(x.astype(np.float32)), weight)[0], view=lambda: normed(other, weight)[0],
                         sum=lambda: y.reshape(8, 64) + ref.wide(other), rotary=lambda: ref.wide(other))[how]()
            # an element that is rounded in between may come out a step (2^-7) apart, which moves it by that and the row's root mean square by as much; one
            # that is computed in front of that too, by three such steps
            result, bound = normed(ref.to_bf16(first.astype(np.float32)), weight)
            steps = 6 if (how, source) == ("norm", "intermediate") else 2
            assert (np.abs(ref.wide(got["out"]) - result) <= bound + steps * 2.0 ** -7 * np.abs(result)).all(), (via, dispatches)
    assert np.array_equal(built.run(device, dispatches=3)["out"], built.run(device)["out"])


def changed(how):
    """The source is written over while the result is still to be read."""
    built = Built()
    p = built.program
    x, weight = rows(1, *SHAPE), rows(2, 64)
    src = built.bind("x", x)
    if how == "intermediate":
        src = p.norm(src, p.constant(np.full(1, 0x3F80, U16)), eps=1.0)
    t = p.transpose(src, TO, init=p.tensor(TURNED, U16))
    p.norm(src, p.constant(np.full(1, 0x4000, U16)), eps=1.0, init=src)  # twice x / sqrt(x^2 + 1)
    p.norm(p.view(t, (8, 64)), built.bind("weight", weight), eps=1e-6, init=built.bind("out", np.zeros((8, 64), U16)))
    return built, x, weight


@pytest.mark.parametrize("how", ["binding", "intermediate"])
def test_a_source_that_is_written_over_leaves_the_result(how):
    kinds = [int(o["kind"]) for o in desc_interp.Descriptor(changed(how)[0].program.serialize()).ops]
    assert kinds == [KIND_NORM] * (how != "binding") + [KIND_TRANSPOSE, KIND_NORM, KIND_NORM]


@pytest.mark.gpu
@pytest.mark.parametrize("how", ["binding", "intermediate"])
def test_gpu_a_source_that_is_written_over(device, how):
    built, x, weight = changed(how)
    got = built.run(device)["out"]
    y = ref.wide(x)
    if how == "binding":
        assert near(got, normed(x, weight))
    else:  # what is normed is known to half a step of each element
        result, bound = normed(ref.to_bf16((y / np.sqrt(y * y + 1)).astype(np.float32)), weight)
        assert (np.abs(ref.wide(got) - result) <= bound + 2 * 2.0 ** -7 * np.abs(result)).all()


def test_a_cache_that_is_written_leaves_what_was_turned_of_it():
    """Keys taken out of a cache in front of a write to it."""
    p = thip.Program()
    cache = p.binding(0, (3, 4, 16, 1), U16)
    t = p.transpose(cache, TO, init=p.tensor((3, 1, 4, 16), U16))
    k = p.view(cache, (3, 4, 1, 16))
    p.cache_write(p.binding(1, (5, 4, 16), U16), p.binding(2, (5, 4, 16), U16), k, p.binding(3, (3, 4, 1, 16), U16), p.binding(4, (1, 3), I32), p.binding(5, (2,), I32),
                  p.binding(6, (1,), I32))
    p.norm(t, p.binding(7, (16,), U16), eps=1e-6, init=p.binding(8, (3, 1, 4, 16), U16))
    assert [int(o["kind"]) for o in desc_interp.Descriptor(p.serialize()).ops] == [KIND_TRANSPOSE, 17, KIND_NORM]


def test_programs_that_write_nothing_over_take_no_record_for_them():
    p = thip.Program()
    t = p.transpose(p.binding(0, SHAPE, U16), TO, init=p.tensor(TURNED, U16))
    y = p.norm(t, p.binding(1, (64,), U16), eps=1e-6)
    back = p.transpose(y, (0, 2, 3, 1), init=p.tensor(SHAPE, U16))
    p.norm(back, p.constant(np.full(1, 0x3F80, U16)), eps=1.0, init=p.binding(2, SHAPE, U16))
    kinds = [int(o["kind"]) for o in desc_interp.Descriptor(p.serialize()).ops]
    assert kinds.count(KIND_NORM) == 2 and kinds[0] == KIND_NORM


def test_records_that_write_to_a_constant_are_refused():
    """What a norm, a rotary turn, an attention or a cache's read writes may not be a constant's bytes, which the next dispatch reads."""
    p = thip.Program()
    q = p.binding(0, (4, 2, 64), U16)
    x = p.binding(1, (1, 512), U16)
    p.norm(x, p.constant(np.zeros(512, U16)), eps=1e-6, residual=x, residual_out=p.binding(2, (1, 512), U16), init=p.binding(3, (1, 512), U16))
    p.rotary(q, p.binding(4, (4, 2, 64), U16), np.zeros((1, 4), I32), np.ones(32, np.float32), query_out=p.binding(5, (4, 2, 64), U16), key_out=p.binding(6, (4, 2, 64), U16))
    p.attention(q, q, q, p.binding(7, (2,), I32), scale=0.125, init=p.binding(8, (4, 2, 64), U16))
    cache, pages, lengths = p.binding(9, (3, 2, 16, 64), U16), p.binding(10, (1, 3), I32), p.binding(11, (1,), I32)
    p.tree_attention(q, cache, cache, pages, p.binding(7, (2,), I32), lengths, p.binding(12, (4,), I32), scale=0.125, init=p.binding(8, (4, 2, 64), U16))
    p.cache_read(cache, cache, pages, p.binding(7, (2,), I32), lengths, key=p.binding(13, (4, 2, 64), U16), value=p.binding(14, (4, 2, 64), U16))
    blob = bytearray(p.serialize())
    d = desc_interp.Descriptor(bytes(blob))

    def status():
        words = (ctypes.c_uint64 * (len(blob) // 8 + 1))()  # 8-byte aligned
        ctypes.memmove(words, bytes(blob), len(blob))
        return rt.lib().thip_descriptor_validate(words, len(blob))

    assert status() == rt.OK
    assert [int(o["kind"]) for o in d.ops] == [KIND_NORM, KIND_ROTARY, 19, 20, KIND_READ]
    constant = d.ops[0]["weights"].tobytes()  # as long as each result
    for op, field in ((0, "out"), (0, "table"), (1, "out"), (1, "weights"), (2, "out"), (3, "out"), (4, "out"), (4, "in1")):
        o = int(d.header["ops_offset"]) + op * d.ops.dtype.itemsize + d.ops.dtype.fields[field][1]
        old = bytes(blob[o:o + 16])
        blob[o:o + 16] = constant
        assert status() == rt.INVALID_ARGUMENT, (op, field)
        blob[o:o + 16] = old
    assert status() == rt.OK
