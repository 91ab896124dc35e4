"""Dispatches that write a part of a binding: the rest of it stays as it is, by host pointers too, where a binding's bytes go to the device and back."""
import numpy as np
import pytest

from oracle import layer as ref
from test_cache_attention import Built
from torq_compiler_amd import runtime as rt

U16, I32, F32, I8 = np.uint16, np.int32, np.float32, np.int8


def _modes(built):
    _, bindings, _ = rt.describe_blob(built.program.serialize())
    return {name: (bool(b["is_read_only"]), bool(b["is_write_only"])) for (name, _), b in zip(built.arrays, bindings)}


def rows(seed, *shape):
    return ref.to_bf16(np.random.default_rng(seed).standard_normal(shape).astype(F32))


def norm_into_a_part():
    built = Built()
    p = built.program
    x, w, out, total = built.bind("x", rows(1, 5, 64)), built.bind("w", rows(2, 64)), built.bind("out", rows(3, 10, 64)), built.bind("sum", rows(4, 700).astype(F32))
    p.norm(x, w, eps=1e-6, init=p.view(out, (5, 64), offset=64), residual_out=p.view(total, (5, 64), offset=300))
    want = ref.norm(built.arrays[0][1], built.arrays[1][1], eps=1e-6, sum_dtype=F32)
    return built, dict(out=(64, want[0]), sum=(300, want[1]))


def rotary_into_a_part():
    built = Built()
    p = built.program
    q, k = built.bind("q", rows(1, 3, 2, 64)), built.bind("k", rows(2, 3, 1, 64))
    qo, ko = built.bind("query_out", rows(3, 9, 2, 64)), built.bind("key_out", rows(4, 800))
    positions, frequencies = np.arange(3, dtype=I32)[None] * 7, np.linspace(0.01, 2, 32, dtype=F32)
    p.rotary(q, k, positions, frequencies, query_out=p.view(qo, (3, 2, 64), offset=256), key_out=p.view(ko, (3, 1, 64), offset=8))
    turned = [ref.rotary(a, positions, frequencies) for a in (built.arrays[0][1], built.arrays[1][1])]
    return built, dict(query_out=(256, turned[0]), key_out=(8, turned[1]))


def bytes_into_a_part():
    built = Built()
    p = built.program
    rng = np.random.default_rng(5)
    a, b = (built.bind(n, rng.integers(-128, 128, 96, dtype=I8)) for n in "ab")
    p.elementwisebinary(2, a, b, init=p.view(built.bind("out", rng.integers(-128, 128, 300, dtype=I8)), (96,), offset=77))
    exact = (built.arrays[0][1] ^ built.arrays[1][1]).astype(np.float64)
    return built, dict(out=(77, (exact, 0 * exact)))


PARTS = [norm_into_a_part, rotary_into_a_part, bytes_into_a_part]


@pytest.mark.parametrize("make", PARTS, ids=lambda m: m.__name__)
def test_a_binding_that_is_written_in_part_is_read_too(make):
    """Or nothing but the part would be on the device, and all of it come back."""
    built, parts = make()
    assert _modes(built) == {name: (name not in parts, False) for name, _ in built.arrays}


def test_a_binding_that_is_written_whole_is_not_read():
    """In one piece, in several that lie side by side or overlap, in whatever order."""
    def modes(pieces, size=320):
        built = Built()
        x, w, out = built.bind("x", rows(1, 1, 64)), built.bind("w", rows(2, 64)), built.bind("out", rows(3, size))
        for at in pieces:
            built.program.norm(x, w, eps=1e-6, init=built.program.view(out, (1, 64), offset=at))
        return _modes(built)["out"]

    assert modes([0], 64) == (False, True)
    assert modes([128, 0, 256, 64, 192]) == (False, True)
    assert modes([0, 64, 100, 164, 200, 256]) == (False, True)
    assert modes([0, 64, 128, 192]) == (False, False)      # the end is missing
    assert modes([64, 128, 192, 256]) == (False, False)    # the beginning
    assert modes([0, 64, 129, 193, 256]) == (False, False)  # an element between


def test_a_binding_of_two_sizes():
    """What is written whole under a smaller shape is a part of what another op names."""
    def modes(first, second):
        built = Built()
        p, x, w = built.program, built.bind("x", rows(1, 1, 64)), built.bind("w", rows(2, 64))
        built.bind("out", rows(3, 2, 64))
        for rows_, at in (first, second):
            p.norm(x, w, eps=1e-6, init=p.view(p.binding(2, (rows_, 64), U16), (1, 64), offset=at))
        return _modes(built)["out"]

    assert modes((1, 0), (2, 64)) == (False, True)
    assert modes((1, 0), (2, 0)) == (False, False)


@pytest.mark.gpu
@pytest.mark.parametrize("via", ["host", "device"])
@pytest.mark.parametrize("make", PARTS, ids=lambda m: m.__name__)
def test_gpu_what_lies_around_a_part_stays(device, make, via):
    built, parts = make()
    for dispatches in (1, 2):
        got = built.run(device, via, dispatches)
        for name, before in built.arrays:
            flat = got[name].reshape(-1)
            if name not in parts:
                assert np.array_equal(got[name], before), name
                continue
            at, (result, bound) = parts[name]
            around = np.ones(flat.size, dtype=bool)
            around[at:at + result.size] = False
            assert np.array_equal(flat[around], before.reshape(-1)[around]), (name, dispatches)
            have = flat[~around].astype(np.float64) if flat.dtype == I8 else ref.wide(flat[~around])
            assert (np.abs(have - result.reshape(-1)) <= bound.reshape(-1)).all(), (name, dispatches)


@pytest.mark.gpu
@pytest.mark.parametrize("N", [129, 2048])
def test_gpu_norm_within_a_host_binding(device, N):
    """Operands in the middle of a binding at odd offsets, by host pointers: what lies around them stays, and NaN there does not come in."""
    rng = np.random.default_rng(6)
    count, around = 5, 3
    whole = rows(7, count * N + 2 * around)
    whole[:around] = whole[-around:] = 0x7FC0
    built = Built()
    p = built.program
    x, out = built.bind("x", whole), built.bind("out", rng.integers(0, 2 ** 16, whole.size).astype(U16))
    w = built.bind("w", rows(8, N))
    p.norm(p.view(x, (count, N), offset=around), w, eps=1e-6, init=p.view(out, (count, N), offset=around))
    got, before = built.run(device, "host")["out"], built.arrays[1][1]
    assert np.array_equal(got[:around], before[:around]) and np.array_equal(got[-around:], before[-around:])
    result, bound = ref.norm(whole[around:-around].reshape(count, N), built.arrays[2][1], eps=1e-6)[0]
    assert (np.abs(ref.wide(got[around:-around]).reshape(count, N) - result) <= bound).all()
