"""Norms and rotary positions (thip_lm_norm, thip_lm_rotary): records and refusals on the CPU, results on the GPU against the 64-bit definition (oracle/layer.py,
which derives the bounds that are held)."""
import ctypes
import struct

import numpy as np
import pytest

import desc_interp
import torq_compiler_amd as thip
from oracle import layer as ref
from test_cache_attention import Built, _serialize_error
from torq_compiler_amd import runtime as rt
from torq_compiler_amd.workloads import NO_CLAMP

U16, F32, I32 = np.uint16, np.float32, np.int32
KIND_TRANSPOSE, KIND_EXPAND, KIND_ROTARY, KIND_NORM = 1, 13, 22, 23


def _id(case):
    return "-".join("%s%s" % (k, v) for k, v in case.items()).replace(" ", "")


def bf16(rng, *shape, scale=1.0):
    return ref.to_bf16((rng.standard_normal(shape) * scale).astype(F32))


def within(got, want, what):
    """Every element within its bound, or no number on both sides."""
    result, bound = want
    got = ref.wide(got).reshape(result.shape)
    nan = np.isnan(result)
    assert np.array_equal(np.isnan(got), nan), "%s: no numbers in other places" % what
    with np.errstate(invalid="ignore"):
        over = ~nan & ~(np.abs(got - result) <= bound) & ~(got == result)
    assert not over.any(), "%s: %d off, by up to %g times what is allowed" % (what, over.sum(), np.max((np.abs(got - result) / bound)[over]))


# ---- norms ------------------------------------------------------------------------------------------------------------

def make_norm(case, seed=0):
    """Named arrays of a norm's operands, and its attributes."""
    rng = np.random.default_rng(seed)
    rows, N, gate = case["rows"], case["N"], case.get("gate")
    channels = np.where(rng.random(N) < 0.05, 20.0, 1.0)
    a = dict(input=bf16(rng, rows, N, scale=channels))
    res = case.get("residual")
    if res:
        r = rng.standard_normal((rows, N)) * 4 * channels
        a["residual"] = r.astype(F32) if res == "f32" else ref.to_bf16(r.astype(F32))
    if gate:
        a["gate"] = bf16(rng, *dict(element=(rows, N), row=(rows, 1), channel=(1, N), one=(1, 1))[gate])
    for name in ("weight", "post_weight"):
        w = 1 - case.get("offset", 0.0) + 0.3 * rng.standard_normal(N)
        a[name] = w.astype(F32) if case.get(name) == "f32" else ref.to_bf16(w.astype(F32))
    if not case.get("post"):
        del a["post_weight"]
    attributes = dict(eps=case.get("eps", 1e-6), weight_offset=case.get("offset", 0.0), residual_scale=case.get("scale", 1.0))
    return a, attributes


def check_norm(device, a, attributes, sum_dtype=U16, norms=True, sums=True, in_place=False, via="device", what="", dispatches=1):
    shape = a["input"].shape
    built = Built()
    v = {name: built.bind(name, x) for name, x in a.items()}
    out = v["input"] if in_place else built.bind("out", np.full(shape, 0x1234, U16)) if norms else None
    total = None
    if sums:
        total = v["residual"] if in_place else built.bind("sum", np.full(shape, 77, sum_dtype))
    built.program.norm(v["input"], v.get("weight"), init=out, residual_out=total, residual=v.get("residual"), post_weight=v.get("post_weight"),
                       gate=v.get("gate"), **attributes)
    got = built.run(device, via, dispatches)
    x = {k: y for k, y in a.items() if k not in ("input", "weight")}
    want = ref.norm(a["input"], a.get("weight"), sum_dtype=sum_dtype, **x, **attributes)
    if norms:
        within(got["input" if in_place else "out"], want[0], "norm " + what)
    if sums:
        within(got["residual" if in_place else "sum"], want[1], "sum " + what)
    for name, x in a.items():
        if not in_place or name not in ("input", "residual"):
            assert np.array_equal(got[name].view(np.uint8), x.view(np.uint8)), name + " was written"
    return got


WIDTHS = [1, 2, 7, 8, 9, 64, 100, 127, 128, 129, 255, 256, 257, 500, 512, 520, 1000, 1152, 2041, 2048, 2050, 4096, 4097, 5000, 8192, 8200, 16384, 16385, 30001, 32768]


@pytest.mark.gpu
@pytest.mark.parametrize("N", WIDTHS)
def test_gpu_norm_widths(device, N):
    """Rows of one element to the longest, all operands there: post norm, a gate for each element, a residual."""
    a, attributes = make_norm(dict(rows=5, N=N, residual="bf16", gate="element", post=True, scale=0.5), seed=N)
    check_norm(device, a, attributes)
    a, attributes = make_norm(dict(rows=3, N=N, residual="f32", weight="f32", offset=1.0), seed=N + 1)
    check_norm(device, a, attributes, sum_dtype=F32)


FORMS = [
    dict(rows=1, N=128),
    dict(rows=1001, N=128),
    dict(rows=70, N=96, post=True),
    dict(rows=33, N=200, residual="bf16"),
    dict(rows=17, N=1152, residual="bf16", post=True, offset=1.0),
    dict(rows=19, N=2305, residual="bf16", post=True, gate="row"),
    dict(rows=40, N=777, residual="f32", gate="channel", scale=0.22),
    dict(rows=6, N=4100, residual="f32", gate="one", scale=-2.0, post=True, post_weight="f32"),
    dict(rows=300, N=64, residual="bf16", gate="element", weight="f32"),
    dict(rows=9, N=12, gate="row", scale=3.0),
    dict(rows=1, N=300, residual="bf16", gate="row", scale=0.0),
    dict(rows=700, N=1, residual="bf16", gate="row"),
    dict(rows=5000, N=16, residual="f32", post=True, eps=0.1),
]


@pytest.mark.gpu
@pytest.mark.parametrize("sums", ["bf16", "f32", "none", "only"])
@pytest.mark.parametrize("case", FORMS, ids=_id)
def test_gpu_norm_forms(device, case, sums):
    """Every operand there and not, each type, both results and each alone; by host pointers too."""
    a, attributes = make_norm(case, seed=len(str(case)))
    kind = dict(sum_dtype=F32 if sums == "f32" else U16, norms=sums != "only", sums=sums != "none")
    if sums == "only":
        del a["weight"]
    check_norm(device, a, attributes, **kind)
    check_norm(device, a, attributes, via="host", **kind)


@pytest.mark.gpu
@pytest.mark.parametrize("N", [33, 128, 1152, 5000])
def test_gpu_norm_in_place(device, N):
    """The norm over its input, the sum over its residual; the second dispatch works on what the first left."""
    a, attributes = make_norm(dict(rows=37, N=N, residual="f32", post=True, gate="channel"), seed=3)
    first = check_norm(device, a, attributes, sum_dtype=F32, in_place=True)
    then = dict(a, input=first["input"], residual=first["residual"])
    second = check_norm(device, then, attributes, sum_dtype=F32, in_place=True)
    got = check_twice(device, a, attributes)
    assert np.array_equal(got["input"], second["input"]) and np.array_equal(got["residual"], second["residual"])


def check_twice(device, a, attributes):
    built = Built()
    v = {name: built.bind(name, x) for name, x in a.items()}
    built.program.norm(v["input"], v["weight"], init=v["input"], residual_out=v["residual"], residual=v["residual"], post_weight=v["post_weight"], gate=v["gate"], **attributes)
    return built.run(device, dispatches=2)


@pytest.mark.gpu
@pytest.mark.parametrize("N", [5, 128, 600, 3000, 20000])
def test_gpu_norm_of_odd_rows(device, N):
    """Zeros, values whose squares pass 32 bits on either side, a row that is no number and one with an infinity, next to ordinary ones."""
    rng = np.random.default_rng(N)
    x = rng.standard_normal((12, N)).astype(F32)
    x[1] = 0
    x[2] *= F32(2.0 ** 120)
    x[3] *= F32(2.0 ** -120)
    x[4, 0] = np.nan
    x[5, N - 1] = np.inf
    x[6] = 0
    x[6, N // 2] = F32(3.38e38)
    x[7] = F32(2.0 ** -130)
    x[8] = F32(3.3e38)
    x[9] *= F32(2.0 ** 63)
    x[10] *= F32(2.0 ** -55)
    for eps in (1e-6, 1e-38, 0.0):
        a = dict(input=ref.to_bf16(x), weight=bf16(rng, N))
        check_norm(device, a, dict(eps=eps), sums=False, what="eps %g" % eps)
        a["post_weight"] = bf16(rng, N)
        check_norm(device, a, dict(eps=eps), sums=False, what="twice, eps %g" % eps)


@pytest.mark.gpu
def test_gpu_norm_of_many_rows(device):
    """More rows than a launch's workgroups hold at once, a last workgroup that is not full, ranks other than two."""
    rng = np.random.default_rng(5)
    a = dict(input=bf16(rng, 1237, 3, 64), weight=bf16(rng, 64))
    built = Built()
    v = {name: built.bind(name, x) for name, x in a.items()}
    out = built.program.norm(v["input"], v["weight"], eps=1e-5, init=built.bind("out", np.zeros((1237, 3, 64), U16)))
    assert out.shape == (1237, 3, 64)
    want = ref.norm(a["input"].reshape(-1, 64), a["weight"], eps=1e-5)
    within(built.run(device)["out"], want[0], "many rows")


@pytest.mark.gpu
@pytest.mark.parametrize("N", [129, 2048])
def test_gpu_norm_reads_and_writes_only_its_rows(device, N):
    """Operands in the middle of a binding at odd offsets: what lies around them stays, and NaN there does not come in."""
    rng = np.random.default_rng(6)
    rows, around = 5, 3
    whole = bf16(rng, rows * N + 2 * around)
    whole[:around] = whole[-around:] = 0x7FC0
    built = Built()
    x, out = built.bind("x", whole), built.bind("out", np.full(rows * N + 2 * around, 0x4321, U16))
    w = built.bind("w", np.concatenate([[0x7FC0], bf16(rng, N), [0x7FC0]]).astype(U16))
    p = built.program
    p.norm(p.view(x, (rows, N), offset=around), p.view(w, (N,), offset=1), eps=1e-6, init=p.view(out, (rows, N), offset=around))
    got = built.run(device)["out"]
    assert (got[:around] == 0x4321).all() and (got[-around:] == 0x4321).all()
    within(got[around:-around], ref.norm(whole[around:-around].reshape(rows, N), built.arrays[2][1][1:-1], eps=1e-6)[0], "views")


def test_norm_bound_tells_a_rounded_sum():
    """The bound is narrow enough to see a norm that is made of the sum as it is stored."""
    a, attributes = make_norm(dict(rows=8, N=256, residual="bf16"), seed=1)
    (y, bound), (h, _) = ref.norm(a["input"], a["weight"], residual=a["residual"], **attributes)
    stored, _ = ref.norm(ref.to_bf16(h.astype(F32)), a["weight"], **attributes)[0]
    again = ref.wide(ref.to_bf16(stored.astype(F32)))
    assert (np.abs(again - y) > bound).mean() > 0.01
    assert (np.abs(ref.wide(ref.to_bf16(y.astype(F32))) - y) <= bound).all()


def test_norm_reference_against_differences():
    """The factor is the derivative of the root mean square's logarithm: d/dx_i log(mean(x^2) + eps) = 2 x_i c^2 / N."""
    a, attributes = make_norm(dict(rows=2, N=9), seed=2)
    x = ref.wide(a["input"])
    y, _ = ref.norm(a["input"], np.full(9, 0x3F80, U16), **attributes)[0]
    f = lambda v: np.log(np.mean(v * v, axis=-1) + attributes["eps"])  # noqa: E731
    for i in range(9):
        d = np.zeros(9)
        d[i] = 1e-6
        c = y[:, i] / x[:, i]
        assert np.allclose((f(x + d) - f(x - d)) / 2e-6, 2 * x[:, i] * c * c / 9, rtol=1e-5, atol=1e-7)


def test_norm_record_and_bindings():
    a, attributes = make_norm(dict(rows=4, N=24, residual="f32", gate="row", post=True))
    built = Built()
    v = {name: built.bind(name, x) for name, x in a.items()}
    p = built.program
    y = p.norm(v["input"], v["weight"], residual=v["residual"], residual_out=v["residual"], post_weight=v["post_weight"], gate=v["gate"], **attributes)
    assert y.kind == "tensor" and y.shape == (4, 24)
    p.norm(y, v["weight"], eps=1e-5, init=built.bind("out", a["input"]))
    blob = p.serialize()
    assert [int(o["kind"]) for o in desc_interp.Descriptor(blob).ops] == [KIND_NORM, KIND_NORM]
    _, bindings, _ = rt.describe_blob(blob)
    modes = {name: (bool(x["is_read_only"]), bool(x["is_write_only"])) for (name, _), x in zip(built.arrays, bindings)}
    assert modes == {name: (name not in ("residual", "out"), name == "out") for name in modes}


def _norm_of(p, rows=4, N=24, **other):
    shapes = dict(input=((rows, N), U16), weight=((N,), U16), residual=((rows, N), U16), post_weight=((N,), U16), gate=((rows, N), U16),
                  out=((rows, N), U16), sum=((rows, N), U16))
    shapes.update(other)
    return {name: p.binding(i, *spec) for i, (name, spec) in enumerate(shapes.items())}


def _norm(p, v, **change):
    args = dict(eps=1e-6, residual=v["residual"], post_weight=v["post_weight"], gate=v["gate"], init=v["out"], residual_out=v["sum"])
    args.update(change)
    p.norm(v["input"], args.pop("weight", v["weight"]), **args)


NORM_REFUSED = [
    (dict(input=((4, 24), F32)), rt.INVALID_ARGUMENT, "bf16"),
    (dict(N=32769), rt.UNIMPLEMENTED, "32768"),
    (dict(weight=((25,), U16)), rt.INVALID_ARGUMENT, "weight"),
    (dict(weight=((24,), np.int16)), rt.INVALID_ARGUMENT, "element type"),
    (dict(weight=((1, 24), U16)), rt.INVALID_ARGUMENT, "weight"),
    (dict(post_weight=((12,), U16)), rt.INVALID_ARGUMENT, "post_weight"),
    (dict(residual=((5, 24), U16)), rt.INVALID_ARGUMENT, "residual"),
    (dict(residual=((24, 4), U16)), rt.INVALID_ARGUMENT, "residual"),
    (dict(residual=((4, 24), I32)), rt.INVALID_ARGUMENT, "element type"),
    (dict(gate=((4, 24), F32)), rt.INVALID_ARGUMENT, "gate"),
    (dict(gate=((2, 24), U16)), rt.INVALID_ARGUMENT, "gate"),
    (dict(gate=((24,), U16)), rt.INVALID_ARGUMENT, "gate"),
    (dict(out=((4, 25), U16)), rt.INVALID_ARGUMENT, "init"),
    (dict(out=((4, 24), F32)), rt.INVALID_ARGUMENT, "init"),
    (dict(sum=((4, 24), I32)), rt.INVALID_ARGUMENT, "residual_out"),
    (dict(sum=((8, 24), U16)), rt.INVALID_ARGUMENT, "init holds"),
    (dict(rows=1 << 31, N=8), rt.UNIMPLEMENTED, "2^31"),
]


@pytest.mark.parametrize("shapes,code,text", NORM_REFUSED, ids=[t[2] + str(i) for i, t in enumerate(NORM_REFUSED)])
def test_norm_refused_shapes(shapes, code, text):
    got, message = _serialize_error(lambda p: _norm(p, _norm_of(p, **shapes)))
    assert got == code and text in message, (got, message)


def test_norm_refused_calls():
    for attribute in (dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")), dict(weight_offset=float("nan")), dict(residual_scale=float("inf"))):
        assert _serialize_error(lambda p: _norm(p, _norm_of(p), **attribute))[0] == rt.INVALID_ARGUMENT, attribute
    # neither result, one of init and its weight
    assert _serialize_error(lambda p: _norm(p, _norm_of(p), weight=None, init=None, residual_out=None))[0] == rt.INVALID_ARGUMENT
    assert _serialize_error(lambda p: _norm(p, _norm_of(p), weight=None))[0] == rt.INVALID_ARGUMENT

    def shares(make):
        def call(p):
            v = _norm_of(p, input=((5, 24), U16))
            v["input"] = p.view(v["input"], (4, 24))
            make(p, v)
        got, message = _serialize_error(call)
        assert got == rt.INVALID_ARGUMENT and "share bytes" in message, message

    shares(lambda p, v: _norm(p, v, init=v["sum"]))
    shares(lambda p, v: _norm(p, v, init=v["residual"]))
    shares(lambda p, v: _norm(p, v, residual_out=v["input"]))
    shares(lambda p, v: _norm(p, v, init=p.view(p.binding(0, (5, 24), U16), (4, 24), offset=8)))
    shares(lambda p, v: _norm(p, v, residual_out=v["gate"]))
    shares(lambda p, v: _norm(p, v, init=p.view(p.binding(1, (200,), U16), (4, 24))))

    def other_type(p):  # a residual of 32 bits may not become one of 16 in place
        v = _norm_of(p, residual=((4, 24), F32))
        _norm(p, v, residual_out=p.view(p.binding(2, (8, 24), U16), (4, 24)))

    assert _serialize_error(other_type)[0] == rt.INVALID_ARGUMENT

    def constant(p):
        v = _norm_of(p)
        _norm(p, v, init=p.constant(np.zeros((4, 24), U16)))

    assert _serialize_error(constant)[0] == rt.INVALID_ARGUMENT

    def undefined(p):
        v = _norm_of(p)
        v["input"] = p.tensor((4, 24), U16)
        _norm(p, v)

    assert _serialize_error(undefined)[0] == rt.FAILED_PRECONDITION
    assert rt.lib().thip_lm_norm(None, None) == rt.INVALID_ARGUMENT


def _written_over(by, what):
    """A product of x [4, 64] and what an op in front of it made (a transpose, expanded weights), written over by a norm or a rotary turn.  The program and its operands."""
    rng = np.random.default_rng(9)
    built = Built()
    x, other = bf16(rng, 4, 64), bf16(rng, 64, 48)
    p = built.program
    made = p.tensor((64, 48), U16)
    if what == "transpose":
        p.transpose(built.bind("source", bf16(rng, 48, 64)), (1, 0), init=made)
    else:
        scale, bias = bf16(rng, 2, 48), np.zeros((2, 48), F32)
        p.expand_weights(rng.integers(-128, 128, (64, 48)).astype(np.int8), scale, bias, block_size=32, output_min=NO_CLAMP[0], output_max=NO_CLAMP[1], init=made)
    v = built.bind("other", other)
    if by == "norm":
        weight = ref.to_bf16(np.ones(48, F32))
        p.norm(v, built.bind("weight", weight), eps=1e-6, init=made)
        held = ref.to_bf16(ref.norm(other, weight, eps=1e-6, weight_offset=0.0)[0][0].astype(F32))
    elif by == "sum":
        p.norm(v, None, eps=1e-6, residual_out=made)
        held = other
    out = built.bind("out", np.zeros((4, 48), U16))
    p.matmul(built.bind("x", x), made, np.array([0.0], F32), init=out, output_zp=0, output_min=NO_CLAMP[0], output_max=NO_CLAMP[1], shift=0)
    return built, x, held


@pytest.mark.parametrize("by", ["norm", "sum"])
@pytest.mark.parametrize("what", ["transpose", "expand"])
def test_norm_over_what_a_product_would_have_folded(by, what):
    """The op whose result is written over stays a record of its own: a product that took it into itself would read what was there before."""
    built, _, _ = _written_over(by, what)
    kinds = [int(o["kind"]) for o in desc_interp.Descriptor(built.program.serialize()).ops]
    assert kinds[:2] == [dict(transpose=KIND_TRANSPOSE, expand=KIND_EXPAND)[what], KIND_NORM], kinds


def test_rotary_over_what_a_product_would_have_folded():
    p = thip.Program()
    made = p.transpose(p.binding(0, (3, 48, 64), U16), (0, 2, 1))
    p.rotary(p.binding(1, (3, 64, 48), U16), None, p.binding(2, (1, 3), I32), np.ones(8, F32), query_out=made)
    p.matmul(p.binding(3, (3, 4, 64), U16), made, np.array([0.0], F32), init=p.binding(4, (3, 4, 48), U16), output_zp=0, output_min=NO_CLAMP[0],
             output_max=NO_CLAMP[1], shift=0)
    kinds = [int(o["kind"]) for o in desc_interp.Descriptor(p.serialize()).ops]
    assert kinds[:2] == [KIND_TRANSPOSE, KIND_ROTARY], kinds


@pytest.mark.gpu
@pytest.mark.parametrize("by", ["norm", "sum"])
@pytest.mark.parametrize("what", ["transpose", "expand"])
def test_gpu_norm_over_what_a_product_would_have_folded(device, by, what):
    built, x, held = _written_over(by, what)
    got = ref.wide(built.run(device, "device")["out"])
    # of each operand of the sum half a step of bf16 (the norm's), of the result another, of 64 products the sum's roundings in 32 bits
    a, b = ref.wide(x), ref.wide(held)
    want, size = a @ b, np.abs(a) @ np.abs(b)
    bound = size * (2.0 ** -8 * (2 if by == "norm" else 0) + 64 * 2.0 ** -24) + np.abs(want) * 2.0 ** -8
    assert (np.abs(got - want) <= bound * 1.01).all()


# ---- rotary positions ---------------------------------------------------------------------------------------------------

def make_rotary(case, seed=0):
    rng = np.random.default_rng(seed)
    T, D, axes = case["T"], case["D"], case.get("axes", 1)
    a = dict(query=bf16(rng, T, case["H"], D))
    if case.get("KVH"):
        a["key"] = bf16(rng, T, case["KVH"], D)
    low, high = case.get("at", (0, 5000))
    a["positions"] = rng.integers(low, high + 1, size=(axes, T)).astype(I32)
    pairs = case.get("pairs", D // 2)
    frequencies = (10000.0 ** (-np.arange(pairs) / pairs)).astype(F32)
    which = (np.arange(pairs) * axes // pairs).astype(I32) if axes > 1 else None
    return a, frequencies, dict(axes=which, interleaved=case.get("interleaved", False))


def check_rotary(device, a, frequencies, how, in_place=False, via="device", constant=False):
    built = Built()
    v = {name: built.bind(name, x) for name, x in a.items() if name != "positions" or not constant}
    names = [n for n in ("query", "key") if n in a]
    outs = {n: v[n] if in_place else built.bind(n + "_out", np.full(a[n].shape, 0x1234, U16)) for n in names}
    built.program.rotary(v["query"], v.get("key"), a["positions"] if constant else v["positions"], frequencies, query_out=outs["query"], key_out=outs.get("key"), **how)
    got = built.run(device, via)
    for n in names:
        within(got[n if in_place else n + "_out"], ref.rotary(a[n], a["positions"], frequencies, how["axes"], how["interleaved"]), n)
        if not in_place:
            assert np.array_equal(got[n], a[n]), n + " was written"


TURNED = [
    dict(T=1, H=1, D=16),
    dict(T=1, H=4, KVH=1, D=256),
    dict(T=16, H=4, KVH=1, D=256, at=(0, 2 ** 31 - 1)),
    dict(T=33, H=6, KVH=2, D=80, pairs=16, axes=2, at=(-2 ** 31, 2 ** 31 - 1)),
    dict(T=130, H=8, KVH=8, D=96, axes=3),
    dict(T=1001, H=5, KVH=5, D=64, pairs=8),
    dict(T=7, H=128, KVH=16, D=128, axes=3, at=(10 ** 6, 10 ** 6 + 5000)),
    dict(T=50, H=3, D=208, pairs=104, axes=4),
    dict(T=300, H=2, KVH=1, D=48, pairs=24),
    dict(T=3, H=700, KVH=100, D=16),
]


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "neighbours"])
@pytest.mark.parametrize("case", TURNED, ids=_id)
def test_gpu_rotary(device, case, interleaved):
    """Tokens and heads from one on, a part of a head, several axes, the farthest positions on both sides; in place, by host pointers, positions that are constants."""
    a, frequencies, how = make_rotary(dict(case, interleaved=interleaved), seed=case["T"])
    check_rotary(device, a, frequencies, how)
    check_rotary(device, a, frequencies, how, in_place=True)
    check_rotary(device, a, frequencies, how, via="host")
    check_rotary(device, a, frequencies, how, constant=True)


@pytest.mark.gpu
def test_gpu_rotary_steps_of_every_kind(device):
    """Frequencies of 0, next to none, negative, of several turns, halves and quarters of a turn, positions 0 and next to the ends."""
    rng = np.random.default_rng(1)
    frequencies = np.array([0, 1e-30, -1, 1, 16, -16, np.pi, -np.pi / 2, 6.2831855, 0.5, 1e-4, 3, 7, -2.5, 2.0 ** -20, 12.566371], dtype=F32)
    positions = np.array([[0, 1, -1, 2, 3, 5, 2 ** 31 - 1, -2 ** 31, 12345678, -7654321, 2 ** 30, 4]], dtype=I32)
    a = dict(query=bf16(rng, positions.shape[1], 2, 32), positions=positions)
    for interleaved in (False, True):
        check_rotary(device, a, frequencies, dict(axes=None, interleaved=interleaved))


@pytest.mark.gpu
def test_gpu_rotary_of_numbers_that_are_none(device):
    """An infinity or NaN reaches its own pair only; what is behind the pairs passes as it is, bit for bit."""
    rng = np.random.default_rng(2)
    x = bf16(rng, 5, 2, 64)
    x[1, 0, 3], x[2, 1, 20], x[3, 0, 40] = 0x7FC0, 0x7F80, 0x7F81  # of a pair, of another, behind them
    a = dict(query=x, positions=np.arange(5, dtype=I32)[None])
    frequencies = (100.0 ** (-np.arange(16) / 16)).astype(F32)
    built = Built()
    q, pos, out = built.bind("query", x), built.bind("positions", a["positions"]), built.bind("out", np.zeros_like(x))
    built.program.rotary(q, None, pos, frequencies, query_out=out)
    got = built.run(device)["out"]
    assert np.array_equal(got[..., 32:], x[..., 32:])
    bad = np.zeros(x.shape, dtype=bool)
    bad[1, 0, [3, 19]] = bad[2, 1, [20, 4]] = True
    real = ref.wide(got)
    assert np.isnan(real[1, 0, [3, 19]]).all() and not np.isfinite(real[2, 1, [20, 4]]).all()
    clean = x.copy()
    clean[bad] = 0
    want = ref.rotary(clean, a["positions"], frequencies)
    keep = ~bad
    keep[..., 32:] = False
    keep[1, 0, [3, 19]] = keep[2, 1, [20, 4]] = False
    assert (np.abs(real - want[0])[keep] <= want[1][keep]).all()


def test_rotary_reference():
    """The reference keeps the length of a pair, turns back by the negative position, and its derivative by the position is the pair a quarter turn on."""
    a, frequencies, how = make_rotary(dict(T=9, H=2, D=32, axes=2), seed=4)
    y, _ = ref.rotary(a["query"], a["positions"], frequencies, **how)
    x = ref.wide(a["query"])
    assert np.allclose(y[..., :16] ** 2 + y[..., 16:] ** 2, x[..., :16] ** 2 + x[..., 16:] ** 2)
    quarter = np.concatenate([-x[..., 16:], x[..., :16]], axis=-1)
    z, _ = ref.rotary(a["query"], np.zeros_like(a["positions"]), frequencies, **how)
    assert np.array_equal(z, x)
    step = (frequencies * 1e-4).astype(F32)  # small angles: the position's derivative at 0
    up, _ = ref.rotary(a["query"], np.ones_like(a["positions"]), step, **how)
    down, _ = ref.rotary(a["query"], -np.ones_like(a["positions"]), step, **how)
    assert np.allclose((up - down) / 2, quarter * np.tile(step.astype(np.float64), 2), rtol=1e-6, atol=1e-12)


def _rotary_of(p, T=4, H=2, KVH=1, D=64, axes=1, **other):
    shapes = dict(query=((T, H, D), U16), key=((T, KVH, D), U16), positions=((axes, T), I32), query_out=((T, H, D), U16), key_out=((T, KVH, D), U16))
    shapes.update(other)
    return {name: p.binding(i, *spec) for i, (name, spec) in enumerate(shapes.items())}


def _rotary(p, v, frequencies=None, **how):
    p.rotary(v["query"], v["key"], v["positions"], np.ones(32, F32) if frequencies is None else frequencies, query_out=v["query_out"], key_out=v["key_out"], **how)


ROTARY_REFUSED = [
    (dict(query=((4, 128), U16)), {}, rt.INVALID_ARGUMENT, "rank"),
    (dict(query=((4, 2, 64), np.int16)), {}, rt.INVALID_ARGUMENT, "bf16"),
    (dict(D=72), {}, rt.UNIMPLEMENTED, "multiples of 16"),
    (dict(D=272), {}, rt.UNIMPLEMENTED, "multiples of 16"),
    (dict(key=((5, 1, 64), U16)), {}, rt.INVALID_ARGUMENT, "key"),
    (dict(key=((4, 1, 32), U16)), {}, rt.INVALID_ARGUMENT, "key"),
    (dict(query_out=((4, 3, 64), U16)), {}, rt.INVALID_ARGUMENT, "query_out"),
    (dict(key_out=((4, 64), U16)), {}, rt.INVALID_ARGUMENT, "key_out"),
    (dict(positions=((1, 5), I32)), {}, rt.INVALID_ARGUMENT, "positions"),
    (dict(positions=((4,), I32)), {}, rt.INVALID_ARGUMENT, "rank"),
    (dict(positions=((1, 4), F32)), {}, rt.INVALID_ARGUMENT, "element type"),
    ({}, dict(frequencies=np.ones(12, F32)), rt.INVALID_ARGUMENT, "multiple of 8"),
    ({}, dict(frequencies=np.ones(40, F32)), rt.INVALID_ARGUMENT, "half"),
    ({}, dict(frequencies=np.full(32, np.nan, F32)), rt.INVALID_ARGUMENT, "frequencies[0]"),
    ({}, dict(frequencies=np.full(32, 16.5, F32)), rt.INVALID_ARGUMENT, "at most 16"),
    ({}, dict(axes=np.zeros(31, I32)), rt.INVALID_ARGUMENT, "axes"),
    ({}, dict(axes=np.full(32, 1, I32)), rt.INVALID_ARGUMENT, "axes[0] is 1"),
    ({}, dict(axes=np.full(32, -1, I32)), rt.INVALID_ARGUMENT, "axes[0]"),
    (dict(query=((4, 1 << 21, 64), U16), query_out=((4, 1 << 21, 64), U16)), {}, rt.UNIMPLEMENTED, "heads"),
    (dict(T=1 << 31), {}, rt.UNIMPLEMENTED, "2^31"),
    (dict(T=1 << 27, H=1), {}, rt.UNIMPLEMENTED, "2^27"),
]


@pytest.mark.parametrize("shapes,how,code,text", ROTARY_REFUSED, ids=[t[3] + str(i) for i, t in enumerate(ROTARY_REFUSED)])
def test_rotary_refused(shapes, how, code, text):
    got, message = _serialize_error(lambda p: _rotary(p, _rotary_of(p, **shapes), **how))
    assert got == code and text in message, (got, message)


def test_rotary_refused_operands():
    def frequencies_at_run_time(p):
        v = _rotary_of(p)
        _rotary(p, v, p.binding(5, (32,), F32))

    def computed_positions(p):
        v = _rotary_of(p)
        v["positions"] = p.tensor((1, 4), I32)
        _rotary(p, v)

    def crossed(p):
        v = _rotary_of(p, key=((4, 2, 64), U16), key_out=((4, 2, 64), U16))
        v["query_out"], v["key_out"] = v["key"], v["query"]
        _rotary(p, v)

    def shifted(p):
        v = _rotary_of(p, query=((5, 2, 64), U16))
        v["query_out"], v["query"] = p.view(v["query"], (4, 2, 64), offset=128), p.view(v["query"], (4, 2, 64))
        _rotary(p, v)

    def odd(p):
        v = _rotary_of(p, query=((5, 2, 64), U16))
        v["query"] = p.view(v["query"], (4, 2, 64), offset=4)
        _rotary(p, v)

    def key_alone(p):
        v = _rotary_of(p)
        freq = p.constant(np.ones(32, F32))
        op = rt.LmRotary(v["query_out"].index, -1, v["query"].index, v["key"].index, v["positions"].index, freq.index, -1, 0)
        rt.check(rt.lib().thip_lm_rotary(p._h, ctypes.byref(op)))

    for make, code in ((frequencies_at_run_time, rt.UNIMPLEMENTED), (computed_positions, rt.INVALID_ARGUMENT), (crossed, rt.INVALID_ARGUMENT),
                       (shifted, rt.INVALID_ARGUMENT), (odd, rt.UNIMPLEMENTED), (key_alone, rt.INVALID_ARGUMENT)):
        assert _serialize_error(make)[0] == code, make.__name__
    assert rt.lib().thip_lm_rotary(None, None) == rt.INVALID_ARGUMENT


# ---- records ------------------------------------------------------------------------------------------------------------

def test_changed_records_are_refused_or_stay_inside():
    """Every 32-bit word of the records and of the steps set to other values: a status each time; every extent that a record names, larger, is refused."""
    p = thip.Program()
    v = _norm_of(p)
    _norm(p, v)
    q, k = p.binding(7, (4, 2, 64), U16), p.binding(8, (4, 1, 64), U16)
    p.rotary(q, k, p.binding(9, (2, 4), I32), np.ones(32, F32), axes=np.arange(32) % 2, query_out=q, key_out=k)
    blob = bytearray(p.serialize())
    d = desc_interp.Descriptor(bytes(blob))
    size = d.ops.dtype.itemsize

    def status(b):
        words = (ctypes.c_uint64 * (len(b) // 8 + 1))()  # 8-byte aligned
        ctypes.memmove(words, bytes(b), len(b))
        return rt.lib().thip_descriptor_validate(words, len(b))

    assert status(blob) == rt.OK
    at = bytes(blob).index(d.ops[0].tobytes())
    for op, fields in ((0, ("M", "C", "KH", "KW", "SH", "SW", "TR", "TS")), (1, ("M", "N", "H", "W", "C", "K"))):
        for word in range(size // 4):
            o = at + op * size + 4 * word
            old = bytes(blob[o:o + 4])
            for value in (0, 1, 3, 0x7FFFFFFF, 0x80000000, 0xFFFFFFFF, struct.unpack("<I", old)[0] + 1):
                blob[o:o + 4] = struct.pack("<I", value & 0xFFFFFFFF)
                assert status(blob) in (rt.OK, rt.INVALID_ARGUMENT)
            blob[o:o + 4] = old
        for field in fields:
            o = at + op * size + d.ops.dtype.fields[field][1]
            old = bytes(blob[o:o + 4])
            blob[o:o + 4] = struct.pack("<i", 2 * int(d.ops[op][field]) + 1)
            assert status(blob) == rt.INVALID_ARGUMENT, field
            blob[o:o + 4] = old
    table = int(d.header["data_offset"]) + int(d.consts[int(d.ops[1]["table"]["index"])]["offset"])
    for pair in (0, 31):
        for value in (2, -1, 2 ** 31 - 1):
            o = table + 16 * pair + 8
            old = bytes(blob[o:o + 4])
            blob[o:o + 4] = struct.pack("<i", value)
            assert status(blob) == rt.INVALID_ARGUMENT
            blob[o:o + 4] = old
    assert status(blob) == rt.OK


@pytest.mark.gpu
@pytest.mark.parametrize("N", [1544, 1601])
def test_gpu_norm_of_rows_for_a_wider_grid(device, N):
    """So many rows of more than a wave that the grid has two dimensions: the same bits for the same row wherever it lies, rows far apart in size next to others."""
    rng = np.random.default_rng(N)
    rows = 65536 + 65536 // 2 + 1
    some = bf16(rng, 1024, N)
    x = np.tile(some, (rows // 1024 + 1, 1))[:rows]
    odd = np.array([5, 65536 + 5, 65536 + 6, 70000])
    x[odd] = ref.to_bf16((ref.from_bf16(x[odd]) * np.array([2.0 ** 70, 2.0 ** -70, 2.0 ** 80, 0.0])[:, None]).astype(F32))
    a = dict(input=x, weight=bf16(rng, N), post_weight=bf16(rng, N))
    built = Built()
    v = {name: built.bind(name, y) for name, y in a.items()}
    built.program.norm(v["input"], v["weight"], post_weight=v["post_weight"], eps=1e-6, init=built.bind("out", np.zeros((rows, N), U16)))
    got = built.run(device)["out"]
    look = np.unique(np.concatenate([odd, odd - 1, odd + 1, [0, 65535, 65536, rows - 2, rows - 1], rng.integers(0, rows, 300)]))
    within(got[look], ref.norm(x[look], a["weight"], eps=1e-6, post_weight=a["post_weight"])[0], "some rows")
    plain = np.ones(rows, dtype=bool)
    plain[odd] = False
    first = got[1024:2048]  # the same rows again and again: the same bits
    for r in range(0, rows - 1024, 1024):
        same = plain[r:r + 1024]
        assert np.array_equal(got[r:r + 1024][same], first[same]), r
