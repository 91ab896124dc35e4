"""Norms and rotary turns of every way that rows are shared out in: lanes and pieces of a row, rows by several a workgroup, tokens by up to eight."""
import numpy as np
import pytest

import torq_compiler_amd as thip
from oracle import layer as ref
from test_cache_attention import Built
from test_layer_rows import check_norm, check_rotary, make_norm, make_rotary, within

U16, F32 = np.uint16, np.float32

# rows, N and how the launch shares them out: lanes of a row, pieces of each.  Rows of a wave's lanes at most go by several a workgroup from 4096 workgroups on.
SHARES = [
    (70001, 128, 16, 1), (70001, 100, 16, 1),  # 16 rows a workgroup: two turns, the last not full
    (140000, 7, 16, 1),                        # the same of rows that are no whole piece; three turns
    (33001, 256, 32, 1), (33001, 203, 32, 1),  # 8 rows
    (16501, 512, 64, 1), (16501, 299, 64, 1),  # 4 rows
    (2049, 1024, 64, 2), (2049, 1001, 64, 2),
    (2049, 1152, 64, 3), (2049, 1500, 64, 3),
    (16390, 520, 64, 2), (16387, 1030, 64, 3),  # in turns
    (2047, 1024, 128, 1), (2047, 1500, 256, 1),  # fewer rows: a workgroup each
    (600, 4096, 256, 2), (600, 2305, 256, 2),
    (512, 4096, 512, 1), (512, 2305, 512, 1),
    (40, 8192, 512, 2), (40, 8101, 512, 2),
    (40, 16384, 1024, 2), (40, 9001, 1024, 2),
    (40, 32768, 1024, 4), (40, 17001, 1024, 4),
]


def launched(device, a, attributes, sum_dtype):
    """The name of the kernel that a norm of these operands takes."""
    built = Built()
    v = {name: built.bind(name, x) for name, x in a.items()}
    shape = a["input"].shape
    built.program.norm(v["input"], v["weight"], init=built.bind("out", np.zeros(shape, U16)), residual_out=built.bind("sum", np.zeros(shape, sum_dtype)),
                       residual=v.get("residual"), post_weight=v.get("post_weight"), gate=v.get("gate"), **attributes)
    exe = thip.Executable(device, built.program.serialize())
    try:
        return exe.op_kernels()[0]
    finally:
        exe.close()


@pytest.mark.gpu
@pytest.mark.parametrize("wide", [False, True], ids=["bf16", "f32"])
@pytest.mark.parametrize("rows,N,lanes,pieces", SHARES, ids=lambda v: str(v))
def test_gpu_norm_shares(device, rows, N, lanes, pieces, wide):
    """All operands there, in 16 and with a residual of 32 bits; into other buffers and over the operands."""
    a, attributes = make_norm(dict(rows=rows, N=N, residual="f32" if wide else "bf16", gate="element" if rows * N < 1 << 22 else "row", post=True, scale=0.5), seed=rows + N)
    sum_dtype = F32 if wide else U16
    kind = 2 if N < 8 else 1 if N % 8 else 0
    assert launched(device, a, attributes, sum_dtype) == "norm<%d,%d,%d,%d>" % (lanes, pieces, kind, wide)
    check_norm(device, a, attributes, sum_dtype=sum_dtype)
    check_norm(device, a, attributes, sum_dtype=sum_dtype, in_place=True)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,N", [(70001, 128), (2049, 1152), (2049, 1001), (600, 2305)])
def test_gpu_norm_rows_do_not_know_one_another(device, rows, N):
    """Rows that are no number, zeros or far in size among many others, at the ends of workgroups and of turns: every row is what it is alone."""
    a, attributes = make_norm(dict(rows=rows, N=N, post=True), seed=N)
    odd = np.unique(np.concatenate([[0, 1, 15, 16, 17, 255, 256, rows - 2, rows - 1], np.random.default_rng(N).integers(0, rows, 60)]))
    x = ref.wide(a["input"]).astype(F32)
    by = np.array([0.0, np.nan, np.inf, 2.0 ** 100, 2.0 ** -100], F32)[np.arange(len(odd)) % 5]
    with np.errstate(invalid="ignore", over="ignore"):
        x[odd] *= by[:, None]
    a["input"] = ref.to_bf16(x)
    built = Built()
    v = {name: built.bind(name, y) for name, y in a.items()}
    built.program.norm(v["input"], v["weight"], post_weight=v["post_weight"], init=built.bind("out", np.zeros((rows, N), U16)), **attributes)
    got = built.run(device)["out"]
    within(got, ref.norm(a["input"], a["weight"], post_weight=a["post_weight"], **attributes)[0], "rows")


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "neighbours"])
@pytest.mark.parametrize("case", [dict(T=4100, H=2, KVH=1, D=64), dict(T=4099, H=1, D=32, pairs=8, axes=2), dict(T=9001, H=1, KVH=1, D=16), dict(T=5001, H=4, KVH=1, D=256),
                                  dict(T=2051, H=3, KVH=1, D=80, pairs=40, axes=3), dict(T=1537, H=8, KVH=8, D=128), dict(T=3587, H=2, D=256, pairs=128),
                                  dict(T=513, H=1, D=128), dict(T=512, H=1, D=128)],
                         ids=lambda c: "-".join("%s%s" % i for i in c.items()))
def test_gpu_rotary_shares(device, case, interleaved):
    """One to eight tokens a workgroup, the last one's fewer; heads that are turned whole and in part, in place and not."""
    a, frequencies, how = make_rotary(dict(case, interleaved=interleaved, at=(-2 ** 31, 2 ** 31 - 1)), seed=case["T"])
    check_rotary(device, a, frequencies, how)
    check_rotary(device, a, frequencies, how, in_place=True)
