"""Attention and its cache (thip_lm_*) where a row's result hangs on what is easily lost: numbers that are none, values next to the largest,
positions at the ends of what 32 bits hold, batches of very unequal sequences, and the programs around the ops."""
import numpy as np
import pytest

from oracle import attention as ref
from test_cache_attention import Batch, attend, check_attention

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
