"""Norms of rows whose elements differ by more than squares of 32 bits hold (thip_lm_norm)."""
import numpy as np
import pytest

from oracle import layer as ref
from test_cache_attention import Built
from test_layer_rows import within

U16, F32 = np.uint16, np.float32


@pytest.mark.gpu
@pytest.mark.parametrize("N", [5, 16, 100, 128, 600, 3000, 4096, 20000])
def test_gpu_norm_of_elements_far_apart(device, N):
    """One element is so large that its square passes 32 bits, the others so small that what becomes of them is only just a bf16 of full precision: every one is
    within the bound of its own size."""
    rng = np.random.default_rng(N)
    big = np.array([2.0 ** 60.5, 2.0 ** 61, 2.0 ** 63, 2.0 ** 90, 2.0 ** 118]) * np.sqrt(N)  # about what the root mean square is times the root of N
    x = np.empty((10, N))
    for r, b in enumerate(np.concatenate([big, -big])):
        low, high = np.log2(abs(b)) - np.log2(N) / 2 - 120, np.log2(abs(b)) - 1  # from results of about 2^-120 on
        x[r] = 2.0 ** rng.uniform(low, high, N) * rng.choice([-1, 1], N)
        x[r, r % N] = b
    x = x[:, rng.permutation(N)]
    ones = np.full(N, 0x3F80, U16)
    for wide in (False, True):
        a = dict(input=ref.to_bf16(x.astype(F32)), weight=ones)
        more = {}
        if wide:  # the same by way of a residual of 32 bits
            more = dict(residual=x.astype(F32))
            a["input"] = np.zeros((10, N), U16)
        for post in (False, True) if not wide else (False,):
            built = Built()
            v = {name: built.bind(name, y) for name, y in {**a, **more}.items()}
            built.program.norm(v["input"], v["weight"], residual=v.get("residual"), post_weight=built.bind("post", ones) if post else None, eps=1e-6,
                               init=built.bind("out", np.zeros((10, N), U16)))
            want = ref.norm(a["input"], ones, eps=1e-6, post_weight=ones if post else None, **more)[0]
            assert (np.abs(want[0]) >= 2.0 ** -126).all()
            within(built.run(device)["out"], want, "wide %d post %d" % (wide, post))
