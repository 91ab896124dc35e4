"""What a decoder's layer has around its linears (thip_lm_norm, thip_lm_rotary in include/thip.h) restated in 64 bits, with how far a result may be off."""
import numpy as np

from .attention import from_bf16, to_bf16  # noqa: F401  (re-exported)

H16, H32 = 2.0 ** -8, 2.0 ** -24  # half a step of bf16 and of 32 bits, relative


def wide(x):
    """bf16 bit patterns (uint16) or float32, in 64 bits."""
    x = np.asarray(x)
    return from_bf16(x) if x.dtype == np.uint16 else x.astype(np.float64)


def _half_step(dtype):
    """(relative, absolute) of what is stored."""
    return (H16, 2.0 ** -134) if np.dtype(dtype) == np.uint16 else (H32, 2.0 ** -150)


def norm(x, weight, *, eps, weight_offset=0.0, residual=None, post_weight=None, gate=None, residual_scale=1.0, sum_dtype=np.uint16):
    """((norm, bound), (h, bound)) of rows x [rows, N]; weight None: no norm of the sum.

    Bounds, with h32 and h16 the half steps: a sum of squares is made of at most 100 additions one behind another, so the mean is off by 102 h32 of itself, its
    root's inverse by half of that and two steps more (54 h32), a normed element by four roundings more: 60 h32 of itself.  The sum h is off by dh = 62
    h32 |s g u| + h32 |h|.  In the second norm that moves an element by itself, and all of the row by c times the root mean square of dh (the mean of h dh is at
    most the product of their roots); its own 60 h32, and the rounding of what is stored."""
    f32 = lambda v: float(np.float32(v))  # noqa: E731  (attributes are held in 32 bits)
    eps, offset, scale = f32(eps), f32(weight_offset), f32(residual_scale)

    def factor(v):
        with np.errstate(all="ignore"):
            return 1.0 / np.sqrt(np.mean(v * v, axis=-1, keepdims=True) + eps)

    with np.errstate(all="ignore"):
        u, du = wide(x), 0.0
        if post_weight is not None:
            u = u * factor(u) * (wide(post_weight) + offset)
            du = 60 * H32 * np.abs(u)
        part = u * scale if gate is None else u * wide(gate) * scale
        dpart = (du * np.abs(scale) if gate is None else du * np.abs(wide(gate)) * np.abs(scale)) + 2 * H32 * np.abs(part)
        h = part if residual is None else wide(residual) + part
        dh = dpart + H32 * np.abs(h)
        relative, absolute = _half_step(sum_dtype)
        sums = h, 1.01 * (dh + relative * np.abs(h)) + absolute
        if weight is None:
            return None, sums
        c, w = factor(h), wide(weight) + offset
        y = h * c * w
        bound = np.abs(c * w) * (dh + np.abs(h) * c * np.sqrt(np.mean(dh * dh, axis=-1, keepdims=True))) + 60 * H32 * np.abs(y)
        return (y, 1.01 * (bound + H16 * np.abs(y)) + 2.0 ** -134), sums


def rotary(x, positions, frequencies, axes=None, interleaved=False):
    """(result, bound) of heads x [T, heads, D].

    Sines and cosines are off by less than 5e-7: the angle by 2^-31 of a turn (3e-9) and two roundings of at most 0.8 (9.4e-8), the series by 2.5e-8, the
    arithmetic of 32 bits by four roundings (2.4e-7).  A result of two products is off by that times both elements, three roundings, and its own."""
    x = wide(x)
    f = np.asarray(frequencies, dtype=np.float32).astype(np.longdouble)
    pairs = len(f)
    which = np.zeros(pairs, dtype=int) if axes is None else np.asarray(axes)
    angle = np.asarray(positions, dtype=np.longdouble)[which].T * f  # [T, pairs]
    turn = np.longdouble("6.283185307179586476925286766559")
    angle = (angle - np.floor(angle / turn) * turn).astype(np.float64)[:, None]
    cos, sin = np.cos(angle), np.sin(angle)
    first, second = (np.arange(pairs) * 2, np.arange(pairs) * 2 + 1) if interleaved else (np.arange(pairs), np.arange(pairs) + pairs)
    out, bound = x.copy(), np.zeros(x.shape)
    a, b = x[..., first], x[..., second]
    out[..., first], out[..., second] = a * cos - b * sin, b * cos + a * sin
    off = (5e-7 + 3 * H32) * (np.abs(a) + np.abs(b))
    for where in (first, second):
        bound[..., where] = 1.01 * (off + H16 * np.abs(out[..., where])) + 2.0 ** -134
    return out, bound
