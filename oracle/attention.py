"""The operators around a decoder's cache (thip_lm_* in include/thip.h) restated in 64 bits: NumPy, one row at a time."""
import numpy as np


def from_bf16(bits):
    return (np.asarray(bits, dtype=np.uint16).astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def to_bf16(values):
    """float32 -> bf16 bit patterns, to nearest, ties to even; NaN stays NaN."""
    u = np.ascontiguousarray(values, dtype=np.float32).view(np.uint32)
    rounded = ((u.astype(np.uint64) + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where((u & 0x7FFFFFFF) > 0x7F800000, (u >> 16).astype(np.uint16) | 0x40, rounded).astype(np.uint16)


def places(row_starts, lengths, rows):
    """(row, sequence, position) of every row that is some sequence's; lengths None: a row's number in its sequence."""
    starts = np.clip(np.asarray(row_starts, dtype=np.int64), 0, rows)
    for s in range(len(starts) - 1):
        n = starts[s + 1] - starts[s]
        for i in range(int(n)):
            yield int(starts[s] + i), s, int((0 if lengths is None else max(int(lengths[s]), 0) - n) + i)


class Cache:
    """A paged cache: arrays [pages, kv_heads, page_size, D] (uint16 bf16 bits, or int8 with float32 scales)."""

    def __init__(self, key, value, pages, key_scales=None, value_scales=None):
        self.arrays, self.scales, self.pages = (key, value), (key_scales, value_scales), np.asarray(pages)
        self.quantised = key_scales is not None

    def find(self, seq, position):
        size = self.arrays[0].shape[2]
        if position < 0 or position >= self.pages.shape[1] * size:
            return None
        page = int(self.pages[seq, position // size])
        return (page, position % size) if 0 <= page < self.arrays[0].shape[0] else None

    def row(self, which, seq, position):
        """[kv_heads, D] in 64 bits, None where there is nothing."""
        at = self.find(seq, position)
        if at is None:
            return None
        x = self.arrays[which][at[0], :, at[1]]
        if not self.quantised:
            return from_bf16(x)
        return x.astype(np.float64) * self.scales[which][at[0], :, at[1]].astype(np.float64)[:, None]


def quantise(x):
    """Rows of bf16 values (any shape, the last axis a row) -> int8 values, float32 scales: the definition's own 32-bit steps."""
    x = np.asarray(x, dtype=np.float32)
    finite = np.isfinite(x).all(axis=-1)
    x = np.where(finite[..., None], x, np.float32(0))
    unit = np.maximum(np.abs(x).max(axis=-1), np.float32(2.0 ** -100)).astype(np.float32)
    q = np.rint(x * (np.float32(127) / unit)[..., None]).astype(np.int8)
    return q, np.where(finite, unit / np.float32(127), np.float32(np.nan)).astype(np.float32)


def cache_write(cache, key, value, row_starts, lengths):
    """Writes into copies; returns (key array, value array, key scales, value scales)."""
    out = [[a.copy() for a in cache.arrays], [None if s is None else s.copy() for s in cache.scales]]
    for row, s, position in places(row_starts, lengths, key.shape[0]):
        at = cache.find(s, position)
        if at is None:
            continue
        for which, x in enumerate((key, value)):
            if cache.quantised:
                q, scale = quantise(from_bf16(x[row]))
                out[0][which][at[0], :, at[1]], out[1][which][at[0], :, at[1]] = q, scale
            else:
                out[0][which][at[0], :, at[1]] = x[row]
    return out[0] + out[1]


def cache_read(cache, key, value, row_starts, lengths):
    """Rows read into copies of key and value (bf16 bits)."""
    out = [key.copy(), value.copy()]
    for row, s, position in places(row_starts, lengths, key.shape[0]):
        at = cache.find(s, position)
        for which in range(2):
            if at is None:
                out[which][row] = 0
            elif cache.quantised:
                q, scale = cache.arrays[which][at[0], :, at[1]], cache.scales[which][at[0], :, at[1]]
                with np.errstate(invalid="ignore"):
                    out[which][row] = to_bf16(q.astype(np.float32) * scale[:, None])
            else:
                out[which][row] = cache.arrays[which][at[0], :, at[1]]
    return out


def attention(query, row_starts, scale, window=0, sinks=0, key=None, value=None, cache=None, lengths=None, fine=False, rounded=False):
    """(result, bound) of each row and head [T, heads, D] in 64 bits, NaN in the result of rows that are no sequence's.

    bound: how far a bf16 result may be that is computed as the definition says with sums, scores and statistics in 32 bits and weights
    rounded to bf16 before they meet the values.  With a half step of h16 = 2^-8 (bf16) and h32 = 2^-24: the weights' rounding moves the result by at
    most h16 A, A = sum w |v| / sum w; the result's own by h16 |o|; a score of D products summed in 32 bits, scaled and taken off the maximum, is off by
    at most e = (D + 4) h32 scale sum |q k| + 4 h32 (|s| + |m|), each weight by a factor of 1 + e + 4 h32 (the exponential), numerator and
    denominator by that and n h32 for sums of n: 2 (e + 4 h32 + n h32) A in all; 5 % for their products.
    fine: weights (of int8, times the value's scale: another h32) go in as two bf16, one and what it leaves, which is off by h16 of at most h16: h16^2 A in
    place of h16 A.
    rounded: the result itself is of weights that are rounded to bf16 once, to see that a bound tells the two apart."""
    q = from_bf16(query)
    T, H, D = q.shape
    out, bound = np.full((T, H, D), np.nan), np.zeros((T, H, D))
    h16, h32 = 2.0 ** -8, 2.0 ** -24
    for row, s, position in places(row_starts, lengths, T):
        start = min(max(int(row_starts[s]), 0), T)
        n = min(max(int(row_starts[s + 1]), start), T) - start
        seen = [j for j in range(position + 1) if window == 0 or position - j < window or j < sinks]
        keys, values = [], []
        for j in seen:
            if cache is None:
                if j < n:
                    keys.append(from_bf16(key[start + j]))
                    values.append(from_bf16(value[start + j]))
            elif cache.find(s, j) is not None:
                keys.append(cache.row(0, s, j))
                values.append(cache.row(1, s, j))
        if not keys:
            out[row] = 0
            continue
        keys, values = np.stack(keys, axis=1), np.stack(values, axis=1)  # [kv_heads, positions, D]
        G = H // keys.shape[0]
        for h in range(H):
            k, v = keys[h // G], values[h // G]
            with np.errstate(all="ignore"):
                x = k @ q[row, h] * scale
                m = np.max(x)
                w = np.exp(x - (m if m != -np.inf else 0.0))
                total = w.sum()
                if rounded:
                    w = from_bf16(to_bf16(w.astype(np.float32)))
                out[row, h] = w @ v / total if total != 0 else 0.0
                A = w @ np.abs(v) / total if total != 0 else np.zeros(D)
                off = (D + 4) * h32 * scale * np.max(np.abs(k) @ np.abs(q[row, h])) + 4 * h32 * 2 * np.max(np.abs(x))
                bound[row, h] = 1.05 * (h16 * np.abs(out[row, h]) + A * ((h16 * h16 + h32 if fine else h16) + 2 * (off + 4 * h32 + len(x) * h32))) + 1e-38
    return out, bound
