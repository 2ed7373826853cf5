"""64-bit oracle of the 8-bit operators (test infrastructure): rows in 8 bits,
their products, the append to paged caches and attention over them, from their
formulas, in numpy.

Error bounds are worst cases by counting roundings: u = 2^-24 is half an fp32
step, HALF[type] half a step of an output type relative to the value."""
import numpy as np

from _fourbit import HALF, TINY, U, norm_rotate, rounding  # noqa: F401

F32 = np.float32


def half_away(v):
    """fp32 v (held in any width) to whole numbers, halves away from zero, in the fp32 steps of the operators."""
    v = np.asarray(v, F32)
    return np.trunc(v + np.copysign(F32(0.5), v)).astype(np.int64)


# --------------------------------------------------------------- rows in 8 bits

# The sum of squares: at most 64 fused additions to a thread, 8 more among
# threads, each within u of sums that only grow, and half of that reaches its
# root. The root's reciprocal (2 u after a Newton step, whose argument's
# rounding counts half), its product with the peak, the division and what they
# are compared with take 5 u more.
NORM_SCALE = (72 / 2 + 8) * U


def norm_rows(h, gain, norm, eps):
    """codes, scales (64 bits) of rows h (values of their type, 64 bits)."""
    with np.errstate(all="ignore"):
        u = h.astype(F32) if gain is None else h.astype(F32) * gain.astype(F32)
        peak = np.abs(u).max(1)
        bad = ~np.isfinite(u).all(1)
        up = np.where(peak < F32(2.0 ** -100), F32(2.0 ** 100), F32(1))
        inverse = F32(127) / (peak * up)
        v = (u * up[:, None]) * inverse[:, None]
        v[bad | (peak == 0)] = 0
        codes = half_away(v)
        scale = peak.astype(np.float64) / 127
        if norm:
            scale = scale / np.sqrt((h * h).mean(1) + eps)
    scale[peak == 0] = 0
    scale[bad] = np.nan
    return codes, scale


# --------------------------------------------------------------------- product

def product(codes, a_scales, levels, col_scales, bias, kind):
    """y and the bound of its evaluation: the sum's conversion, its product with
    the row's scale (u each of the product), the fused last step (u of y, and
    where factors are that small a smallest step each), y's rounding."""
    s = (codes.astype(np.float64) @ levels.astype(np.float64)) * a_scales.astype(np.float64)[:, None] * col_scales
    y = s if bias is None else s + bias
    return y, 2.01 * U * np.abs(s) + 1.01 * U * np.abs(y) + 1.01 * rounding(y, kind)


def product_error(got, ref, bound, kind):
    """|got - ref|, 0 where an infinity is the right fp16 value: fp16 rounds what
    lies at 65520 (half a step above its largest, 65504) and beyond to one."""
    with np.errstate(invalid="ignore"):
        beyond = (kind == "f16") & np.isinf(got) & (got * np.sign(ref) > 0) & (np.abs(ref) + bound >= 65520)
        return np.where(beyond, 0.0, np.abs(got - ref))


# ------------------------------------------------------------------------ cache

class Cache:
    """Codes and scales of a paged cache in host arrays."""

    def __init__(self, rng, pages, page, kv_heads, hd, table):
        self.page, self.hd, self.hk, self.pages, self.table = page, hd, kv_heads, pages, np.asarray(table, np.int32)
        self.codes = {n: np.clip(np.rint(rng.randn(pages, kv_heads, page, hd) * 40), -127, 127).astype(np.int8) for n in "kv"}
        self.scales = {n: (np.exp(0.5 * rng.randn(pages, kv_heads)) / 40).astype(F32) for n in "kv"}

    def page_of(self, b, p):
        j = p // self.page
        at = int(self.table[b, j]) if j < self.table.shape[1] else -1
        return at if 0 <= at < self.pages else -1

    def append(self, name, b, first, y):
        """Rows y [n, heads, hd] (fp32) of sequence b from position `first`. Returns
        codes before their rounding at the same places, for comparison near borders."""
        n, j = len(y), 0
        exact = {}
        while j < n:
            off = (first + j) % self.page
            m = min(self.page - off, n - j)
            at = self.page_of(b, first + j)
            if at >= 0:
                for h in range(self.hk):
                    x = y[j:j + m, h].astype(F32)
                    with np.errstate(all="ignore"):
                        old = self.scales[name][at, h] if off else F32(0)
                        fresh = F32(np.abs(x).max()) / F32(127)
                        poisoned = not np.isfinite(x).all() or np.isnan(old)
                        scale = F32(np.nan) if poisoned else max(old, fresh)
                        early = self.codes[name][at, h, :off]
                        was = early.astype(np.float64)
                        if scale > old and off:
                            v = early.astype(F32) * F32(old / scale)
                            was = v.astype(np.float64)
                            self.codes[name][at, h, :off] = half_away(v)
                        v = x * (F32(1) / scale)
                        v = np.zeros_like(x) if poisoned or scale == 0 else np.clip(np.nan_to_num(v, nan=0), F32(-127.4), F32(127.4))
                    self.codes[name][at, h, off:off + m] = half_away(v)
                    self.scales[name][at, h] = scale
                    exact[at, h] = np.concatenate([was, v.astype(np.float64)])
            j += m
        return exact

    def values(self, name, b, lo, hi, h):
        """(values [hi - lo, hd] in 64 bits, which positions have a page)."""
        out, there = np.zeros((hi - lo, self.hd)), np.zeros(hi - lo, bool)
        for p in range(lo, hi):
            at = self.page_of(b, p)
            if at >= 0:
                there[p - lo] = True
                out[p - lo] = self.codes[name][at, h, p % self.page].astype(np.float64) * np.float64(self.scales[name][at, h])
        return out, there


def near_border(scaled):
    """Whether a key's scaled value lies so near a border between two codes that
    its roundings may cross it: the value, the scale, its inverse and the product
    each within u and the evaluation it is compared with the same, |value| <= 127.5."""
    a = np.abs(scaled)
    return np.abs(a - np.floor(a) - 0.5) <= 127.5 * 8 * U


# -------------------------------------------------------------------- attention

def attend(q, k, v, scale, kind):
    """One query over what it sees, and the bound of an evaluation with fp32 sums.
    Scores: an element is held to 2^-22 of itself (two fp16 parts: 11 bits, then the
    rest to 11) or to 2^-30 of the head's largest (counted in steps of which that has
    at least 2^29, rounded to half a step); an MMA of 16-bit parts adds 16 products to
    a running sum, each alignment and the sum within 2 u of the largest in play, in hd
    / 16 steps of up to two parts; four roundings of factors and the difference from
    the maximum, u each of what they round. A weight: the exponential and its parts
    2^-21 in all, or 2^-39 of the largest, for bf16 its one fp16 part 2^-12 of itself.
    Sums: two steps of two parts per tile of 32 tokens and its scale, the same again
    for statistics and joins of parts."""
    q, k, v = (t.astype(np.float64) for t in (q, k, v))
    s = scale * (k @ q)
    e = np.exp(s - s.max())
    p = e / e.sum()
    wide = abs(scale) * (np.abs(k) @ np.abs(q)).max()
    held = 2.0 ** -22 * wide + 2.0 ** -30 * abs(scale) * np.abs(q).max() * np.abs(k).sum(1).max()
    score = (2 * q.size / 16 * 2 + 8) * 2 * U * wide + held
    weight = p @ np.abs(v)
    n = len(s)
    one = 2.0 ** -12 if kind == "bf16" else 0.0
    return p @ v, (2 * score + 2.0 ** -20 + one + (n / 32 * 6 + 128) * 2 * U) * weight + 2.0 ** -39 * n * np.abs(v).max() * p.max()
