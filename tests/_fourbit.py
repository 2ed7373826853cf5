"""64-bit oracle of the 4-bit operators (test infrastructure): the group-scaled
product, the norm + rotation + 4-bit append, and attention over the ring, from
their formulas, in numpy.

Error bounds are worst cases by counting roundings: u = 2^-24 is half an fp32
step, HALF[type] half a step of an output type relative to the value."""
import numpy as np

U = 2.0 ** -24
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f32": 2.0 ** -149, "f16": 2.0 ** -24, "bf16": 2.0 ** -133}   # a step among the smallest values
GROUP = 64


def rounding(y, kind):
    return np.abs(y) * HALF[kind] + TINY[kind]


def unpack(packed, count):
    c = np.empty(2 * packed.size, np.int64)
    c[0::2], c[1::2] = packed.reshape(-1) & 15, packed.reshape(-1) >> 4
    return c[:count]


# ------------------------------------------------------------------ product

def dequant(scales, packed, rows, cols, group):
    level = unpack(packed, rows * cols).reshape(rows, cols) - 7
    return level * scales.astype(np.float64).repeat(group, 0)[:rows]


HELD = {"f32": 2.0 ** -22, "f16": 1 / 32639, "bf16": 1 / 32639}


def product(x, w, kind="f32"):
    """y and its bound. fp32 activations are held to 2^-22 of the largest of
    their 128 consecutive ones, 16-bit ones to 1 / 32639: each is rounded to an
    integer after a power of two that puts the largest in [2^22, 2^23) or
    [2^14, 2^15), halved where that is above 8355711 or 32639 (the top digit
    would not fit). The largest is then at least 4177855 or 16319.5, and half
    a step is 1/2. Each of the K / 32 + 64 additions
    rounds once, and so does the scale of a sum."""
    x = x.astype(np.float64)
    m, k = x.shape
    pad = -k % 128
    top = np.abs(np.pad(x, ((0, 0), (0, pad)))).reshape(m, -1, 128).max(-1)
    a = np.abs(w)
    block = np.pad(a, ((0, pad), (0, 0))).reshape(-1, 128, w.shape[1]).sum(1)
    bound = HELD[kind] * (top @ block) + (k / 32 + 64) * U * (np.abs(x) @ a)
    return x @ w, bound


# ------------------------------------------------------------------- append

def quantize_rows(x):
    """(codes, scales, scaled) of fp32 rows [..., head_dim] in groups of 64: the
    framework's quantizer; `scaled` is x * 7 / peak in 64 bits."""
    x = x.astype(np.float32).reshape(*x.shape[:-1], -1, GROUP)
    with np.errstate(all="ignore"):
        peak = np.abs(x).max(-1, keepdims=True)
        v = x * (np.float32(7) / peak)
        level = np.where(v >= 0, np.floor(v + np.float32(0.5)), np.ceil(v - np.float32(0.5)))
        level = np.where(np.isnan(v) | ~(peak > 0), 0, np.clip(level, -7, 7))
        poisoned = ~np.isfinite(x).all(-1, keepdims=True)
        level = np.where(poisoned, 0, level)
        scale = np.where(poisoned, np.float32("nan"), peak / np.float32(7))
        scaled = x.astype(np.float64) * 7 / peak
    flat = x.shape[:-2] + (-1,)
    return (level + 7).astype(np.int64).reshape(flat), scale[..., 0], scaled.reshape(flat)


def norm_rotate(x, gain, eps, pos, base, halves):
    """x [rows, heads, head_dim] at positions pos [rows]; returns y and |a| + |b|
    of each element's pair before the rotation (what its roundings scale with)."""
    x = x.astype(np.float64)
    hd = x.shape[-1]
    if gain is not None:
        with np.errstate(all="ignore"):
            x = gain.astype(np.float64) * x / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    if not base:
        return x, np.abs(x)
    angle = pos.astype(np.float64)[:, None, None] * base ** (-2.0 * np.arange(hd // 2) / hd)
    c, s = np.cos(angle), np.sin(angle)
    ia = np.arange(hd // 2) if halves else np.arange(0, hd, 2)
    ib = ia + hd // 2 if halves else ia + 1
    y, mag = np.empty_like(x), np.empty_like(x)
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, a * s + b * c
    mag[..., ia] = mag[..., ib] = np.abs(a) + np.abs(b)
    return y, mag


def slot(p, sinks, capacity):
    return p if p < sinks else sinks + (p - sinks) % (capacity - sinks)


def codes_agree(got, want, scaled):
    """Equal, but for an element whose scaled value lies next to a border
    between two codes: keys are rounded to fp32 once and scaled by two more
    fp32 operations, at most 7 * 4 * 2^-24 of error."""
    frac = np.abs(scaled)
    near = np.abs(frac - np.floor(frac) - 0.5) <= 2.0 ** -18
    return (np.abs(got - want) <= near).all()


# ---------------------------------------------------------------- attention

def visible(pos, last, sinks, capacity, window):
    """Positions that the query at `pos` sees once the ring holds up to `last`."""
    ring = capacity - sinks
    oldest = max(sinks, last - ring + 1)
    if window:
        oldest = max(oldest, pos - window + 1)
    return list(range(min(sinks, pos + 1))) + list(range(oldest, pos + 1))


def attend(q, k, v, scale, v_scales, kind="f32"):
    """One query head over its visible keys and values (64 bits), and the bound
    of an evaluation with fp32 sums: scores within (hd / 16 + 8) u of sum |q k|,
    the exponential within 2^-21, n / 16 + 64 additions. On top of that the
    query's elements and the weights x value scales enter as integers:
    - an element is off by half a step where the largest of its 64 is at least
      4177855 steps (fp32) or 16319.5 (16 bits), HELD as in product();
    - a weight by half a step where the largest of its tile of 32 tokens, all
      within 31 places of it, is at least 2^22 (2^14) steps, times a level of
      at most 7."""
    q, k, v = (t.astype(np.float64) for t in (q, k, v))
    s = scale * (k @ q)
    e = np.exp(s - s.max())
    p = e / e.sum()
    wide = (abs(scale) * (np.abs(k) @ np.abs(q))).max()
    tops = np.abs(q).reshape(-1, GROUP).max(1)
    held = (abs(scale) * HELD[kind] * (np.abs(k).reshape(len(k), -1, GROUP).sum(2) @ tops)).max()
    weight = p @ np.abs(v)
    w = np.pad(p * v_scales.max(1), 31)
    near = np.lib.stride_tricks.sliding_window_view(w, 63).max(1)
    least = 7 * (2.0 ** -23 if kind == "f32" else 2.0 ** -15) * near.sum()
    score = (q.size / 16 + 8) * U * wide + held
    return p @ v, (2 * score + 2.0 ** -21 + (len(s) / 16 + 64) * U) * weight + least
