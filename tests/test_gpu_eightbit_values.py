"""8-bit operators on the device at values where their arithmetic could lose:
weights that nearly cancel, scores, scales and values far from 1."""
import numpy as np
import pytest

import _eightbit as eb
from test_gpu_eightbit import TYPES, Device, _attend_all, _attention, _dev, _np, _typed

pytestmark = pytest.mark.gpu

# (query heads, tokens) of one key head: one pair and up to 8 in integer digits, 16 in fp16 by warps, 128 and more in
# blocks
PAIRS = [(1, 1), (4, 2), (4, 4), (8, 17), (2, 90)]


@pytest.mark.parametrize("hq,tokens", PAIRS)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("kind", list(TYPES))
def test_weights_keep_22_bits(gpu, kind, hd, hq, tokens):
    """Weights 1 and a little more than 1/2 of values that cancel but for that little: an output as small as 2^-12 of its
    parts, which weights of 11 bits read as 0. The bound is that of weights in two parts, the type's only in the output."""
    n = 96
    c = eb.Cache(np.random.RandomState(0), 3, 32, 1, hd, [[0, 1, 2]])
    for name in "kv":
        c.codes[name][:] = 0
    at = np.arange(n)
    second = at % 3 > 0                      # two of three tokens weigh about a half
    flat = {name: c.codes[name].reshape(n, hd) for name in "kv"}     # pages in order: tokens in order
    flat["k"][~second, 0] = 127
    flat["v"][:] = np.where(second, -100, 100)[:, None]
    c.scales["k"][:] = np.float32(1 / 127)
    c.scales["v"][:] = np.float32(0.013)
    d = Device(gpu, c)
    scale = float(np.float32(np.log(2 / (1 + 0.9 * 2.0 ** -11)) / (127 * np.float64(np.float32(1 / 127)))))
    q = np.zeros((tokens, hq, hd))
    q[:, :, 0] = 1
    qt, qv = _typed(q.reshape(tokens, -1), kind)
    position = n - tokens
    out = _np(_attention(gpu, d, _dev(np.array([position], np.int64)), tokens, kind, qt, hq, scale=scale)).reshape(tokens, hq, hd)
    y, bound = _attend_all(c, qv.reshape(tokens, hq, hd), [position], tokens, hq, 0, scale, "f32")
    whole = (position + np.arange(tokens)) % 3 == 2                  # rows that see whole triples
    assert (np.abs(y[whole]) < 2.0 ** -11 * 1.3).all() and (bound[whole] < 2.0 ** -14).all()
    assert (np.abs(out - y) <= bound + 1.01 * eb.rounding(y, kind)).all()
