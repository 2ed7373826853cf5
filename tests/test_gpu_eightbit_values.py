"""8-bit operators on the device at values where their arithmetic could lose:
weights that nearly cancel, scores, scales and values far from 1."""
import numpy as np
import pytest
import torch

import _eightbit as eb
from test_gpu_eightbit import TYPES, Device, _attend_all, _attention, _dev, _np, _quantized, _stream, _typed

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


def _one_hot(c, q, table, positions, tokens, window, scale):
    """Rows whose scores lie so far apart that only the tokens of the largest one weigh: the mean of their values
    [rows, heads, hd], and the bound of its evaluation (eb.attend's without the scores', and a weight that is a power of two)."""
    batch, hd = len(positions), q.shape[-1]
    y, bound = np.zeros(q.shape), np.zeros(q.shape)
    for b in range(batch):
        (k, there), (v, _) = (c.values(n, b, 0, positions[b] + tokens, 0) for n in "kv")
        for t in range(tokens):
            i = positions[b] + t
            see = there & (np.arange(len(there)) <= i)
            if window:
                see &= np.arange(len(there)) > i - window
            for h in range(q.shape[1]):
                s = scale * (k @ q[b * tokens + t, h])
                best = s == s[see].max()
                best &= see
                rest = s[see & ~best]
                assert not rest.size or s[best].max() - rest.max() > 2.0 ** -17 * np.abs(s[see]).max() + 100
                y[b * tokens + t, h] = v[best].mean(0)
                bound[b * tokens + t, h] = (2.0 ** -20 + (see.sum() / 32 * 6 + 128) * 2 * eb.U) * np.abs(v[best]).mean(0)
    return y, bound


def _far_scores(gpu, kind, hd, hq, tokens, size, page=32):
    """Scores of about +-size, by one element of the query and codes 20..120 of the keys, some of them twice."""
    rng = np.random.RandomState(hd + hq)
    per = (200 + tokens) // page + 1
    c = eb.Cache(rng, 2 * per, page, 1, hd, np.arange(2 * per).reshape(2, per))
    c.codes["k"][:] = 0
    c.codes["k"][:, :, :, 3] = rng.randint(20, 121, (2 * per, 1, page))
    c.scales["k"][:] = np.float32(0.0123)    # of one size: a page's scale does not part equal codes
    d = Device(gpu, c)
    q = np.zeros((2 * tokens, hq, hd))
    q[:, :, 3] = np.exp(rng.uniform(-0.3, 0.3, (2 * tokens, hq))) * rng.choice([-1, 1], (2 * tokens, hq))
    qt, qv = _typed(q.reshape(2 * tokens, -1), kind)
    scale = float(np.float32(size / 1.2))
    positions = [150, 200 - tokens]
    qv = qv.reshape(-1, hq, hd)
    for window in (0, 70):
        out = _np(_attention(gpu, d, _dev(np.array(positions, np.int64)), tokens, kind, qt, hq, window, scale)).reshape(-1, hq, hd)
        y, bound = _one_hot(c, qv, c.table, positions, tokens, window, scale)
        assert (np.abs(out - y) <= bound + 1.01 * eb.rounding(y, kind)).all()


@pytest.mark.parametrize("hq,tokens", [(1, 1), (4, 2), (4, 4), (3, 10)])
@pytest.mark.parametrize("size", [2.0 ** 14, 2.0 ** 17, 2.0 ** 24, 2.0 ** 26, 2.0 ** 33, 2.0 ** 41])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("kind", list(TYPES))
def test_scores_far_from_0(gpu, kind, hd, size, hq, tokens):
    """The largest score's tokens weigh alone, whatever the scores' steps in fp32 are."""
    _far_scores(gpu, kind, hd, hq, tokens, size)


@pytest.mark.parametrize("hq,tokens,page", [(2, 70, 32), (8, 20, 64), (3, 45, 64)])
@pytest.mark.parametrize("size", [2.0 ** 14, 2.0 ** 17, 2.0 ** 24, 2.0 ** 26, 2.0 ** 33, 2.0 ** 41])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("kind", list(TYPES))
def test_scores_far_from_0_of_many_queries(gpu, kind, hd, size, hq, tokens, page):
    _far_scores(gpu, kind, hd, hq, tokens, size, page)


@pytest.mark.parametrize("hq,tokens", PAIRS)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_scores_past_fp32(gpu, kind, hd, hq, tokens):
    """A query whose every score is -inf in fp32 reads NaN, as the formula gives it; beside finite ones they weigh nothing;
    a query that sees nothing reads 0."""
    page, per = 32, 12
    c = eb.Cache(np.random.RandomState(hd), 2 * per, page, 1, hd, np.arange(2 * per).reshape(2, per))
    c.codes["k"][:] = 7
    c.scales["k"][:] = np.float32(1e30)
    c.scales["k"][per + 5] = np.float32(1e-30)                   # sequence 1, tokens 160..191: finite
    table = np.concatenate([c.table, np.full((1, per), -1, np.int32)])
    c.table = table                          # sequence 2: no page
    d = Device(gpu, c)
    q = np.full((3 * tokens, hq, hd), -1e30)
    qt, _ = _typed(q.reshape(3 * tokens, -1), kind)
    first = per * page - tokens
    out = _np(_attention(gpu, d, _dev(np.array([first] * 3, np.int64)), tokens, kind, qt, hq)).reshape(3, tokens, hq, hd)
    assert np.isnan(out[0]).all() and (out[2] == 0).all()
    y = c.values("v", 1, 160, 192, 0)[0].mean(0)                 # all 32 scores are alike
    bound = (2.0 ** -20 + (per + 128) * 2 * eb.U) * np.abs(c.values("v", 1, 160, 192, 0)[0]).mean(0)
    assert (np.abs(out[1] - y) <= bound + 1.01 * eb.rounding(y, kind)).all()


@pytest.mark.parametrize("size", [2.0 ** 12, 2.0 ** 30, 2.0 ** 60, 2.0 ** 120])
@pytest.mark.parametrize("hq,tokens,hd", [(4, 4, 64), (8, 17, 64), (2, 90, 128)])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_weights_on_pages_of_small_scales(gpu, kind, hq, tokens, hd, size):
    """The softmax sits on pages whose neighbours' values are `size` times as large and weigh nothing: every weight keeps its
    bits. The bound is eb.attend's with the largest weight x value in place of the largest value."""
    rng = np.random.RandomState(hd)
    page, per = 32, 7
    c = eb.Cache(rng, 2 * per, page, 1, hd, np.arange(2 * per).reshape(2, per))
    c.codes["k"][:, :, :, 0] = 100
    c.scales["k"][:] = np.float32(0.01)
    for b in range(2):                       # every second page, from the first or the second on
        for j in range(b, per, 2):
            c.codes["k"][b * per + j, :, :, 0] = -100
            c.scales["v"][b * per + j] *= size * 2.0 ** -40
    for at in range(2 * per):
        if (at % per - at // per) % 2:
            c.scales["v"][at] *= 2.0 ** -40
    d = Device(gpu, c)
    q = 0.05 * rng.randn(2 * tokens, hq, hd)
    q[:, :, 0] = 30
    qt, qv = _typed(q.reshape(2 * tokens, -1), kind)
    positions = [190 - tokens, 200 - tokens]
    scale = float(np.float32(4.0))           # the others' scores lie 240 below: weights of 2^-346
    out = _np(_attention(gpu, d, _dev(np.array(positions, np.int64)), tokens, kind, qt, hq, scale=scale)).reshape(-1, hq, hd)
    qv = qv.reshape(-1, hq, hd)
    seen = 0
    for b in range(2):
        k, v = (c.values(n, b, 0, positions[b] + tokens, 0)[0] for n in "kv")
        for t in range(tokens):
            n = positions[b] + t + 1
            for h in range(hq):
                s = scale * (k[:n] @ qv[b * tokens + t, h])
                p = np.exp(s - s.max())
                p /= p.sum()
                assert p[k[:n, 0] < 0].sum() < 1e-80
                small = k[:n, 0] > 0
                y, bound = eb.attend(qv[b * tokens + t, h], k[:n][small], v[:n][small], scale, "f32")
                o = out[b * tokens + t, h]
                assert (np.abs(o - y) <= bound + 1.01 * eb.rounding(y, kind)).all()
                seen += 1
    assert seen == 2 * tokens * hq


@pytest.mark.parametrize("m,k,n", [(40, 1024, 1100), (8, 1024, 1100), (40, 4096, 300)])
def test_fp32_products_on_the_tensor_cores_after_a_long_row(gpu, m, k, n):
    """The kernels of fp32 products whose waits are bounded (matrices of 2^20 codes and more: the GEMM with and without parts
    of k, the GEMV) wait without limit behind the longest row, which lets them start early: no NaN, and nothing left for the
    matrix's next call."""
    assert k * n >= 1 << 20
    width = 1 << 30
    x = torch.ones(width, device="cuda")
    out, scale = torch.empty(width, dtype=torch.int8, device="cuda"), torch.empty(1, device="cuda")
    levels = np.random.RandomState(m).randint(-127, 128, (k, n)).astype(np.int8)
    w = _quantized(gpu, levels, np.ones(n, np.float32))
    ones, y = torch.ones(m, k, device="cuda"), torch.zeros(m, n, device="cuda")
    for turn in range(2):                    # the first call of a kernel waits for what is under way
        torch.cuda.synchronize()
        y.zero_()
        gpu.norm_q8(1, width if turn else 1000000, type=gpu.TYPE_F32, x=x.data_ptr(), residual=x.data_ptr(),
                    gain=x.data_ptr(), codes=out.data_ptr(), scales=scale.data_ptr(), stream_ptr=_stream())
        w.matmul_async(ones.data_ptr(), y.data_ptr(), m, _stream())
    want = levels.sum(0, dtype=np.int64).astype(np.float32)
    assert torch.equal(y, _dev(want).expand(m, n))
    np.testing.assert_array_equal(w.matmul(np.ones((m, k), np.float32)), np.broadcast_to(want, (m, n)))
    w.close()


@pytest.mark.parametrize("hq,tokens,windows", [(1, 1, (0, 333)), (4, 4, (0, 65)), (8, 40, (1, 100, 300))])
@pytest.mark.parametrize("page", [32, 64])
def test_the_end_of_the_longest_table(gpu, page, hq, tokens, windows):
    """Append and attention at the last positions that a table can reach, and past them."""
    rng = np.random.RandomState(page)
    hd, per = 64, ((1 << 31) - 64) // page
    table = np.full((1, per), -1, np.int32)
    table[0, -12:] = rng.permutation(13)[:12]
    c = eb.Cache(rng, 13, page, 1, hd, table)
    d = Device(gpu, c)
    for first in (per * page - tokens, per * page - 30):         # up to the end; some tokens past it, where they are many
        x = rng.randn(tokens, 1, hd).astype(np.float32)
        xt, pos = _dev(x), _dev(np.array([first], np.int64))
        d.cache.append(pos.data_ptr(), tokens, k=xt.data_ptr(), v=xt.data_ptr(), stream_ptr=_stream())
        for n, codes, scales in (("k", d.k, d.ks), ("v", d.v, d.vs)):
            c.append(n, 0, first, x)
            np.testing.assert_array_equal(codes.cpu().numpy(), c.codes[n])
            np.testing.assert_array_equal(scales.cpu().numpy(), c.scales[n])
        qt, qv = _typed(rng.randn(tokens, hq * hd), "f32")
        for window in windows:
            out = _np(_attention(gpu, d, pos, tokens, "f32", qt, hq, window, longest=1000)).reshape(tokens, hq, hd)
            held = window if window else 12 * page + tokens      # nothing lies before the last twelve pages
            y, bound = _attend_all(c, qv.reshape(tokens, hq, hd), [first], tokens, hq, held, hd ** -0.5, "f32")
            assert (np.abs(out - y) <= bound + 1.01 * eb.rounding(y, "f32")).all()


@pytest.mark.parametrize("hq,tokens", PAIRS)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_values_near_the_end_of_fp32(gpu, kind, hd, hq, tokens):
    """Values of up to 2^119, 190 of them: their sum lies in fp32's range."""
    rng = np.random.RandomState(hd + tokens)
    c = eb.Cache(rng, 6, 32, 1, hd, [np.arange(6)])
    c.scales["v"][:] = np.float32(2.0 ** 112)
    c.scales["v"][2] = np.float32(2.0 ** 90)
    d = Device(gpu, c)
    qt, qv = _typed(0.01 * rng.randn(tokens, hq * hd), kind)
    first = 190 - tokens
    out = _np(_attention(gpu, d, _dev(np.array([first], np.int64)), tokens, kind, qt, hq)).reshape(tokens, hq, hd)
    y, bound = _attend_all(c, qv.reshape(tokens, hq, hd), [first], tokens, hq, 0, hd ** -0.5, "f32")
    assert (np.abs(out - y) <= bound + 1.01 * eb.rounding(y, kind)).all()


@pytest.mark.parametrize("width", [40, 4096, 5003, 20000])
@pytest.mark.parametrize("kind", list(TYPES))
def test_row_scales_near_the_end_of_fp32(gpu, kind, width):
    """Gains so large that peak / root-mean-square leaves fp32 where the scale, a 127th of it, does not."""
    x = np.zeros((3, width))
    x[0, width // 2] = 2.0 ** -10            # root-mean-square: 2^-10 / sqrt(width)
    x[1, :] = 1.0
    x[2, 3:7] = -2.0 ** -12
    gain = np.full(width, min(2.0 ** 127, 2.0 ** 134 / np.sqrt(width)), np.float32)
    xt, xv = _typed(x, kind)
    gt = _dev(gain)
    codes = torch.empty(3, -(-width // 16) * 16, dtype=torch.int8, device="cuda")
    scales = torch.empty(3, device="cuda")
    gpu.norm_q8(3, width, type={"f32": gpu.TYPE_F32, "f16": gpu.TYPE_F16, "bf16": gpu.TYPE_BF16}[kind], x=xt.data_ptr(),
                gain=gt.data_ptr(), eps=0.0, codes=codes.data_ptr(), scales=scales.data_ptr(), stream_ptr=_stream())
    want, scale = eb.norm_rows(xv, gain, True, 0.0)
    assert 2.0 ** 128 < 127 * scale[0] < 2.0 ** 134.99          # peak / rms of the first row
    np.testing.assert_array_equal(codes[:, :width].cpu().numpy(), want)
    assert (np.abs(_np(scales) - scale) <= eb.NORM_SCALE * scale).all()


@pytest.mark.parametrize("kind,hd,tokens,halves,pad", [("f32", 64, 1, 0, 0), ("bf16", 128, 1, 1, 0), ("f16", 128, 1, 0, 1), ("bf16", 128, 77, 1, 0),
                                                       ("f32", 128, 150, 0, 0), ("f16", 64, 40, 1, 0), ("bf16", 64, 33, 0, 3)])
def test_append_in_place(gpu, kind, hd, tokens, halves, pad):
    """Outputs that are their own input rows: what other rows of output get, for more heads than are read ahead."""
    rng = np.random.RandomState(hd + tokens)
    hq, hk, batch, page = 21, 3, 3, 32
    per = (60 + tokens) // page + 1
    caches = [eb.Cache(np.random.RandomState(1), batch * per, page, hk, hd, np.arange(batch * per).reshape(batch, per))
              for _ in range(2)]
    devices = [Device(gpu, c) for c in caches]
    width, rows = (hq + 2 * hk) * hd + pad, batch * tokens
    xt, _ = _typed(rng.randn(rows, width) * 3, kind)
    own = xt.clone()
    gains = [_dev((1 + 0.2 * rng.randn(hd)).astype(np.float32)) for _ in range(2)]
    pos, size = _dev(np.array([0, 31, 60], np.int64)), xt.element_size()
    outs = [torch.full_like(xt, 5.0) for _ in range(3)]
    for x, d, to in ((xt, devices[0], outs), (own, devices[1], None)):
        at = [x.data_ptr() + n * hd * size for n in (0, hq, hq + hk)]
        o = at if to is None else [t.data_ptr() + n * hd * size for t, n in zip(to, (0, hq, hq + hk))]
        d.cache.append(pos.data_ptr(), tokens, type={"f32": gpu.TYPE_F32, "f16": gpu.TYPE_F16, "bf16": gpu.TYPE_BF16}[kind],
                       q_heads=hq, q=at[0], k=at[1], v=at[2], q_stride=width, k_stride=width, v_stride=width, q_out=o[0],
                       q_out_stride=width, k_out=o[1], k_out_stride=width, v_out=o[2], v_out_stride=width,
                       q_gain=gains[0].data_ptr(), k_gain=gains[1].data_ptr(), rope_base=10000.0, halves=bool(halves),
                       stream_ptr=_stream())
    parts = [outs[0][:, :hq * hd], outs[1][:, hq * hd:(hq + hk) * hd], outs[2][:, (hq + hk) * hd:(hq + 2 * hk) * hd]]
    assert torch.equal(own[:, :(hq + 2 * hk) * hd], torch.cat(parts, 1))
    assert torch.equal(own[:, (hq + 2 * hk) * hd:], xt[:, (hq + 2 * hk) * hd:]) and not torch.equal(own, xt)
    for name in ("k", "v", "ks", "vs"):
        assert torch.equal(getattr(devices[0], name), getattr(devices[1], name))


def test_many_queries_past_32_bits(gpu):
    """Pages beyond 2^31 codes of a pool, read by blocks of 128 pairs."""
    rng = np.random.RandomState(5)
    page, hk, hd, pages, tokens = 64, 8, 128, 40000, 33          # 2.6e9 codes
    c = eb.Cache(rng, 4, page, hk, hd, [[0, 1, 2, 3]])
    at = torch.tensor([39999, 0, 33000, 39001], device="cuda")
    k = torch.zeros(pages, hk, page, hd, dtype=torch.int8, device="cuda")
    v = torch.zeros_like(k)
    ks, vs = torch.ones(pages, hk, device="cuda"), torch.ones(pages, hk, device="cuda")
    for big, small in ((k, c.codes["k"]), (v, c.codes["v"]), (ks, c.scales["k"]), (vs, c.scales["v"])):
        big[at] = _dev(small)
    table, pos = at.to(torch.int32)[None].contiguous(), _dev(np.array([200], np.int64))
    cache = gpu.KV8Cache(k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), pages, page, hk, hd, table.data_ptr(), 1, 4)
    qt, qv = _typed(rng.randn(tokens, 2 * hk * hd), "bf16")
    out = torch.empty_like(qt)
    cache.attention(pos.data_ptr(), tokens, type=gpu.TYPE_BF16, q_heads=2 * hk, q=qt.data_ptr(), out=out.data_ptr(), stream_ptr=_stream())
    y, bound = _attend_all(c, qv.reshape(tokens, 2 * hk, hd), [200], tokens, 2, 0, hd ** -0.5, "f32")
    assert (np.abs(_np(out).reshape(y.shape) - y) <= bound + 1.01 * eb.rounding(y, "bf16")).all()
