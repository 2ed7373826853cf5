"""The 8-bit operators on the device against their 64-bit formulas
(tests/_eightbit.py): rows in 8 bits, products of them, the append to paged
caches, attention over them, and a run of the four."""
import numpy as np
import pytest
import torch

import _eightbit as eb

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _dz_type(gpu, kind):
    return {"f32": gpu.TYPE_F32, "f16": gpu.TYPE_F16, "bf16": gpu.TYPE_BF16}[kind]


def _typed(a, kind):
    """`a` rounded to the type: (device tensor, the values it holds in 64 bits)."""
    t = torch.from_numpy(np.ascontiguousarray(a, np.float32)).to(TYPES[kind])
    return t.cuda(), t.double().numpy()


def _np(t):
    return t.double().cpu().numpy()


def _dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _ptr(t):
    return None if t is None else t.data_ptr()


# --------------------------------------------------------------- rows in 8 bits

WIDTHS = [1, 2, 7, 31, 64, 100, 256, 257, 511, 512, 513, 1000, 1024, 2048, 2051, 4096, 5003, 8192, 8200, 16384, 16385,
          20011]


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("pad,shift", [(0, 0), (8, 0), (3, 1)])
def test_norm_q8(gpu, width, kind, pad, shift):
    """Every combination of residual, norm and gain, rows of wider buffers on and off 16-byte boundaries."""
    rows = 1 + 40 // (1 + width // 500)
    rng = np.random.RandomState(width + pad)
    ld = width + pad
    buffers = [_typed(np.r_[np.zeros(shift), (rng.randn(rows * ld) * np.exp(rng.randn(rows * ld) * 0.5))], kind) for _ in range(2)]
    xt, rt = (b[0][shift:] for b in buffers)
    xv, rv = (b[1][shift:].reshape(rows, ld)[:, :width] for b in buffers)
    gain = (1 + 0.3 * rng.randn(width)).astype(np.float32)
    gt = _dev(gain)
    for residual, norm, gained in [(1, 1, 1), (0, 1, 1), (1, 0, 0), (0, 0, 0), (0, 0, 1), (1, 1, 0)]:
        h = xv
        if residual:
            h = torch.from_numpy((xv + rv).astype(np.float32)).to(TYPES[kind]).double().numpy()
        lc = width + (16 - width) % 16 + pad
        codes = torch.full((rows, lc), 99, dtype=torch.int8, device="cuda")
        scales = torch.full((rows + 1,), 7.0, device="cuda")
        total = torch.full((rows, ld), 5.0, dtype=TYPES[kind], device="cuda")
        gpu.norm_q8(rows, width, type=_dz_type(gpu, kind), x=xt.data_ptr(), x_stride=ld,
                    residual=rt.data_ptr() if residual else None, residual_stride=ld, sum_out=total.data_ptr(),
                    sum_stride=ld, gain=gt.data_ptr() if gained else None, norm=bool(norm), eps=1e-5,
                    codes=codes.data_ptr(), codes_stride=lc, scales=scales.data_ptr(), stream_ptr=_stream())
        want, scale = eb.norm_rows(h, gain if gained else None, norm, 1e-5)
        got = codes.cpu().numpy().astype(np.int64)
        np.testing.assert_array_equal(got[:, :width], want)
        assert (got[:, width:] == 99).all() and float(scales[rows]) == 7.0
        tolerance = eb.NORM_SCALE if norm else eb.U
        assert (np.abs(_np(scales[:rows]) - scale) <= tolerance * scale + 2.0 ** -149).all()
        np.testing.assert_array_equal(_np(total[:, :width]), h)
        assert (total[:, width:] == 5.0).all()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("width", [40, 2000, 20000])
def test_norm_q8_special_rows(gpu, kind, width):
    rng = np.random.RandomState(3)
    x = rng.randn(12, width)
    x[0] = 0
    x[1, width // 2] = np.inf
    x[2, width - 1] = np.nan
    x[3] *= 1e30
    x[4] *= 2.0 ** -110
    x[5] *= 1e-38
    x[6] = 0
    x[6, 3] = 2.0 ** -126
    x[7] = 3e38 * np.sign(x[7])
    x[8] = 0
    x[8, 1] = -1.0
    x[9, 0] = -np.inf
    xt, xv = _typed(x, kind)
    for norm, eps in [(False, 0.0), (True, 0.0), (True, 1e-6)]:
        lc = -(-width // 16) * 16
        codes, scales = torch.empty(12, lc, dtype=torch.int8, device="cuda"), torch.empty(12, device="cuda")
        gpu.norm_q8(12, width, type=_dz_type(gpu, kind), x=xt.data_ptr(), norm=norm, eps=eps, codes=codes.data_ptr(),
                    scales=scales.data_ptr(), stream_ptr=_stream())
        want, scale = eb.norm_rows(xv, None, norm, eps)
        np.testing.assert_array_equal(codes[:, :width].cpu().numpy(), want)
        got = _np(scales)
        assert np.isnan(got[[1, 2, 9]]).all() and got[0] == 0
        ok = [0, 3, 4, 5, 6, 7, 8, 10, 11]
        # fp32's smallest numbers: a step of them instead of a relative one
        assert (np.abs(got - scale)[ok] <= eb.NORM_SCALE * scale[ok] + 2.0 ** -148).all(), (norm, eps)


@pytest.mark.parametrize("width", [96, 3000, 20000])
def test_norm_q8_in_place(gpu, width):
    """The sum may replace x or the residual."""
    torch.manual_seed(1)
    for which in (0, 1):
        x, r = torch.randn(5, width, device="cuda").bfloat16(), torch.randn(5, width, device="cuda").bfloat16()
        want = (x.float() + r.float()).bfloat16()
        codes, scales = torch.empty(2, 5, width, dtype=torch.int8, device="cuda"), torch.empty(2, 5, device="cuda")
        for n, total in enumerate((torch.empty_like(x), (x, r)[which])):
            gpu.norm_q8(5, width, type=gpu.TYPE_BF16, x=x.data_ptr(), residual=r.data_ptr(), sum_out=total.data_ptr(),
                        codes=codes[n].data_ptr(), codes_stride=width, scales=scales[n].data_ptr(), stream_ptr=_stream())
        assert torch.equal((x, r)[which], want)
        assert torch.equal(codes[0], codes[1]) and torch.equal(scales[0], scales[1])


# --------------------------------------------------------------------- products

SHAPES = [(1, 1, 1), (1, 16, 16), (3, 31, 5), (8, 128, 128), (9, 129, 127), (16, 1000, 130), (17, 257, 33), (31, 500, 1003),
          (32, 4099, 40), (33, 384, 384), (64, 2048, 2048), (65, 130, 129), (127, 1111, 300), (128, 128, 4096),
          (129, 4096, 1000), (200, 256, 256), (256, 640, 1024), (257, 1025, 513), (500, 3000, 700), (1, 4096, 32000),
          (1000, 2048, 2048), (2, 100000, 40), (20, 70000, 24), (300, 131072, 130), (5, 131072, 17)]


def _quantized(gpu, levels, scales, bits=8):
    qmax = 127 if bits == 8 else 7
    codes = (levels.astype(np.int64) + qmax).astype(np.uint8).reshape(-1)
    if bits == 4:
        codes = np.r_[codes, np.zeros(codes.size % 2, np.uint8)]
        codes = codes[0::2] | codes[1::2] << 4
    gran = gpu.GRAN_COLUMN if scales.size == levels.shape[1] and levels.shape[1] > 1 else gpu.GRAN_TENSOR
    return gpu.QuantizedWeightMatrix(scales, codes, levels.shape[0], levels.shape[1], bits, gran)


@pytest.mark.parametrize("m,k,n", SHAPES)
def test_products(gpu, m, k, n):
    rng = np.random.RandomState(m + k + n)
    levels = np.clip(np.rint(rng.randn(k, n) * 50), -127, 127).astype(np.int8)
    col = (np.exp(rng.randn(n)) * 1e-3).astype(np.float32)
    lda = -(-k // 16) * 16 + 16 * (m % 3)
    codes = rng.randint(-128, 128, (m, lda)).astype(np.int8)        # whatever lies past k
    scales = np.exp(rng.randn(m)).astype(np.float32)
    bias = rng.randn(n).astype(np.float32)
    w = _quantized(gpu, levels, col)
    ct, st, bt = _dev(codes), _dev(scales), _dev(bias)
    for kind in TYPES:
        for b in (None, bt):
            ldc = n + (m % 2) * 3
            y = torch.full((m, ldc), 3.0, dtype=TYPES[kind], device="cuda")
            w.matmul_q8_async(ct.data_ptr(), st.data_ptr(), y.data_ptr(), m, _stream(), type=_dz_type(gpu, kind), lda=lda,
                              ldc=ldc, bias_ptr=_ptr(b))
            ref, bound = eb.product(codes[:, :k], scales, levels, col, None if b is None else bias, kind)
            err = eb.product_error(_np(y[:, :n]), ref, bound, kind)
            assert (err <= bound).all(), (kind, b is None, (err / np.maximum(bound, 1e-300)).max())
            assert (y[:, n:] == 3.0).all()
    w.close()


@pytest.mark.parametrize("m", [4, 40, 300])
def test_products_of_4_bit_and_one_scale_matrices(gpu, m):
    rng = np.random.RandomState(m)
    k, n = 333, 211
    codes, scales = rng.randint(-127, 128, (m, 336)).astype(np.int8), np.ones(m, np.float32)
    for levels, col, bits in [(rng.randint(-7, 8, (k, n)), np.exp(rng.randn(n)), 4),
                              (rng.randint(-127, 128, (k, n)), np.array([0.25]), 8)]:
        levels, col = levels.astype(np.int8), col.astype(np.float32)
        w = _quantized(gpu, levels, col, bits)
        y = torch.empty(m, n, device="cuda")
        ct, st = _dev(codes), _dev(scales)
        w.matmul_q8_async(ct.data_ptr(), st.data_ptr(), y.data_ptr(), m, _stream())
        ref, bound = eb.product(codes[:, :k], scales, levels, col, None, "f32")
        assert (np.abs(_np(y) - ref) <= bound).all()
        w.close()


@pytest.mark.parametrize("m", [2, 30, 140])
def test_product_extremes(gpu, m):
    """Every code at its largest over the most rows, a NaN scale, columns of scale 0."""
    k, n = 131072, 20
    levels = np.full((k, n), 127, np.int8)
    levels[:, 1] = -127
    col = np.full(n, 1e-6, np.float32)
    col[2] = 0
    codes = np.full((m, k), -128, np.int8)
    scales = np.ones(m, np.float32)
    scales[m // 2] = np.nan
    w = _quantized(gpu, levels, col)
    y = torch.empty(m, n, device="cuda")
    ct, st = _dev(codes), _dev(scales)
    w.matmul_q8_async(ct.data_ptr(), st.data_ptr(), y.data_ptr(), m, _stream())
    ref, bound = eb.product(codes, scales, levels, col, None, "f32")
    got = _np(y)
    assert np.isnan(got[m // 2]).all()
    keep = np.arange(m) != m // 2
    assert (np.abs(got - ref)[keep] <= bound[keep]).all() and (got[keep, 2] == 0).all()
    w.close()


@pytest.mark.parametrize("m,k,n", [(40, 512, 300), (1000, 1024, 9000)])
def test_products_after_a_long_kernel(gpu, m, k, n):
    """A product waits, however long, for a kernel that lets it start before it ends: the longest row,
    of one block, takes 3.7 s."""
    width = 1 << 30
    x = torch.ones(width, device="cuda")
    out, scale = torch.empty(width, dtype=torch.int8, device="cuda"), torch.empty(1, device="cuda")
    levels = np.random.RandomState(m).randint(-127, 128, (k, n)).astype(np.int8)
    w = _quantized(gpu, levels, np.ones(n, np.float32))
    codes, ones = torch.ones(m, k, dtype=torch.int8, device="cuda"), torch.ones(m, device="cuda")
    y = torch.zeros(m, n, device="cuda")
    for turn in range(2):                    # the first call of a kernel waits for what is under way
        torch.cuda.synchronize()
        y.zero_()
        gpu.norm_q8(1, width if turn else 1000000, type=gpu.TYPE_F32, x=x.data_ptr(), residual=x.data_ptr(),
                    gain=x.data_ptr(), codes=out.data_ptr(), scales=scale.data_ptr(), stream_ptr=_stream())
        w.matmul_q8_async(codes.data_ptr(), ones.data_ptr(), y.data_ptr(), m, _stream())
    assert torch.equal(y, _dev(levels.sum(0, dtype=np.int64).astype(np.float32)).expand(m, n))
    assert int(out[0]) == int(out[width - 1]) == 127
    w.close()


def test_fp32_products_after_a_long_row(gpu):
    """The product of fp32 rows, whose waits are bounded too, behind the longest row."""
    width, m, k, n = 1 << 30, 40, 512, 300
    x = torch.ones(width, device="cuda")
    out, scale = torch.empty(width, dtype=torch.int8, device="cuda"), torch.empty(1, device="cuda")
    levels = np.random.RandomState(1).randint(-127, 128, (k, n)).astype(np.int8)
    w = _quantized(gpu, levels, np.ones(n, np.float32))
    ones, y = torch.ones(m, k, device="cuda"), torch.zeros(m, n, device="cuda")
    for turn in range(2):
        torch.cuda.synchronize()
        y.zero_()
        gpu.norm_q8(1, width if turn else 1000000, type=gpu.TYPE_F32, x=x.data_ptr(), residual=x.data_ptr(),
                    gain=x.data_ptr(), codes=out.data_ptr(), scales=scale.data_ptr(), stream_ptr=_stream())
        w.matmul_async(ones.data_ptr(), y.data_ptr(), m, _stream())
    assert torch.equal(y, _dev(levels.sum(0, dtype=np.int64).astype(np.float32)).expand(m, n))
    w.close()


def test_product_refusals(gpu):
    rng = np.random.RandomState(0)
    v = rng.randn(64, 48).astype(np.float32)
    w, row = gpu.QuantizedWeightMatrix.encode(v, 8), gpu.QuantizedWeightMatrix.encode(v, 8, gpu.GRAN_ROW)
    big = gpu.QuantizedWeightMatrix(np.ones(1, np.float32), np.full(131073, 127, np.uint8), 131073, 1, 8, gpu.GRAN_COLUMN)
    a, s, c = (torch.zeros(4096, dtype=torch.int8, device="cuda"), torch.ones(64, device="cuda"),
               torch.full((8, 48), 2.0, device="cuda"))
    good = dict(codes_ptr=a.data_ptr(), scales_ptr=s.data_ptr(), c_ptr=c.data_ptr(), m=8, stream_ptr=_stream(), lda=64)
    for change in [dict(codes_ptr=a.data_ptr() + 8), dict(lda=72), dict(lda=48), dict(ldc=47), dict(m=0),
                   dict(m=(1 << 24) + 1), dict(type=5), dict(scales_ptr=None), dict(codes_ptr=None), dict(c_ptr=None),
                   dict(c_ptr=c.data_ptr() + 2), dict(bias_ptr=s.data_ptr() + 2), dict(scales_ptr=s.data_ptr() + 1)]:
        with pytest.raises(gpu.DzError) as e:
            w.matmul_q8_async(**{**good, **change})
        assert e.value.status == -1, change
    for other, lda in ((row, 64), (big, 131088)):
        with pytest.raises(gpu.DzError) as e:
            other.matmul_q8_async(**{**good, "lda": lda, "m": 1})
        assert e.value.status == -6
    torch.cuda.synchronize()
    assert (c == 2.0).all()
    for m in (w, row, big):
        m.close()


# ----------------------------------------------------------------------- append

class Device:
    """The cache of an oracle (_eightbit.Cache) on the device."""

    def __init__(self, gpu, c):
        self.k, self.v = _dev(c.codes["k"]), _dev(c.codes["v"])
        self.ks, self.vs = _dev(c.scales["k"]), _dev(c.scales["v"])
        self.table = _dev(c.table)
        self.cache = gpu.KV8Cache(self.k.data_ptr(), self.v.data_ptr(), self.ks.data_ptr(), self.vs.data_ptr(), c.pages,
                                  c.page, c.hk, c.hd, self.table.data_ptr(), *c.table.shape)


def _table(rng, batch, per, pages):
    return rng.permutation(pages)[:batch * per].reshape(batch, per).astype(np.int32)


APPENDS = [
    # kind, page, heads (queries, keys), head dim, positions, tokens, norm, rope, halves, pad
    ("f32", 32, (4, 4), 64, [0, 31, 32, 5], 1, 0, 0.0, 0, 0),
    ("bf16", 64, (8, 2), 128, [0, 63, 64, 100, 127], 1, 1, 10000.0, 0, 0),
    ("f16", 64, (6, 3), 64, [7, 60], 9, 1, 500.0, 1, 3),
    ("f32", 32, (2, 1), 128, [0, 17], 200, 1, 10000.0, 1, 0),
    ("bf16", 32, (0, 2), 64, [3], 33, 0, 10000.0, 0, 4),
    ("f16", 64, (5, 5), 128, [1, 0, 63], 64, 0, 0.0, 0, 1),
    ("bf16", 64, (8, 1), 128, [130], 130, 0, 1e6, 1, 0),
    ("f32", 64, (3, 1), 64, [100000], 17, 1, 10000.0, 0, 0),
    ("f32", 32, (1, 2), 128, [11, 12, 13, 14, 15, 16, 17], 2, 1, 0.0, 0, 0),
]


@pytest.mark.parametrize("kind,page,heads,hd,positions,tokens,norm,rope,halves,pad", APPENDS)
def test_append(gpu, kind, page, heads, hd, positions, tokens, norm, rope, halves, pad):
    (hq, hk), batch = heads, len(positions)
    rng = np.random.RandomState(hq * 7 + hk + tokens)
    per = (max(positions) + tokens - 1) // page + 2
    base = min(positions) // page            # pages before the first new tokens: none
    table = np.full((batch, per), -1, np.int32)
    table[:, base:] = _table(rng, batch, per - base, batch * (per - base) + 2)
    c = eb.Cache(rng, batch * (per - base) + 2, page, hk, hd, table)
    d = Device(gpu, c)
    rows, width = batch * tokens, (hq + 2 * hk) * hd + pad
    xt, xv = _typed(rng.randn(rows, width) * np.exp(rng.randn(rows, 1)), kind)
    q_gain, k_gain = ((1 + 0.2 * rng.randn(hd)).astype(np.float32) for _ in range(2))
    qg, kg, size, at = _dev(q_gain), _dev(k_gain), xt.element_size(), xt.data_ptr()
    outs = [torch.full((rows, max(h, 1) * hd + pad), 9.0, dtype=TYPES[kind], device="cuda") for h in (hq, hk, hk)]
    pos = _dev(np.array(positions, np.int64))
    d.cache.append(pos.data_ptr(), tokens, type=_dz_type(gpu, kind), q_heads=hq, q=at, k=at + hq * hd * size,
                   v=at + (hq + hk) * hd * size, q_stride=width, k_stride=width, v_stride=width,
                   q_out=outs[0].data_ptr(), q_out_stride=outs[0].shape[1], k_out=outs[1].data_ptr(),
                   k_out_stride=outs[1].shape[1], v_out=outs[2].data_ptr(), v_out_stride=outs[2].shape[1],
                   q_gain=qg.data_ptr() if norm else None, k_gain=kg.data_ptr() if norm else None, eps=1e-5,
                   rope_base=rope, halves=bool(halves), stream_ptr=_stream())
    p = (np.array(positions)[:, None] + np.arange(tokens)).reshape(-1)
    x = xv[:, :(hq + 2 * hk) * hd].reshape(rows, hq + 2 * hk, hd)
    if hq:
        y, mag = eb.norm_rotate(x[:, :hq], q_gain if norm else None, 1e-5, p, rope, halves)
        got = _np(outs[0][:, :hq * hd]).reshape(y.shape)
        # norm: sum (hd / 32 + 5 additions), root, two products; rotation: two products and angles rounded to fp32
        assert (np.abs(got - y) <= 24 * eb.U * mag + 1.01 * eb.rounding(y, kind)).all()
    assert (outs[0][:, hq * hd:] == 9.0).all()
    key, _ = eb.norm_rotate(x[:, hq:hq + hk], k_gain if norm else None, 1e-5, p, rope, halves)
    new = {"k": key.astype(np.float32).reshape(batch, tokens, hk, hd),
           "v": x[:, hq + hk:].astype(np.float32).reshape(batch, tokens, hk, hd)}
    before = {n: c.codes[n].copy() for n in "kv"}
    exact = {n: {} for n in "kv"}
    for b in range(batch):
        for n in "kv":
            exact[n].update(c.append(n, b, positions[b], new[n][b]))
    for n, codes, scales in (("k", d.k, d.ks), ("v", d.v, d.vs)):
        got, got_scales = codes.cpu().numpy(), scales.cpu().numpy()
        if n == "v" or not (norm or rope):
            np.testing.assert_array_equal(got_scales, c.scales[n])
            np.testing.assert_array_equal(got, c.codes[n])
        else:                                 # one rounding to fp32 of a value that two evaluations have in 64 bits
            assert (np.abs(got_scales - c.scales[n]) <= 4 * eb.U * c.scales[n]).all()
            off = np.abs(got.astype(int) - c.codes[n].astype(int))
            for (page_at, h), v in exact[n].items():
                assert (off[page_at, h, :len(v)] <= eb.near_border(v)).all()
                off[page_at, h, :len(v)] = 0
            assert not off.any()
        held = outs[1 if n == "k" else 2]
        for b in range(batch):
            for h in range(hk):
                # what the device's cache now holds
                c.codes[n], c.scales[n] = got, got_scales
                y, there = c.values(n, b, positions[b], positions[b] + tokens, h)
                assert there.all()
                o = _np(held[b * tokens:(b + 1) * tokens, h * hd:(h + 1) * hd])
                assert (np.abs(o - y) <= 1.01 * eb.rounding(y, kind) + eb.U * np.abs(y)).all()
        assert (held[:, hk * hd:] == 9.0).all()
        untouched = np.ones(got.shape[:2], bool)
        for page_at, h in exact[n]:
            untouched[page_at, h] = False
        np.testing.assert_array_equal(got[untouched], before[n][untouched])


def test_append_grows_scales_and_keeps_what_was_there(gpu):
    """Token by token with growing values: every scale and code of the page as the formula has them."""
    rng = np.random.RandomState(5)
    c = eb.Cache(rng, 3, 32, 2, 64, [[1]])
    d = Device(gpu, c)
    for j in range(32):
        y = (rng.randn(1, 2, 64) * (1 + j % 7)).astype(np.float32)
        t, pos = _dev(y), torch.tensor([j], device="cuda")
        d.cache.append(pos.data_ptr(), 1, k=t.data_ptr(), v=t.data_ptr(), stream_ptr=_stream())
        for n in "kv":
            c.append(n, 0, j, y)
        torch.cuda.synchronize()
    for n, codes, scales in (("k", d.k, d.ks), ("v", d.v, d.vs)):
        np.testing.assert_array_equal(codes.cpu().numpy(), c.codes[n])
        np.testing.assert_array_equal(scales.cpu().numpy(), c.scales[n])


def test_append_special_values(gpu):
    """Infinities and NaN mark a page until it is begun anew; zeros, tiny and huge values; a page of zeros that grows."""
    rng = np.random.RandomState(6)
    c = eb.Cache(rng, 8, 32, 1, 64, [[i, 7 - i] for i in range(4)])
    d = Device(gpu, c)

    def step(positions, rows):
        y = np.stack(rows).reshape(4, -1, 1, 64).astype(np.float32)
        t, pos = _dev(y), torch.tensor(positions, device="cuda")
        d.cache.append(pos.data_ptr(), y.shape[1], k=t.data_ptr(), v=t.data_ptr(), stream_ptr=_stream())
        torch.cuda.synchronize()
        with np.errstate(all="ignore"):
            for b in range(4):
                for n in "kv":
                    c.append(n, b, positions[b], y[b])
        for n, codes, scales in (("k", d.k, d.ks), ("v", d.v, d.vs)):
            np.testing.assert_array_equal(scales.cpu().numpy(), c.scales[n])
            np.testing.assert_array_equal(codes.cpu().numpy(), c.codes[n])

    r = [rng.randn(64) for _ in range(4)]
    r[0][5], r[1][0] = np.inf, np.nan
    r[2] *= 0
    r[3] *= 1e-37
    step([0, 3, 0, 0], r)
    r = [rng.randn(64) for _ in range(4)]
    r[2] *= 1e-30
    r[3] *= 1e38
    step([1, 4, 1, 1], r)                    # the first two stay without values
    assert np.isnan(c.scales["k"][0, 0]) and np.isnan(c.scales["v"][1, 0])
    step([0, 0, 2, 2], [rng.randn(64) for _ in range(4)])      # begun anew
    assert np.isfinite(c.scales["k"]).all()


def test_append_skips_and_bounds(gpu):
    """Skipped sequences, entries that name no page, tokens past the table: nothing else changes, queries are done all the same."""
    rng = np.random.RandomState(7)
    table = np.array([[0, 1], [2, 3], [8, 4], [-1, 5], [6, 2 ** 31 - 1], [-2 ** 31, 7]], np.int32)
    positions = [-1, 1 << 62, 30, 30, 60, 2 ** 40]
    c = eb.Cache(rng, 8, 32, 2, 64, table)
    d = Device(gpu, c)
    x = rng.randn(6 * 5, 6 * 64).astype(np.float32)
    xt, pos = _dev(x), _dev(np.array(positions, np.int64))
    q, k = torch.full((30, 128), 4.0, device="cuda"), torch.full((30, 128), 4.0, device="cuda")
    d.cache.append(pos.data_ptr(), 5, q_heads=2, q=xt.data_ptr(), k=xt.data_ptr() + 512, v=xt.data_ptr() + 1024,
                   q_stride=384, k_stride=384, v_stride=384, q_out=q.data_ptr(), k_out=k.data_ptr(), stream_ptr=_stream())
    stored = np.zeros((6, 5), bool)
    for b in (2, 3, 4, 5):
        for n, lo in (("k", 128), ("v", 256)):
            c.append(n, b, positions[b], x[b * 5:b * 5 + 5, lo:lo + 128].reshape(5, 2, 64))
        stored[b] = [c.page_of(b, positions[b] + j) >= 0 for j in range(5)]
    assert stored.sum() == 3 + 3 + 0 and not stored[4].any()
    for n, codes, scales in (("k", d.k, d.ks), ("v", d.v, d.vs)):
        np.testing.assert_array_equal(codes.cpu().numpy(), c.codes[n])
        np.testing.assert_array_equal(scales.cpu().numpy(), c.scales[n])
    assert (q[:10] == 4.0).all() and torch.equal(q[10:], xt[10:, :128])
    assert ((k != 4.0).any(1).cpu().numpy() == stored.reshape(-1)).all()


# -------------------------------------------------------------------- attention

ATTENTIONS = [
    # kind, page, heads, head dim, positions, tokens, window, pad, scale
    ("f32", 32, (2, 2), 64, [0], 1, 0, 0, None),
    ("bf16", 64, (4, 1), 128, [0, 1, 31, 32, 63, 64, 200], 1, 0, 0, None),
    ("f16", 32, (3, 3), 128, [5, 77], 2, 0, 3, None),
    ("f32", 64, (16, 2), 64, [100, 3], 3, 0, 0, None),
    ("bf16", 32, (8, 1), 64, [0, 50], 24, 0, 0, -0.3),
    ("f32", 32, (20, 1), 128, [40], 5, 0, 1, 0.05),
    ("f16", 64, (4, 2), 64, [500, 1000], 1, 100, 0, None),
    ("bf16", 64, (2, 1), 128, [300], 70, 33, 0, None),
    ("f32", 32, (4, 4), 64, [255, 256, 257], 4, 1, 0, None),
    ("f16", 32, (17, 1), 64, [31], 65, 0, 0, 0.0),
    ("f32", 64, (8, 8), 128, [5000, 12], 1, 0, 0, None),
    ("bf16", 32, (8, 2), 128, [9000, 4000], 1, 0, 0, None),
    ("f16", 64, (32, 4), 64, [3000], 16, 777, 0, None),
]


def _attend_all(c, q, positions, tokens, share, window, scale, kind):
    """The oracle's outputs and bounds [rows, heads, hd], and whether a row sees anything."""
    batch, (rows, hq, hd) = len(positions), q.shape
    y, bound = np.zeros(q.shape), np.zeros(q.shape)
    for b in range(batch):
        lo = max(0, positions[b] - window + 1) if window else 0
        hi = positions[b] + tokens
        for h in range(hq // share):
            (k, there), (v, _) = (c.values(n, b, lo, hi, h) for n in "kv")
            for j in range(tokens):
                i = positions[b] + j
                first = max(0, i - window + 1) if window else 0
                see = there[first - lo:i + 1 - lo]
                if not see.any():
                    continue
                for g in range(share):
                    r = (b * tokens + j, h * share + g)
                    with np.errstate(all="ignore"):
                        y[r], bound[r] = eb.attend(q[r], k[first - lo:i + 1 - lo][see], v[first - lo:i + 1 - lo][see], scale,
                                                   kind)
    return y, bound


def _attention(gpu, d, pos, tokens, kind, q, hq, window=0, scale=None, pad=0, longest=0, stream=None):
    out = torch.full_like(q, 8.0)
    d.cache.attention(pos.data_ptr(), tokens, type=_dz_type(gpu, kind), q_heads=hq, q=q.data_ptr(), out=out.data_ptr(),
                      q_stride=q.shape[1], out_stride=out.shape[1], scale=scale, window=window, longest=longest,
                      stream_ptr=_stream() if stream is None else stream)
    return out


@pytest.mark.parametrize("kind,page,heads,hd,positions,tokens,window,pad,scale", ATTENTIONS)
def test_attention(gpu, kind, page, heads, hd, positions, tokens, window, pad, scale):
    (hq, hk), batch = heads, len(positions)
    rng = np.random.RandomState(hq + hd + tokens)
    per = (max(positions) + tokens - 1) // page + 1
    c = eb.Cache(rng, batch * per + 1, page, hk, hd, _table(rng, batch, per, batch * per + 1))
    d = Device(gpu, c)
    qt, qv = _typed(rng.randn(batch * tokens, hq * hd + pad) * np.exp(rng.randn(batch * tokens, 1)), kind)
    pos = _dev(np.array(positions, np.int64))
    s = hd ** -0.5 if scale is None else float(np.float32(scale))
    y, bound = _attend_all(c, qv[:, :hq * hd].reshape(-1, hq, hd), positions, tokens, hq // hk, window, s, kind)
    for longest in (0, 1, max(positions) + tokens):
        out = _attention(gpu, d, pos, tokens, kind, qt, hq, window, scale, longest=longest)
        err = np.abs(_np(out[:, :hq * hd]).reshape(y.shape) - y) - 1.01 * eb.rounding(y, kind)
        assert (err <= bound).all(), (longest, (err / np.maximum(bound, 1e-300)).max())
        assert (out[:, hq * hd:] == 8.0).all()


@pytest.mark.parametrize("kind", list(TYPES))
def test_attention_pages(gpu, kind):
    """Pages that two sequences share, entries that name no page, a sequence without any, tokens past the table."""
    rng = np.random.RandomState(8)
    table = np.array([[0, 1, 2], [0, 1, 3], [-1, 4, -7], [9, 10, 2 ** 31 - 1], [5, 99, 6], [0, 1, 2]], np.int32)
    positions, tokens, hq, hk, hd = [70, 90, 80, 60, 85, 200], 3, 4, 2, 64
    c = eb.Cache(rng, 8, 32, hk, hd, table)
    d = Device(gpu, c)
    qt, qv = _typed(rng.randn(18, hq * hd), kind)
    pos = _dev(np.array(positions, np.int64))
    for window in (0, 20, 1000):
        out = _np(_attention(gpu, d, pos, tokens, kind, qt, hq, window)).reshape(18, hq, hd)
        y, bound = _attend_all(c, qv.reshape(18, hq, hd), positions, tokens, 2, window, hd ** -0.5, kind)
        assert (np.abs(out - y) <= bound + 1.01 * eb.rounding(y, kind)).all()
        assert (out[9:12] == 0).all()        # a sequence of which no page is there
        if window == 20:
            assert (out[15:] == 0).all()     # a window past the table


MANY = [
    # kind, page, heads, head dim, positions, tokens, window, pad, scale
    ("f16", 64, (1, 1), 64, [0], 128, 0, 0, None),
    ("bf16", 64, (2, 2), 128, [0, 37], 128, 0, 0, None),
    ("f32", 32, (4, 1), 64, [3, 90], 33, 0, 0, None),
    ("f16", 32, (4, 2), 128, [200], 65, 0, 3, None),
    ("f32", 64, (8, 2), 128, [1000, 17, 640], 40, 0, 0, -0.2),
    ("bf16", 32, (16, 1), 64, [700], 24, 130, 0, None),
    ("f16", 64, (6, 3), 64, [2500, 1], 150, 31, 1, None),
    ("f32", 32, (1, 1), 128, [0], 300, 0, 0, 0.0),
    ("f16", 64, (64, 1), 64, [6000], 1, 0, 0, None),
    ("bf16", 64, (32, 2), 128, [3000, 0, 9], 4, 5, 0, None),
    ("f32", 64, (12, 1), 64, [1500], 64, 777, 0, None),
]


@pytest.mark.parametrize("kind,page,heads,hd,positions,tokens,window,pad,scale", MANY)
def test_attention_of_many_queries(gpu, kind, page, heads, hd, positions, tokens, window, pad, scale):
    """Blocks of 128 pairs, whole and ragged, of few tiles and of many, with and without a cluster."""
    test_attention(gpu, kind, page, heads, hd, positions, tokens, window, pad, scale)


@pytest.mark.parametrize("kind", list(TYPES))
def test_pages_of_many_queries(gpu, kind):
    """What test_attention_pages has, with 72 queries to a key head: shared pages, entries that name none, tokens past the table."""
    rng = np.random.RandomState(18)
    table = np.array([[0, 1, 2, 3, 4, 5], [0, 1, 3, -1, 6, 7], [-1, 4, -7, 2, 99, 5], [9, 10, 2 ** 31 - 1, -1, -1, -1],
                      [5, 99, 6, 0, 1, 2], [0, 1, 2, 3, 4, 5], [6, 7, 0, 1, 2, 3]], np.int32)
    positions, tokens, hq, hk, hd = [70, 90, 180, 60, 130, 300, -1], 9, 16, 2, 64
    c = eb.Cache(rng, 8, 32, hk, hd, table)
    d = Device(gpu, c)
    qt, qv = _typed(rng.randn(7 * tokens, hq * hd), kind)
    pos = _dev(np.array(positions, np.int64))
    positions[6] = 0
    for window in (0, 20, 100, 1 << 40):
        out = _np(_attention(gpu, d, pos, tokens, kind, qt, hq, window)).reshape(-1, hq, hd)
        y, bound = _attend_all(c, qv.reshape(-1, hq, hd), positions, tokens, 8, window, hd ** -0.5, kind)
        err = np.abs(out - y) - 1.01 * eb.rounding(y, kind)
        assert (err <= bound)[:6 * tokens].all()
        assert (out[3 * tokens:4 * tokens] == 0).all() and (out[6 * tokens:] == 8.0).all()
        if window in (20, 100):
            assert (out[5 * tokens:6 * tokens] == 0).all()       # a window past the table


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("hd,page", [(64, 32), (128, 64)])
def test_nan_of_many_queries(gpu, kind, hd, page):
    """A NaN scale counts where a token of its page is seen, whatever its weight, and nowhere else; so do queries that are not finite."""
    rng = np.random.RandomState(20)
    share, tokens = 3, 2 * page
    c = eb.Cache(rng, 24, page, 1, hd, np.arange(24).reshape(3, 8))
    c.scales["v"][2] = np.nan                # sequence 0, tokens of its third page
    c.scales["k"][8 + 3] = np.nan            # sequence 1, of its fourth
    d = Device(gpu, c)
    q = rng.randn(3 * tokens, share, hd)
    q[2 * tokens + 2, 1, 3], q[2 * tokens + 5, 0, 60], q[2 * tokens + 6, 2, 7] = np.inf, np.nan, -np.inf
    qt, _ = _typed(q.reshape(-1, share * hd), kind)
    first = [page + 5, 2 * page + 1, page]
    pos = _dev(np.array(first, np.int64))
    for window in (0, page // 2):
        out = _np(_attention(gpu, d, pos, tokens, kind, qt, share, window)).reshape(3, tokens, share, hd)
        bad = np.isnan(out).all(-1)
        assert (np.isnan(out).any(-1) == bad).all()
        want = np.zeros(bad.shape, bool)
        for b, at in ((0, 2), (1, 3)):
            p = first[b] + np.arange(tokens)
            want[b] = ((p >= at * page) & ((p - window + 1 < (at + 1) * page) if window else True))[:, None]
        for t, h in ((2, 1), (5, 0), (6, 2)):
            want[2, t, h] = True
        np.testing.assert_array_equal(bad, want)


@pytest.mark.parametrize("kind", list(TYPES))
def test_small_beside_large_of_many_queries(gpu, kind):
    """Elements, scales of either sign and weights beside much larger ones, in pages of 32 that share a thread's tokens."""
    rng = np.random.RandomState(21)
    hd, tokens = 64, 80
    c = eb.Cache(rng, 16, 32, 1, hd, np.arange(16).reshape(2, 8))
    c.scales["v"][2] *= 2.0 ** 12
    c.scales["v"][5] *= -1
    c.scales["v"][10] = 0
    c.scales["k"][1] *= -0.5
    c.scales["k"][12] *= 2.0 ** -20
    c.scales["k"][13] = 0
    d = Device(gpu, c)
    q = rng.randn(2 * tokens, hd)
    q[:40, :32] *= 2.0 ** -10
    q[100:, 5] *= 100
    if kind != "f16":
        q[50:60] *= 2.0 ** -60
    qt, qv = _typed(q, kind)
    positions = [170, 100]
    for scale in (0.1, -0.05):
        out = _np(_attention(gpu, d, _dev(np.array(positions, np.int64)), tokens, kind, qt, 1, scale=scale)).reshape(-1, 1, hd)
        y, bound = _attend_all(c, qv.reshape(-1, 1, hd), positions, tokens, 1, 0, float(np.float32(scale)), kind)
        assert (np.abs(out - y) <= bound + 1.01 * eb.rounding(y, kind)).all()


def test_attention_skips(gpu):
    rng = np.random.RandomState(9)
    c = eb.Cache(rng, 8, 32, 1, 128, [[0, 1], [2, 3], [4, 5]])
    d = Device(gpu, c)
    q = torch.randn(6, 128, device="cuda")
    out = _attention(gpu, d, _dev(np.array([-5, 3, 1 << 62], np.int64)), 2, "f32", q, 1)
    assert (out[:2] == 8.0).all() and (out[4:] == 8.0).all() and (out[2:4] != 8.0).any()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_attention_nan(gpu, kind):
    """A NaN scale counts where a token of its page is seen, and nowhere else; queries that are not finite read NaN."""
    rng = np.random.RandomState(10)
    hd, page = 64, 32
    c = eb.Cache(rng, 12, page, 1, hd, np.arange(12).reshape(3, 4))
    c.scales["v"][1] = np.nan                # sequence 0, tokens 32..63
    c.scales["k"][6] = np.nan                # sequence 1, tokens 64..95
    d = Device(gpu, c)
    positions, tokens = [28, 60, 100], 8
    q = rng.randn(24, hd)
    q[16 + 2, 3], q[16 + 5, 60], q[16 + 6, 7] = np.inf, np.nan, -np.inf
    qt, _ = _typed(q, kind)
    out = _np(_attention(gpu, d, _dev(np.array(positions, np.int64)), tokens, kind, qt, 1))
    bad = np.isnan(out).all(1)
    assert (np.isnan(out).any(1) == bad).all()
    want = np.zeros(24, bool)
    want[4:8] = True                         # from position 32 on
    want[8 + 4:16] = True                    # from position 64 on
    want[[18, 21, 22]] = True
    np.testing.assert_array_equal(bad, want)
    # a window that has passed the page, and one that ends before it
    out = _np(_attention(gpu, d, _dev(np.array([90, 100, 100], np.int64)), 1, kind, qt[:3].contiguous(), 1, window=27))
    np.testing.assert_array_equal(np.isnan(out).all(1), [False, True, False])
    # a value without weight: the marked page's keys score far below the rest
    c.codes["k"][:] = 1
    c.codes["k"][1] = -127
    c.scales["k"][:] = 100.0
    d = Device(gpu, c)
    qt, _ = _typed(np.ones((3, hd)), kind)
    out = _np(_attention(gpu, d, _dev(np.array([100, 20, 20], np.int64)), 1, kind, qt, 1))
    np.testing.assert_array_equal(np.isnan(out).all(1), [True, False, False])


@pytest.mark.parametrize("kind", list(TYPES))
def test_attention_small_beside_large(gpu, kind):
    """Elements, scales and weights beside much larger ones keep the precision that is promised; scales of either sign."""
    rng = np.random.RandomState(11)
    hd, hq = 128, 2
    c = eb.Cache(rng, 8, 64, 1, hd, np.arange(8).reshape(2, 4))
    c.scales["v"][2] *= 2.0 ** 12
    c.scales["v"][5] *= -1
    c.scales["k"][1] *= -0.5
    c.scales["k"][6] *= 2.0 ** -20
    d = Device(gpu, c)
    q = rng.randn(2, hq * hd)
    q[0, :64] *= 2.0 ** -10
    q[1, 5] *= 100
    if kind != "f16":
        q[1] *= 2.0 ** -60
    qt, qv = _typed(q, kind)
    scale = [0.1, 0.1 if kind == "f16" else 0.1 * 2.0 ** 60]
    for b in range(2):
        s = float(np.float32(scale[b]))
        pos = np.array([-1, -1])
        pos[b] = 250
        out = _np(_attention(gpu, d, _dev(pos.astype(np.int64)), 1, kind, qt, hq, scale=s))[b].reshape(hq, hd)
        k, v = c.values("k", b, 0, 251, 0)[0], c.values("v", b, 0, 251, 0)[0]
        for h in range(hq):
            y, bound = eb.attend(qv[b].reshape(hq, hd)[h], k, v, s, kind)
            assert (np.abs(out[h] - y) <= bound + 1.01 * eb.rounding(y, kind)).all()


def test_offsets_past_32_bits(gpu):
    """Pages beyond 2^31 elements of a pool, appended to and read."""
    rng = np.random.RandomState(12)
    page, hk, hd, pages = 64, 8, 128, 40000                     # 2.6e9 codes
    table = np.array([[39999, 0, 33000]], np.int32)
    k = torch.zeros(pages, hk, page, hd, dtype=torch.int8, device="cuda")
    v = torch.zeros_like(k)
    ks, vs = torch.ones(pages, hk, device="cuda"), torch.ones(pages, hk, device="cuda")
    tt, pos = _dev(table), torch.tensor([10], device="cuda")
    cache = gpu.KV8Cache(k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), pages, page, hk, hd, tt.data_ptr(), 1, 3)
    c = eb.Cache(rng, 3, page, hk, hd, [[0, 1, 2]])
    for n in "kv":
        c.codes[n][:] = 0
        c.scales[n][:] = 1
    x = rng.randn(150, 2, hk, hd).astype(np.float32)
    xt = _dev(x)
    cache.append(pos.data_ptr(), 150, k=xt.data_ptr(), v=xt.data_ptr() + hk * hd * 4, k_stride=2 * hk * hd,
                 v_stride=2 * hk * hd, stream_ptr=_stream())
    for i, n in enumerate("kv"):
        c.append(n, 0, 10, x[:, i])
        got = (k, v)[i][table[0].tolist()].cpu().numpy()
        np.testing.assert_array_equal(got, c.codes[n])
        assert int((k, v)[i].abs().sum(dtype=torch.int64)) == int(np.abs(got.astype(np.int64)).sum())
    q = torch.randn(1, 16 * hd, device="cuda")
    out = torch.empty_like(q)
    last = torch.tensor([159], device="cuda")
    cache.attention(last.data_ptr(), 1, q_heads=16, q=q.data_ptr(), out=out.data_ptr(), stream_ptr=_stream())
    y, bound = _attend_all(c, _np(q).reshape(1, 16, hd), [159], 1, 2, 0, hd ** -0.5, "f32")
    assert (np.abs(_np(out).reshape(1, 16, hd) - y) <= bound + eb.rounding(y, "f32")).all()
    # a product whose output passes 2^31 elements
    m, n = 70000, 32768
    w = gpu.QuantizedWeightMatrix(np.full(n, 0.5, np.float32), np.full(n * 16, 128, np.uint8), 16, n, 8)
    a = torch.randint(-127, 128, (m, 16), dtype=torch.int8, device="cuda")
    s = torch.ones(m, device="cuda")
    y = torch.empty(m, n, dtype=torch.bfloat16, device="cuda")
    w.matmul_q8_async(a.data_ptr(), s.data_ptr(), y.data_ptr(), m, _stream(), type=gpu.TYPE_BF16)
    want = (a.sum(1, dtype=torch.int32).float() * 0.5).bfloat16()
    for at in (0, 1, 777, n - 1):
        assert torch.equal(y[:, at], want)
    assert torch.equal(y[m - 1], want[m - 1].expand(n))
    w.close()


# ---------------------------------------------------------------- a run of them

def _layer(gpu, seed, kind, batch, hq, hk, hd, page, per, stream):
    """Weights, cache and buffers of one attention block, and its step as a function."""
    torch.manual_seed(seed)
    rng = np.random.RandomState(seed)
    d_model, t, dt = hq * hd, _dz_type(gpu, kind), TYPES[kind]
    qkv = gpu.QuantizedWeightMatrix.encode((rng.randn(d_model, (hq + 2 * hk) * hd) * 0.05).astype(np.float32), 8)
    wo = gpu.QuantizedWeightMatrix.encode((rng.randn(hq * hd, d_model) * 0.05).astype(np.float32), 8)
    c = eb.Cache(rng, batch * per, page, hk, hd, _table(rng, batch, per, batch * per))
    d = Device(gpu, c)
    gains = [(1 + 0.1 * torch.randn(n, device="cuda")) for n in (d_model, hd, hd)]
    s = dict(x=torch.randn(batch, d_model, device="cuda").to(dt), delta=torch.randn(batch, d_model, device="cuda").to(dt),
             h=torch.empty(batch, d_model, dtype=dt, device="cuda"),
             codes=torch.empty(batch, d_model, dtype=torch.int8, device="cuda"), scales=torch.empty(batch, device="cuda"),
             row=torch.empty(batch, (hq + 2 * hk) * hd, dtype=dt, device="cuda"),
             q=torch.empty(batch, hq * hd, dtype=dt, device="cuda"), o=torch.empty(batch, hq * hd, dtype=dt, device="cuda"),
             codes2=torch.empty(batch, hq * hd, dtype=torch.int8, device="cuda"), scales2=torch.empty(batch, device="cuda"),
             y=torch.empty(batch, d_model, dtype=dt, device="cuda"),
             pos=torch.tensor([3 * b for b in range(batch)], device="cuda"))

    def step():
        st = stream.cuda_stream
        size, at, w = s["row"].element_size(), s["row"].data_ptr(), s["row"].shape[1]
        gpu.norm_q8(batch, d_model, type=t, x=s["x"].data_ptr(), residual=s["delta"].data_ptr(), sum_out=s["h"].data_ptr(),
                    gain=gains[0].data_ptr(), codes=s["codes"].data_ptr(), codes_stride=d_model,
                    scales=s["scales"].data_ptr(), stream_ptr=st)
        qkv.matmul_q8_async(s["codes"].data_ptr(), s["scales"].data_ptr(), at, batch, st, type=t)
        d.cache.append(s["pos"].data_ptr(), 1, type=t, q_heads=hq, q=at, k=at + hq * hd * size,
                       v=at + (hq + hk) * hd * size, q_stride=w, k_stride=w, v_stride=w, q_out=s["q"].data_ptr(),
                       q_gain=gains[1].data_ptr(), k_gain=gains[2].data_ptr(), rope_base=10000.0, stream_ptr=st)
        d.cache.attention(s["pos"].data_ptr(), 1, type=t, q_heads=hq, q=s["q"].data_ptr(), out=s["o"].data_ptr(),
                          stream_ptr=st)
        gpu.norm_q8(batch, hq * hd, type=t, x=s["o"].data_ptr(), norm=False, codes=s["codes2"].data_ptr(),
                    codes_stride=hq * hd, scales=s["scales2"].data_ptr(), stream_ptr=st)
        wo.matmul_q8_async(s["codes2"].data_ptr(), s["scales2"].data_ptr(), s["y"].data_ptr(), batch, st, type=t)
    return s, c, d, (qkv, wo, gains), step


@pytest.mark.parametrize("kind,hq,hk,hd,page", [("f32", 4, 4, 64, 32), ("bf16", 8, 2, 128, 64)])
def test_a_decode_step_of_the_four(gpu, kind, hq, hk, hd, page):
    """Each operator's result against its formula on what the one before left, eagerly over several steps."""
    batch, per = 5, 3
    s, c, d, (qkv, wo, gains), step = _layer(gpu, 20, kind, batch, hq, hk, hd, page, per, torch.cuda.current_stream())
    w, size = {n: m.unpack() for n, m in (("qkv", qkv), ("wo", wo))}, hq * hd
    for turn in range(4):
        for n, codes, scales in (("k", d.k, d.ks), ("v", d.v, d.vs)):
            c.codes[n], c.scales[n] = codes.cpu().numpy().copy(), scales.cpu().numpy().copy()
        step()
        torch.cuda.synchronize()
        h = (s["x"].float() + s["delta"].float()).to(TYPES[kind])
        assert torch.equal(s["h"], h)
        want, scale = eb.norm_rows(_np(h), gains[0].cpu().numpy(), True, 1e-6)
        np.testing.assert_array_equal(s["codes"].cpu().numpy(), want)
        assert (np.abs(_np(s["scales"]) - scale) <= eb.NORM_SCALE * scale).all()
        for name, codes, scales, out in (("qkv", "codes", "scales", "row"), ("wo", "codes2", "scales2", "y")):
            # unpacked values are level x scale rounded once: u of each product's size in all
            a = _np(s[codes]) * _np(s[scales])[:, None]
            ref = a @ w[name].astype(np.float64)
            bound = 6 * eb.U * (np.abs(a) @ np.abs(w[name].astype(np.float64))) + 1.01 * eb.rounding(ref, kind)
            assert (np.abs(_np(s[out]) - ref) <= bound).all()
        positions = s["pos"].tolist()
        row = _np(s["row"]).reshape(batch, hq + 2 * hk, hd)
        q, mag = eb.norm_rotate(row[:, :hq], gains[1].cpu().numpy(), 1e-6, np.array(positions), 10000.0, False)
        assert (np.abs(_np(s["q"]).reshape(q.shape) - q) <= 24 * eb.U * mag + 1.01 * eb.rounding(q, kind)).all()
        for b in range(batch):
            c.append("v", b, positions[b], row[b:b + 1, hq + hk:].astype(np.float32))
        np.testing.assert_array_equal(d.v.cpu().numpy(), c.codes["v"])
        c.codes["k"], c.scales["k"] = d.k.cpu().numpy(), d.ks.cpu().numpy()
        y, bound = _attend_all(c, _np(s["q"]).reshape(batch, hq, hd), positions, 1, hq // hk, 0, hd ** -0.5, kind)
        assert (np.abs(_np(s["o"]).reshape(y.shape) - y) <= bound + 1.01 * eb.rounding(y, kind)).all()
        want, scale = eb.norm_rows(_np(s["o"]), None, False, 0)
        np.testing.assert_array_equal(s["codes2"].cpu().numpy(), want)
        s["pos"] += 1
        s["x"], s["delta"] = s["h"].clone(), s["y"].clone()
    qkv.close()
    wo.close()


def test_captured_steps_on_two_streams(gpu):
    """Two layers' steps captured on streams of their own, replayed side by side, give what eager steps give."""
    layers, graphs = [], []
    for i in range(2):
        stream = torch.cuda.Stream()
        layers.append((stream, _layer(gpu, 30 + i, "bf16", 7, 8, 2, 128, 64, 4, stream),
                       _layer(gpu, 30 + i, "bf16", 7, 8, 2, 128, 64, 4, torch.cuda.current_stream())))
    torch.cuda.synchronize()
    for stream, (s, _, _, _, step), _ in layers:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step()
            s["pos"] += 1
        graphs.append(graph)
    for turn in range(20):
        for (stream, _, _), graph in zip(layers, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for _, (s, _, d, _, _), (eager, _, d2, _, step) in layers:
        for turn in range(20):
            step()
            eager["pos"] += 1
        torch.cuda.synchronize()
        for name in ("h", "codes", "scales", "row", "q", "o", "y"):
            assert torch.equal(s[name], eager[name]), name
        assert torch.equal(d.k, d2.k) and torch.equal(d.v, d2.v) and torch.equal(d.ks, d2.ks) and torch.equal(d.vs, d2.vs)


def test_products_and_many_queries_side_by_side(gpu):
    """Kernels with tensor memory one after another on two streams: every turn gives what the first one gives."""
    lanes = []
    for seed in range(2):
        rng = np.random.RandomState(40 + seed)
        hd, hq, hk, tokens, page = (64, 8, 1, 16, 32) if seed else (128, 16, 2, 16, 64)
        c = eb.Cache(rng, 40, page, hk, hd, np.arange(40).reshape(2, 20))
        d = Device(gpu, c)
        k, m = 256, 2 * tokens
        w = [_quantized(gpu, rng.randint(-127, 128, (a, b)).astype(np.int8), np.full(b, 1e-4, np.float32))
             for a, b in ((k, hq * hd), (hq * hd, k))]
        lanes.append(dict(d=d, w=w, hq=hq, tokens=tokens, m=m, k=k, x=torch.randn(m, k, device="cuda").bfloat16(),
                          codes=torch.empty(m, hq * hd, dtype=torch.int8, device="cuda"), scales=torch.empty(m, device="cuda"),
                          q=torch.empty(m, hq * hd, dtype=torch.bfloat16, device="cuda"),
                          o=torch.empty(m, hq * hd, dtype=torch.bfloat16, device="cuda"),
                          pos=_dev(np.array([300, 500], np.int64)), stream=torch.cuda.Stream(), outs=[]))
    torch.cuda.synchronize()

    def turn(s):
        st, t = s["stream"].cuda_stream, gpu.TYPE_BF16
        y = torch.empty(s["m"], s["k"], dtype=torch.bfloat16, device="cuda")
        width = s["hq"] * s["d"].cache.head_dim
        gpu.norm_q8(s["m"], s["k"], type=t, x=s["x"].data_ptr(), codes=s["codes"].data_ptr(), scales=s["scales"].data_ptr(), stream_ptr=st)
        s["w"][0].matmul_q8_async(s["codes"].data_ptr(), s["scales"].data_ptr(), s["q"].data_ptr(), s["m"], st, type=t)
        s["d"].cache.attention(s["pos"].data_ptr(), s["tokens"], type=t, q_heads=s["hq"], q=s["q"].data_ptr(), out=s["o"].data_ptr(),
                               stream_ptr=st)
        gpu.norm_q8(s["m"], width, type=t, x=s["o"].data_ptr(), norm=False, codes=s["codes"].data_ptr(),
                    scales=s["scales"].data_ptr(), stream_ptr=st)
        s["w"][1].matmul_q8_async(s["codes"].data_ptr(), s["scales"].data_ptr(), y.data_ptr(), s["m"], st, type=t)
        s["outs"].append(y)
    for _ in range(40):
        for s in lanes:
            with torch.cuda.stream(s["stream"]):
                turn(s)
    torch.cuda.synchronize()
    for s in lanes:
        assert bool(s["outs"][0].isfinite().all()) and float(s["outs"][0].abs().max()) > 0
        assert all(torch.equal(s["outs"][0], y) for y in s["outs"])
        for w in s["w"]:
            w.close()
