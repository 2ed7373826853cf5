"""The 4-bit operators on the device against their 64-bit formulas
(tests/_fourbit.py): group-scaled products, the norm + rotation + append pass,
attention over the 4-bit ring with windows and sinks, and a run of them."""
import numpy as np
import pytest
import torch

import _fourbit as fb

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


def _stream():
    return torch.cuda.current_stream().cuda_stream


# ------------------------------------------------------------------ products

SHAPES = [(1, 1, 1), (1, 31, 3), (2, 32, 16), (3, 128, 17), (1, 129, 33), (5, 100, 77), (8, 1000, 130), (9, 4099, 40),
          (16, 257, 1003), (17, 640, 48), (33, 384, 100), (1, 4096, 4096), (2, 8192, 512), (16, 2048, 2048),
          (4, 16384, 64), (16, 12000, 80), (2, 70, 90001), (1, 100000, 40)]


@pytest.mark.parametrize("m,k,n", SHAPES)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("half_scales", [False, True])
def test_products(gpu, m, k, n, group, half_scales):
    rng = np.random.RandomState(m * 7 + k + n)
    w = (rng.randn(k, n) * 0.05 * np.exp(rng.randn(k, 1))).astype(np.float32)
    w[:, n // 2] = 0
    s, p = gpu.quantize_pack_grouped(w, group)
    if half_scales:
        s = s.astype(np.float16)
    q = gpu.GroupedWeightMatrix(s, p, k, n, group)
    values = fb.dequant(s, p, k, n, group)
    np.testing.assert_array_equal(q.unpack(), values.astype(np.float32))
    x = rng.randn(m, k) * np.exp(rng.randn(k))
    for kind in TYPES:
        xt, xv = _typed(x, kind)
        y = torch.full((m, n), 7.0, dtype=TYPES[kind], device="cuda")
        q.matmul_async(xt.data_ptr(), y.data_ptr(), m, _stream(), type=_dz_type(gpu, kind))
        ref, bound = fb.product(xv, values, kind)
        err = np.abs(_np(y) - ref) - fb.rounding(ref, kind)
        assert (err <= bound).all(), (kind, err.max(), (err / np.maximum(bound, 1e-30)).max())
    np.testing.assert_array_equal(q.matmul(x.astype(np.float32)).shape, (m, n))
    q.close()


def test_product_rows_do_not_depend_on_each_other(gpu):
    """A row's result is the same alone and among others, strided or not, and in every repetition."""
    rng = np.random.RandomState(1)
    k, n, m = 1111, 210, 16
    q = gpu.GroupedWeightMatrix.encode(rng.randn(k, n), 64)
    x = torch.randn(m, k + 5, device="cuda")
    y = torch.full((m, n + 3), 5.0, device="cuda")
    q.matmul_async(x.data_ptr(), y.data_ptr(), m, _stream(), lda=k + 5, ldc=n + 3)
    again = torch.empty_like(y)
    again.fill_(5.0)
    q.matmul_async(x.data_ptr(), again.data_ptr(), m, _stream(), lda=k + 5, ldc=n + 3)
    assert torch.equal(y, again) and (y[:, n:] == 5.0).all()
    ref, bound = fb.product(_np(x[:, :k]), _np(torch.from_numpy(q.unpack())))
    for r in range(m):
        one = torch.empty(1, n, device="cuda")
        q.matmul_async(x[r].data_ptr(), one.data_ptr(), 1, _stream())
        assert (np.abs(_np(one[0]) - ref[r]) <= bound[r] + fb.rounding(ref[r], "f32")).all()
    q.close()


def test_product_special_values(gpu):
    rng = np.random.RandomState(2)
    k, n = 700, 50
    q = gpu.GroupedWeightMatrix.encode(rng.randn(k, n) * 0.1, 32)
    w = q.unpack().astype(np.float64)
    x = rng.randn(8, k).astype(np.float32)
    x[0] = 0
    x[1, 5] = np.inf
    x[2, 699] = np.nan
    x[3] *= 1e30
    x[4] *= 1e-30
    x[5, :] = 0
    x[5, 300] = -2.0 ** 100
    x[6, ::2] *= 2.0 ** 40
    y = q.matmul(x)
    ref, bound = fb.product(np.nan_to_num(x, posinf=0), w)
    assert (y[0] == 0).all() and np.isnan(y[1]).all() and np.isnan(y[2]).all()
    for r in (3, 4, 5, 6, 7):
        assert (np.abs(y[r] - ref[r]) <= bound[r] + fb.rounding(ref[r], "f32")).all(), r
    q.close()


def test_product_offsets_past_32_bits(gpu):
    """Five gigabytes of records: rows and columns at both ends, some of each against the formula."""
    k, n, group, m = 65536, 150016, 128, 3
    g = torch.Generator("cuda").manual_seed(4)
    low = torch.randint(0, 15, (k, n // 2), dtype=torch.uint8, device="cuda", generator=g)
    packed = low.mul_(16).add_(torch.randint(0, 15, (k, n // 2), dtype=torch.uint8, device="cuda", generator=g))
    scales = torch.rand(k // group, n, device="cuda", generator=g) * 0.01
    q = gpu.GroupedWeightMatrix.from_device(scales.data_ptr(), packed.data_ptr(), k, n, group)
    assert q.nbytes > 1 << 32
    x = torch.randn(m, k, device="cuda", generator=g)
    y = torch.empty(m, n, device="cuda")
    q.matmul_async(x.data_ptr(), y.data_ptr(), m, _stream())
    torch.cuda.synchronize()
    pick = torch.cat([torch.arange(6), torch.arange(n // 2, n // 2 + 6), torch.arange(n - 6, n)]).cuda()
    byte = packed[:, pick // 2].long()
    level = torch.where(pick % 2 == 0, byte & 15, byte >> 4).double() - 7
    w = (level * scales[:, pick].double().repeat_interleave(group, 0)).cpu().numpy()
    ref, bound = fb.product(_np(x), w)
    assert (np.abs(_np(y[:, pick]) - ref) <= bound + fb.rounding(ref, "f32")).all()
    q.close()


def test_product_refusals_on_device(gpu):
    k, n = 64, 16
    q = gpu.GroupedWeightMatrix.encode(np.ones((k, n), np.float32), 32)
    x, y = torch.ones(2, k, device="cuda"), torch.empty(2, n, device="cuda")
    L, ok = gpu.lib(), gpu.TYPE_F32
    call = lambda a=x.data_ptr(), lda=k, c=y.data_ptr(), ldc=n, m=1, kk=k, t=ok: \
        L.dz_cuda_matmul_grouped_async(a, lda, q.handle, c, ldc, m, kk, t, None)  # noqa: E731
    assert call() == 0
    for bad in (dict(m=0), dict(kk=k + 1), dict(lda=k - 1), dict(ldc=n - 1), dict(t=3), dict(a=None), dict(c=None),
                dict(a=x.data_ptr() + 2), dict(m=(1 << 24) + 1)):
        assert call(**bad) == -1, bad
    s, p = gpu.quantize_pack_grouped(np.ones((k, n), np.float32), 32)
    for scale in (np.nan, np.inf, -1.0):
        t = s.copy()
        t[1, 3] = scale
        with pytest.raises(gpu.DzError):
            gpu.GroupedWeightMatrix(t, p, k, n, 32)
    p2 = p.copy()
    p2[100] = 0xF7
    with pytest.raises(gpu.DzError):
        gpu.GroupedWeightMatrix(s, p2, k, n, 32)
    torch.cuda.synchronize()
    q.close()


def test_products_on_two_streams_and_in_a_graph(gpu):
    """One matrix used on two streams at once, and captured twice: nothing is shared between calls."""
    rng = np.random.RandomState(3)
    k, n, m = 3000, 900, 5
    q = gpu.GroupedWeightMatrix.encode(rng.randn(k, n) * 0.1, 128)
    xs = [torch.randn(m, k, device="cuda") for _ in range(4)]
    want = []
    for x in xs:
        y = torch.empty(m, n, device="cuda")
        q.matmul_async(x.data_ptr(), y.data_ptr(), m, _stream())
        want.append(y)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [torch.empty(m, n, device="cuda") for _ in xs]
    for rep in range(10):
        for i, (x, y) in enumerate(zip(xs, got)):
            q.matmul_async(x.data_ptr(), y.data_ptr(), m, streams[i % 2].cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graphs = []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            q.matmul_async(xs[i].data_ptr(), got[i].data_ptr(), m, _stream())
        graphs.append(g)
    for i in range(2):
        xs[i].copy_(xs[i + 2])
        got[i].zero_()
    torch.cuda.synchronize()
    with torch.cuda.stream(streams[0]):
        graphs[0].replay()
    with torch.cuda.stream(streams[1]):
        graphs[1].replay()
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[2]) and torch.equal(got[1], want[3])
    q.close()


# -------------------------------------------------------------------- caches

class Ring:
    """A 4-bit ring cache with its device buffers; guard rows behind each show writes out of place."""

    def __init__(self, gpu, batch, heads, hd, cap, sinks=0, rng=None):
        self.batch, self.heads, self.hd, self.cap, self.sinks = batch, heads, hd, cap, sinks
        rows, rng = batch * heads * cap, rng or np.random.RandomState(0)
        self.codes, self.scales = [], []
        for _ in range(2):
            c = rng.randint(0, 15, (rows + 4, hd // 2)) | rng.randint(0, 15, (rows + 4, hd // 2)) << 4
            self.codes.append(torch.from_numpy(c.astype(np.uint8)).cuda())
            s = (0.1 + rng.rand(rows + 4, hd // 64)).astype(np.float32) / 4
            self.scales.append(torch.from_numpy(s).cuda())
        self.cache = gpu.KV4Cache(self.codes[0].data_ptr(), self.codes[1].data_ptr(), self.scales[0].data_ptr(),
                                  self.scales[1].data_ptr(), batch, heads, hd, cap, sinks)
        self.before = self.snapshot()

    def snapshot(self):
        return [(c.cpu().numpy().copy(), s.cpu().numpy().copy()) for c, s in zip(self.codes, self.scales)]

    def scale_rows(self, which, b, h, slots):
        return _np(self.scales[which])[(b * self.heads + h) * self.cap + np.asarray(slots)]

    def rows(self, which, b, h, slots):
        """Values [len(slots), hd] of the keys (0) or values (1)."""
        at = ((b * self.heads + h) * self.cap + np.asarray(slots))
        codes = self.codes[which].cpu().numpy()[at]
        scales = self.scales[which].cpu().numpy()[at].astype(np.float64)
        level = np.stack([codes & 15, codes >> 4], -1).reshape(len(slots), self.hd).astype(np.float64) - 7
        return level * scales.repeat(64, 1)


def _append(gpu, ring, kind, pos, n, hq, q, k, v, gains=(None, None), base=0.0, halves=False, outs=True, eps=1e-6,
            inplace=False):
    """Runs append on rows [batch * n] of q, k, v inside one wider buffer; returns (q_out, k_out, v_out)."""
    hk, hd, rows = ring.heads, ring.hd, ring.batch * n
    width = (hq + 2 * hk) * hd + 24
    buf = torch.full((rows, width), 3.0, dtype=TYPES[kind], device="cuda")
    cuts = np.cumsum([0, hq * hd + 8, hk * hd + 8, hk * hd + 8])
    for at, t, h in zip(cuts, (q, k, v), (hq, hk, hk)):
        buf[:, at:at + h * hd] = t.view(rows, h * hd)
    size, ptr = buf.element_size(), buf.data_ptr()
    ins = [ptr + int(c) * size for c in cuts[:3]]
    if inplace:
        targets, strides = ins, [width] * 3
        views = [buf[:, c:c + h * hd] for c, h in zip(cuts, (hq, hk, hk))]
    else:
        views = [torch.full((rows, h * hd + 4), 9.0, dtype=TYPES[kind], device="cuda") for h in (hq, hk, hk)]
        targets, strides = [t.data_ptr() for t in views], [t.shape[1] for t in views]
    g = [None if x is None else torch.from_numpy(x).cuda() for x in gains]
    ring.cache.append(
        pos.data_ptr(), n, type=_dz_type(gpu, kind), q_heads=hq, q=ins[0], k=ins[1], v=ins[2], q_stride=width,
        k_stride=width, v_stride=width, q_out=targets[0], q_out_stride=strides[0], k_out=targets[1] if outs else None,
        v_out=targets[2] if outs else None, k_out_stride=strides[1], v_out_stride=strides[2],
        q_gain=None if g[0] is None else g[0].data_ptr(), k_gain=None if g[1] is None else g[1].data_ptr(), eps=eps,
        rope_base=base, halves=halves, stream_ptr=_stream())
    torch.cuda.synchronize()
    if inplace:
        gap = torch.ones(width, dtype=torch.bool)
        for c, h in zip(cuts, (hq, hk, hk)):
            gap[c:c + h * hd] = False
        assert (buf[:, gap.cuda()] == 3.0).all()
        return views
    assert all((t[:, -4:] == 9.0).all() for t in views)
    return [t[:, :-4] for t in views]


APPENDS = [  # batch, n, hq, hk, hd, cap, sinks, first positions, norm, base, halves
    (1, 1, 1, 1, 64, 1, 0, [0], True, 1e4, False),
    (1, 1, 2, 1, 128, 5, 4, [3], True, 1e4, True),
    (3, 1, 4, 4, 128, 17, 0, [0, 16, 100], True, 1e4, False),
    (3, 5, 6, 2, 64, 9, 4, [0, 2, 77], True, 5e5, True),
    (2, 9, 3, 3, 128, 9, 0, [4, 1000003], False, 1e4, True),
    (2, 4, 0, 2, 64, 40, 33, [31, -1], True, 0.0, False),
    (4, 2, 8, 1, 128, 30, 1, [-5, 0, 29, 200000], False, 0.0, False),
    (1, 70, 16, 8, 64, 100, 7, [60], True, 1e4, False),
    (1, 3, 2, 2, 128, 64, 2, [(1 << 33) + 5], True, 0.0, True),
]


@pytest.mark.parametrize("case", APPENDS)
@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("inplace", [False, True])
def test_append(gpu, case, kind, inplace):
    batch, n, hq, hk, hd, cap, sinks, first, norm, base, halves = case
    rng = np.random.RandomState(cap + hq)
    ring = Ring(gpu, batch, hk, hd, cap, sinks, rng)
    rows = batch * n
    qt, qv = _typed(rng.randn(rows, hq, hd) * 2, kind)
    kt, kv = _typed(rng.randn(rows, hk, hd) * np.exp(rng.randn(hd)), kind)
    vt, vv = _typed(rng.randn(rows, hk, hd), kind)
    gains = [(1 + 0.3 * rng.randn(hd)).astype(np.float32) if norm else None for _ in range(2)]
    pos = torch.tensor(first, dtype=torch.int64, device="cuda")
    q, k, v = _append(gpu, ring, kind, pos, n, hq, qt, kt, vt, gains, base, halves, inplace=inplace)
    where = (np.asarray(first)[:, None] + np.arange(n)).reshape(-1)
    live = np.repeat(np.asarray(first) >= 0, n)
    after = ring.snapshot()
    touched = np.zeros(ring.before[0][1].shape[0], bool)
    yk, _ = fb.norm_rotate(kv, gains[1], 1e-6, where, base, halves)
    yq, mag = fb.norm_rotate(qv, gains[0], 1e-6, where, base, halves)
    for which, values, out in ((0, yk, k), (1, vv, v)):
        want, scales, scaled = fb.quantize_rows(values.astype(np.float32))
        out = _np(out).reshape(rows, hk, hd)
        for r in np.flatnonzero(live):
            s = fb.slot(int(where[r]), sinks, cap)
            at = (r // n * hk + np.arange(hk)) * cap + s
            touched[at] = True
            got_s = after[which][1][at]
            # fp32 of the peak of rows rounded once from 64 bits: at most one step apart
            assert (np.abs(got_s.astype(np.float64) - scales[r]) <= 2 * fb.U * scales[r]).all()
            raw = after[which][0][at]
            codes = np.stack([raw & 15, raw >> 4], -1).reshape(hk, hd).astype(np.int64)
            assert fb.codes_agree(codes, want[r], scaled[r]), (which, r)
            held = (codes - 7) * got_s.astype(np.float64).repeat(64, 1)
            assert (np.abs(out[r] - held) <= fb.rounding(held, kind)).all()
    for which in range(2):                               # slots of no new token, and the guard rows, are as they were
        for x, y in zip(ring.before[which], after[which]):
            np.testing.assert_array_equal(x[~touched], y[~touched])
    if hq:
        got = _np(q).reshape(rows, hq, hd)
        # about a dozen fp32 roundings of a norm (its sum is a tree) and three of a rotation
        assert (np.abs(got - yq)[live] <= (2.0 ** -20 * mag + fb.rounding(yq, kind))[live]).all()
        if not inplace and (~live).any():
            assert (got[~live] == 9.0).all()
    if not inplace and (~live).any():
        assert (_np(k)[~live] == 9.0).all() and (_np(v)[~live] == 9.0).all()


def test_append_poisons_only_what_holds_a_nan(gpu):
    ring = Ring(gpu, 1, 2, 128, 8)
    k = torch.randn(1, 2, 128, device="cuda")
    v = torch.randn(1, 2, 128, device="cuda")
    v[0, 0, 3], v[0, 1, 100], k[0, 1, 70] = float("nan"), float("inf"), float("-inf")
    v[0, 1, :64] = 0
    pos = torch.zeros(1, dtype=torch.int64, device="cuda")
    _append(gpu, ring, "f32", pos, 1, 0, torch.empty(1, 0, device="cuda"), k, v)
    codes, scales = zip(*ring.snapshot())
    at = np.array([0, 8])
    assert np.isnan(scales[1][at]).tolist() == [[True, False], [False, True]]
    assert np.isnan(scales[0][at]).tolist() == [[False, False], [False, True]]
    assert (codes[1][0, :32] == 0x77).all() and (codes[1][8] == 0x77).all() and scales[1][8, 0] == 0


def test_append_smallest_and_largest_values(gpu):
    ring = Ring(gpu, 1, 1, 64, 4)
    rows = torch.zeros(4, 1, 64, device="cuda")
    rows[0, 0, 5] = 2.0 ** -140
    rows[1, 0, 7] = 3e38
    rows[1, 0, 8] = -1e38
    rows[2] = 1e-30
    pos = torch.zeros(1, dtype=torch.int64, device="cuda")
    _append(gpu, ring, "f32", pos, 4, 0, torch.empty(4, 0, device="cuda"), rows, rows)
    want, scales, _ = fb.quantize_rows(rows.cpu().numpy())
    for codes, got in ring.snapshot():
        np.testing.assert_array_equal(got[:4], scales.reshape(4, 1))
        np.testing.assert_array_equal(np.stack([codes[:4] & 15, codes[:4] >> 4], -1).reshape(4, 64),
                                      want.reshape(4, 64))


# ----------------------------------------------------------------- attention

ATTENDS = [  # batch, n, hq, hk, hd, cap, sinks, window, first positions
    (1, 1, 1, 1, 64, 1, 0, 0, [0]),
    (1, 1, 1, 1, 128, 1, 0, 1, [9]),
    (2, 1, 2, 2, 64, 33, 0, 0, [0, 31]),
    (3, 1, 4, 1, 128, 31, 0, 0, [30, 31, 1000]),
    (2, 1, 8, 8, 128, 700, 0, 0, [640, 5]),
    (1, 1, 16, 1, 64, 300, 0, 0, [299]),
    (2, 1, 6, 2, 64, 77, 4, 16, [10, 5000]),
    (4, 1, 4, 4, 128, 260, 4, 256, [2, 258, 261, -1]),
    (2, 1, 3, 3, 128, 150, 149, 0, [148, 70000]),
    (2, 1, 5, 5, 64, 150, 100, 7, [50, 333]),
    (2, 5, 4, 2, 64, 64, 0, 0, [0, 59]),
    (2, 7, 9, 3, 128, 100, 3, 40, [0, 777]),
    (1, 24, 12, 1, 64, 90, 2, 64, [55]),
    (2, 33, 2, 2, 128, 80, 40, 0, [0, 61]),
    (1, 1, 7, 7, 128, 3000, 1, 0, [2999]),
    (1, 2, 2, 1, 128, 4000, 0, 1000, [(1 << 33) + 17]),
    (70, 1, 1, 1, 64, 50, 0, 0, list(range(70))),
]


def _check_attention(gpu, ring, kind, n, hq, window, first, q, scale, rows_out=None):
    hk, hd, batch = ring.heads, ring.hd, ring.batch
    qt, qv = _typed(q, kind)
    pos = torch.tensor(first, dtype=torch.int64, device="cuda")
    wide = torch.full((batch * n, hq * hd + 6), 3.0, dtype=TYPES[kind], device="cuda")
    wide[:, :hq * hd] = qt.view(batch * n, -1)
    out = torch.full((batch * n, hq * hd + 2), 9.0, dtype=TYPES[kind], device="cuda")
    ring.cache.attention(pos.data_ptr(), n, type=_dz_type(gpu, kind), q_heads=hq, q=wide.data_ptr(),
                         q_stride=wide.shape[1], out=out.data_ptr(), out_stride=out.shape[1], scale=scale,
                         window=window, stream_ptr=_stream())
    torch.cuda.synchronize()
    assert (out[:, -2:] == 9.0).all()
    got = _np(out[:, :-2]).reshape(batch, n, hq, hd)
    qv = qv.reshape(batch, n, hq, hd)
    cached = {}
    for b, f in enumerate(first):
        if f < 0:
            assert (got[b] == 9.0).all()
            continue
        for j in range(n):
            seen = fb.visible(f + j, f + n - 1, ring.sinks, ring.cap, window)
            slots = [fb.slot(p, ring.sinks, ring.cap) for p in seen]
            for h in range(hq):
                key = (b, h // (hq // hk))
                if key not in cached:
                    every = list(range(ring.cap))
                    cached[key] = ring.rows(0, *key, every), ring.rows(1, *key, every), ring.scale_rows(1, *key, every)
                k, v, s = (c[slots] for c in cached[key])
                ref, bound = fb.attend(qv[b, j, h], k, v, scale, s, kind)
                err = np.abs(got[b, j, h] - ref)
                assert (err <= bound + fb.rounding(ref, kind) + 2.0 ** -10 * fb.rounding(ref, kind)).all(), \
                    (b, j, h, (err / bound).max())
    return got


@pytest.mark.parametrize("case", ATTENDS)
@pytest.mark.parametrize("kind", sorted(TYPES))
def test_attention(gpu, case, kind):
    batch, n, hq, hk, hd, cap, sinks, window, first = case
    rng = np.random.RandomState(cap + n)
    ring = Ring(gpu, batch, hk, hd, cap, sinks, rng)
    _check_attention(gpu, ring, kind, n, hq, window, first, rng.randn(batch * n, hq, hd), hd ** -0.5)
    for old, new in zip(ring.before, ring.snapshot()):    # the cache is only read
        np.testing.assert_array_equal(old[0], new[0])
        np.testing.assert_array_equal(old[1], new[1])


@pytest.mark.parametrize("kind", sorted(TYPES))
def test_attention_with_scales_of_every_size(gpu, kind):
    """Value scales from 2^-60 to 2^20, keys that make one token win, and a first
    token that wins and holds nothing: the others must still count."""
    rng = np.random.RandomState(8)
    ring = Ring(gpu, 2, 2, 128, 400, 0, rng)
    s = ring.scales[1]
    s.copy_(torch.from_numpy(2.0 ** rng.randint(-60, 20 if kind == "f32" else 10, s.shape).astype(np.float32)))
    ring.scales[0][17] = 8.0
    _check_attention(gpu, ring, kind, 1, 4, 0, [399, 300], rng.randn(2, 4, 128), 128 ** -0.5)
    # a first token that takes nearly all weight and holds nothing: the rest decides the result
    ring = Ring(gpu, 1, 1, 64, 300, 0, rng)
    ring.scales[1][0] = 0
    ring.scales[0][0] = 4.0
    q = np.zeros((1, 1, 64))
    q[0, 0] = ring.rows(0, 0, 0, [0])[0]
    _check_attention(gpu, ring, kind, 1, 1, 0, [299], q * (12.0 / (q * q).sum() ** 0.5), 1.0)


def test_attention_ignores_what_it_does_not_see(gpu):
    """NaN scales and any codes in slots out of the window, in unwritten slots and behind the ring change nothing."""
    rng = np.random.RandomState(9)
    for cap, sinks, window, first in ((300, 4, 64, 5000), (300, 0, 0, 100), (64, 3, 10, 12), (131, 0, 100, 131)):
        ring = Ring(gpu, 1, 2, 64, cap, sinks, rng)
        q = rng.randn(1, 4, 64)
        clean = _check_attention(gpu, ring, "f32", 1, 4, window, [first], q, 0.125)
        seen = {fb.slot(p, sinks, cap) for p in fb.visible(first, first, sinks, cap, window)}
        hidden = torch.tensor([h * cap + s for h in range(2) for s in range(cap) if s not in seen], device="cuda",
                              dtype=torch.int64)
        for which in range(2):
            ring.scales[which][hidden] = float("nan")
            ring.codes[which][hidden] = 0xFF
            ring.scales[which][2 * cap:] = float("nan")
        again = _check_attention(gpu, ring, "f32", 1, 4, window, [first], q, 0.125)
        np.testing.assert_array_equal(clean, again)
        # and what it sees, it sees
        ring.scales[1][cap + sorted(seen)[-1]] = float("nan")
        out = torch.zeros(1, 4 * 64, device="cuda")
        pos = torch.tensor([first], device="cuda")
        qt = torch.from_numpy(q.astype(np.float32)).cuda()
        ring.cache.attention(pos.data_ptr(), 1, q_heads=4, q=qt.data_ptr(), out=out.data_ptr(), window=window,
                             stream_ptr=_stream())
        torch.cuda.synchronize()
        assert torch.isnan(out.view(4, 64)[2:]).all() and torch.isfinite(out.view(4, 64)[:2]).all()


def test_attention_extreme_scores(gpu):
    """Scores of +-1e4 and all equal: no overflow, exact zeros where the formula underflows."""
    rng = np.random.RandomState(10)
    ring = Ring(gpu, 1, 1, 128, 200, 0, rng)
    _check_attention(gpu, ring, "f32", 1, 2, 0, [199], np.zeros((1, 2, 128)), 1.0)
    big = rng.randn(1, 2, 128)
    ring.scales[0][:] = 2.0 ** -4
    _check_attention(gpu, ring, "f32", 1, 2, 0, [199], big, -1.0)
    ring.codes[0][50] = 0xEE
    ring.scales[0][50] = 64.0
    out = torch.zeros(1, 2 * 128, device="cuda")
    q = torch.ones(1, 2 * 128, device="cuda")
    pos = torch.tensor([199], device="cuda")
    ring.cache.attention(pos.data_ptr(), 1, q_heads=2, q=q.data_ptr(), out=out.data_ptr(), scale=1.0,
                         stream_ptr=_stream())
    torch.cuda.synchronize()
    want = ring.rows(1, 0, 0, [50])[0].astype(np.float32)
    got = out.view(2, 128).cpu().numpy()
    assert (np.abs(got - want) <= 2.0 ** -20 * np.abs(want)).all()


@pytest.mark.parametrize("kind", sorted(TYPES))
def test_attention_queries_of_every_size(gpu, kind):
    """A NaN or an infinity in one query head reaches that head alone; tiny, huge and zero queries, a few large elements."""
    rng = np.random.RandomState(13)
    big = 3.0e4 if kind == "f16" else 1e30
    for hq, n in ((6, 1), (4, 3)):
        ring = Ring(gpu, 1, 2, 128, 90, 0, rng)
        ring.scales[0][:] = 2.0 ** -3
        q = rng.randn(n, hq, 128)
        q[0, 1] = 0
        q[0, 2, 5] = 100.0
        q[0, 3] *= 1e-6
        _check_attention(gpu, ring, kind, n, hq, 0, [80], q, 0.25)
        q[0, 0, 77] = np.nan
        q[n - 1, 1, 3] = -np.inf
        q[0, 3, 9] = big
        qt, _ = _typed(q, kind)
        out = torch.zeros(n, hq * 128, dtype=TYPES[kind], device="cuda")
        pos = torch.tensor([80], device="cuda")
        ring.cache.attention(pos.data_ptr(), n, type=_dz_type(gpu, kind), q_heads=hq, q=qt.data_ptr(),
                             out=out.data_ptr(), scale=0.25, stream_ptr=_stream())
        torch.cuda.synchronize()
        got = out.view(n, hq, 128)
        assert torch.isnan(got[0, 0]).all() and torch.isnan(got[n - 1, 1]).all()
        keep = torch.ones(n, hq, dtype=torch.bool)
        keep[0, 0] = keep[n - 1, 1] = keep[0, 3] = False
        assert torch.isfinite(got[keep.cuda()]).all()


def test_cache_offsets_past_32_bits(gpu):
    """A ring of 70 million slots: 4.5 GB of codes, the newest tokens at its far end."""
    cap, hd, n = 70_000_000, 128, 5
    codes = [torch.zeros(cap, hd // 2, dtype=torch.uint8, device="cuda") for _ in range(2)]
    scales = [torch.zeros(cap, hd // 64, device="cuda") for _ in range(2)]
    cache = gpu.KV4Cache(codes[0].data_ptr(), codes[1].data_ptr(), scales[0].data_ptr(), scales[1].data_ptr(), 1, 1, hd,
                         cap, 2)
    first = cap - n
    pos = torch.tensor([first], device="cuda")
    k, v, q = (torch.randn(n, hd, device="cuda") for _ in range(3))
    held = [torch.empty(n, hd, device="cuda") for _ in range(2)]
    cache.append(pos.data_ptr(), n, k=k.data_ptr(), v=v.data_ptr(), k_out=held[0].data_ptr(),
                 v_out=held[1].data_ptr(), stream_ptr=_stream())
    out = torch.empty(n, hd, device="cuda")
    cache.attention(pos.data_ptr(), n, q_heads=1, q=q.data_ptr(), out=out.data_ptr(), window=n, stream_ptr=_stream())
    torch.cuda.synchronize()
    kv = [_np(t) for t in held]
    for j in range(n):
        # the window's older tokens and the two sinks are zeros
        seen = [np.concatenate([np.zeros((2 + n - 1 - j, hd)), t[:j + 1]]) for t in kv]
        tops = np.abs(seen[1]).reshape(len(seen[1]), -1, 64).max(2) / 7
        ref, bound = fb.attend(_np(q)[j], seen[0], seen[1], hd ** -0.5, tops)
        assert (np.abs(_np(out)[j] - ref) <= bound + fb.rounding(ref, "f32")).all(), j
    assert int((scales[0] != 0).sum()) == 2 * n and (scales[0][-n:] != 0).all()


# Many pairs to a key head: queries enter as fp16 parts (2^-22 of an element or finer), weights as bf16 parts
# (2^-18 of a weight; 2^-27 for fp32), both within what fb.attend() allows for integers.
CHUNKS = [  # batch, n, hq, hk, hd, cap, sinks, window, first positions
    (1, 17, 1, 1, 64, 17, 0, 0, [0]),
    (1, 1, 17, 1, 128, 1, 0, 0, [0]),
    (2, 1, 32, 1, 64, 700, 3, 0, [5000, 31]),
    (3, 5, 4, 1, 128, 300, 4, 32, [-1, 297, 4]),
    (2, 3, 12, 2, 64, 2500, 0, 0, [2490, 600]),
    (1, 6, 6, 2, 128, 5000, 2, 0, [(1 << 33) + 3]),
    (40, 20, 2, 2, 64, 60, 4, 33, [3 * i for i in range(40)]),
    (2, 31, 3, 3, 128, 64, 33, 1, [0, 3000]),
    (1, 9, 10, 5, 128, 41, 0, 33, [32]),
    (1, 16, 5, 1, 64, 400, 1, 100, [700]),
]


@pytest.mark.parametrize("case", CHUNKS)
@pytest.mark.parametrize("kind", sorted(TYPES))
def test_attention_of_chunks(gpu, case, kind):
    batch, n, hq, hk, hd, cap, sinks, window, first = case
    rng = np.random.RandomState(cap + n)
    ring = Ring(gpu, batch, hk, hd, cap, sinks, rng)
    _check_attention(gpu, ring, kind, n, hq, window, first, rng.randn(batch * n, hq, hd), hd ** -0.5)
    for old, new in zip(ring.before, ring.snapshot()):
        np.testing.assert_array_equal(old[0], new[0])
        np.testing.assert_array_equal(old[1], new[1])


@pytest.mark.parametrize("kind", sorted(TYPES))
def test_chunks_with_scales_of_every_size(gpu, kind):
    rng = np.random.RandomState(18)
    ring = Ring(gpu, 2, 2, 128, 400, 0, rng)
    s = ring.scales[1]
    s.copy_(torch.from_numpy(2.0 ** rng.randint(-60, 20 if kind == "f32" else 10, s.shape).astype(np.float32)))
    ring.scales[0][17] = 8.0
    _check_attention(gpu, ring, kind, 9, 4, 0, [391, 300], rng.randn(18, 4, 128), 128 ** -0.5)


def test_chunks_ignore_what_they_do_not_see(gpu):
    """NaN scales in slots that no query of the chunk sees change nothing; one that the later queries alone see
    reaches them alone."""
    rng = np.random.RandomState(19)
    n, hq = 6, 8
    for cap, sinks, window, first in ((300, 4, 64, 5000), (300, 0, 0, 100), (64, 3, 10, 12), (140, 0, 100, 131)):
        ring = Ring(gpu, 1, 2, 64, cap, sinks, rng)
        q = rng.randn(n, hq, 64)
        clean = _check_attention(gpu, ring, "f32", n, hq, window, [first], q, 0.125)
        seen = {fb.slot(p, sinks, cap) for j in range(n)
                for p in fb.visible(first + j, first + n - 1, sinks, cap, window)}
        hidden = torch.tensor([h * cap + s for h in range(2) for s in range(cap) if s not in seen], device="cuda",
                              dtype=torch.int64)
        for which in range(2):
            ring.scales[which][hidden] = float("nan")
            ring.codes[which][hidden] = 0xFF
            ring.scales[which][2 * cap:] = float("nan")
        again = _check_attention(gpu, ring, "f32", n, hq, window, [first], q, 0.125)
        np.testing.assert_array_equal(clean, again)
        for which in range(2):               # the chunk's fourth token, of the second key head
            ring.scales[which][cap + fb.slot(first + 3, sinks, cap)] = float("nan")
            out = torch.zeros(n, hq * 64, device="cuda")
            pos = torch.tensor([first], device="cuda")
            qt = torch.from_numpy(q.astype(np.float32)).cuda()
            ring.cache.attention(pos.data_ptr(), n, q_heads=hq, q=qt.data_ptr(), out=out.data_ptr(), window=window,
                                 stream_ptr=_stream())
            torch.cuda.synchronize()
            got = out.view(n, hq, 64).cpu().numpy()
            np.testing.assert_array_equal(got[:3], clean[0, :3])
            np.testing.assert_array_equal(got[:, :4], clean[0, :, :4])
            assert np.isnan(got[3:, 4:]).all()
            ring.scales[which][cap + fb.slot(first + 3, sinks, cap)] = 1.0
            clean = _check_attention(gpu, ring, "f32", n, hq, window, [first], q, 0.125)


@pytest.mark.parametrize("kind", sorted(TYPES))
def test_chunks_of_queries_of_every_size(gpu, kind):
    rng = np.random.RandomState(23)
    n, hq = 7, 6
    ring = Ring(gpu, 1, 2, 128, 90, 0, rng)
    ring.scales[0][:] = 2.0 ** -3
    q = rng.randn(n, hq, 128)
    q[0, 1] = 0
    q[0, 2, 5] = 100.0
    q[0, 3] *= 1e-6
    clean = _check_attention(gpu, ring, kind, n, hq, 0, [80], q, 0.25)
    q[0, 0, 77] = np.nan
    q[n - 1, 1, 3] = -np.inf
    q[2, 4, 9] = np.inf
    qt, _ = _typed(q, kind)
    out = torch.zeros(n, hq * 128, dtype=TYPES[kind], device="cuda")
    pos = torch.tensor([80], device="cuda")
    ring.cache.attention(pos.data_ptr(), n, type=_dz_type(gpu, kind), q_heads=hq, q=qt.data_ptr(), out=out.data_ptr(),
                         scale=0.25, stream_ptr=_stream())
    torch.cuda.synchronize()
    got = _np(out).reshape(n, hq, 128)
    bad = np.zeros((n, hq), bool)
    bad[0, 0] = bad[n - 1, 1] = bad[2, 4] = True
    assert np.isnan(got[bad]).all()
    np.testing.assert_array_equal(got[~bad], clean[0][~bad])


def test_chunk_offsets_past_32_bits(gpu):
    """The last of 70 million slots, seen by a chunk of 20 pairs of the second key head of two."""
    cap, hd, n = 35_000_000, 128, 5
    codes = [torch.full((2 * cap, hd // 2), 0x77, dtype=torch.uint8, device="cuda") for _ in range(2)]
    scales = [torch.zeros(2 * cap, hd // 64, device="cuda") for _ in range(2)]
    rng = np.random.RandomState(3)
    small = Ring(gpu, 1, 2, hd, 2 * n, 0, rng)
    for which in range(2):
        for h in range(2):
            at = (h + 1) * cap - 2 * n
            codes[which][at:at + 2 * n] = small.codes[which][h * 2 * n:(h + 1) * 2 * n]
            scales[which][at:at + 2 * n] = small.scales[which][h * 2 * n:(h + 1) * 2 * n]
    cache = gpu.KV4Cache(codes[0].data_ptr(), codes[1].data_ptr(), scales[0].data_ptr(), scales[1].data_ptr(), 1, 2, hd,
                         cap, 0)
    q = torch.from_numpy(rng.randn(n, 8, hd).astype(np.float32)).cuda()
    out = torch.empty(n, 8 * hd, device="cuda")
    pos = torch.tensor([cap - n], device="cuda")
    cache.attention(pos.data_ptr(), n, q_heads=8, q=q.data_ptr(), out=out.data_ptr(), window=n, stream_ptr=_stream())
    torch.cuda.synchronize()
    want = _check_attention(gpu, small, "f32", n, 8, n, [n], _np(q), hd ** -0.5)
    np.testing.assert_array_equal(_np(out).reshape(n, 8, hd), want[0])


@pytest.mark.parametrize("n", [1, 9])
def test_positions_that_are_skipped(gpu, n):
    """Negative positions and those of 2^62 and more: neither the cache nor any output row is touched."""
    skipped = [-1, -(1 << 63), 1 << 62, (1 << 63) - 1, (1 << 62) + 12345]
    ring = Ring(gpu, len(skipped), 2, 64, 40, 3, np.random.RandomState(5))
    pos = torch.tensor(skipped, dtype=torch.int64, device="cuda")
    rows = len(skipped) * n
    x = torch.ones(rows, 4 * 64, device="cuda")
    out = [torch.full((rows, 4 * 64), 9.0, device="cuda") for _ in range(2)]
    ring.cache.append(pos.data_ptr(), n, q_heads=4, q=x.data_ptr(), k=x.data_ptr(), v=x.data_ptr(), q_stride=256,
                      k_stride=256, v_stride=256, q_out=out[0].data_ptr(), rope_base=1e4, stream_ptr=_stream())
    ring.cache.attention(pos.data_ptr(), n, q_heads=4, q=x.data_ptr(), out=out[1].data_ptr(), window=20,
                         stream_ptr=_stream())
    torch.cuda.synchronize()
    assert all((t == 9.0).all() for t in out)
    for old, new in zip(ring.before, ring.snapshot()):
        np.testing.assert_array_equal(old[0], new[0])
        np.testing.assert_array_equal(old[1], new[1])


def test_attention_graph_follows_positions(gpu):
    """A captured append + attention is replayed as the sequences grow, the positions changed in place."""
    rng = np.random.RandomState(11)
    hq, hk, hd, cap = 4, 2, 64, 40
    a, b = (Ring(gpu, 2, hk, hd, cap, 2, np.random.RandomState(4)) for _ in range(2))
    pos = torch.tensor([0, 30], dtype=torch.int64, device="cuda")
    qkv = torch.zeros(2, (hq + 2 * hk) * hd, device="cuda")
    out = torch.zeros(2, hq * hd, device="cuda")
    rot = torch.zeros(2, hq * hd, device="cuda")

    def step(ring):
        w = qkv.shape[1]
        base = qkv.data_ptr()
        ring.cache.append(pos.data_ptr(), 1, q_heads=hq, q=base, k=base + 4 * hq * hd, v=base + 4 * (hq + hk) * hd,
                          q_stride=w, k_stride=w, v_stride=w, q_out=rot.data_ptr(), rope_base=1e4,
                          stream_ptr=_stream())
        ring.cache.attention(pos.data_ptr(), 1, q_heads=hq, q=rot.data_ptr(), out=out.data_ptr(), window=20,
                             stream_ptr=_stream())

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(a)
    for i in range(60):
        x = torch.from_numpy(rng.randn(*qkv.shape).astype(np.float32)).cuda()
        qkv.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        step(b)
        torch.cuda.synchronize()
        assert torch.equal(got, out), i
        for x, y in zip(a.snapshot(), b.snapshot()):
            np.testing.assert_array_equal(x[0], y[0])
        pos.add_(1)


def test_run_of_the_operators(gpu):
    """One attention block of a decode step as it is used, on a side stream: the
    group-scaled QKV product, append, attention, the group-scaled output
    product; each stage against its formula on what the stage before gave."""
    rng = np.random.RandomState(12)
    batch, hq, hk, hd, cap, d = 3, 8, 4, 64, 200, 500
    ring = Ring(gpu, batch, hk, hd, cap, 4, rng)
    width = (hq + 2 * hk) * hd
    wi = gpu.GroupedWeightMatrix.encode(rng.randn(d, width) * d ** -0.5, 128)
    wo = gpu.GroupedWeightMatrix.encode(rng.randn(hq * hd, d) * 0.05, 32)
    gains = [(1 + 0.2 * rng.randn(hd)).astype(np.float32) for _ in range(2)]
    g = [torch.from_numpy(x).cuda() for x in gains]
    first = [199, 3, 1234]
    pos = torch.tensor(first, dtype=torch.int64, device="cuda")
    x = torch.randn(batch, d, device="cuda")
    qkv, rot = torch.empty(batch, width, device="cuda"), torch.empty(batch, hq * hd, device="cuda")
    att, y = torch.empty(batch, hq * hd, device="cuda"), torch.empty(batch, d, device="cuda")
    torch.cuda.synchronize()
    side = torch.cuda.Stream().cuda_stream
    wi.matmul_async(x.data_ptr(), qkv.data_ptr(), batch, side)
    base = qkv.data_ptr()
    ring.cache.append(pos.data_ptr(), 1, q_heads=hq, q=base, k=base + 4 * hq * hd, v=base + 4 * (hq + hk) * hd,
                      q_stride=width, k_stride=width, v_stride=width, q_out=rot.data_ptr(), q_gain=g[0].data_ptr(),
                      k_gain=g[1].data_ptr(), rope_base=1e4, stream_ptr=side)
    ring.cache.attention(pos.data_ptr(), 1, q_heads=hq, q=rot.data_ptr(), out=att.data_ptr(), window=128,
                         stream_ptr=side)
    wo.matmul_async(att.data_ptr(), y.data_ptr(), batch, side)
    torch.cuda.synchronize()
    ref, bound = fb.product(_np(x), wi.unpack().astype(np.float64))
    assert (np.abs(_np(qkv) - ref) <= bound + fb.rounding(ref, "f32")).all()
    where = np.asarray(first)
    rows = _np(qkv).reshape(batch, hq + 2 * hk, hd)
    yq, mag = fb.norm_rotate(rows[:, :hq], gains[0], 1e-6, where, 1e4, False)
    assert (np.abs(_np(rot).reshape(batch, hq, hd) - yq) <= 2.0 ** -20 * mag + fb.rounding(yq, "f32")).all()
    yk, _ = fb.norm_rotate(rows[:, hq:hq + hk], gains[1], 1e-6, where, 1e4, False)
    for b, p in enumerate(first):
        s = fb.slot(p, 4, cap)
        for h in range(hk):
            for which, values in ((0, yk[b, h]), (1, rows[b, hq + hk + h])):
                held = ring.rows(which, b, h, [s])[0]
                step = np.abs(values).max() / 7
                assert (np.abs(held - values) <= step * (0.5 + 2.0 ** -18)).all()
        seen = [fb.slot(i, 4, cap) for i in fb.visible(p, p, 4, cap, 128)]
        for h in range(hq):
            ref, bound = fb.attend(_np(rot)[b, h * hd:(h + 1) * hd], ring.rows(0, b, h // 2, seen),
                                      ring.rows(1, b, h // 2, seen), hd ** -0.5, ring.scale_rows(1, b, h // 2, seen))
            assert (np.abs(_np(att)[b, h * hd:(h + 1) * hd] - ref) <= bound + fb.rounding(ref, "f32")).all()
    ref, bound = fb.product(_np(att), wo.unpack().astype(np.float64))
    assert (np.abs(_np(y) - ref) <= bound + fb.rounding(ref, "f32")).all()
    wi.close()
    wo.close()
