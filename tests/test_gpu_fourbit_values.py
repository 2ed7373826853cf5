"""The 4-bit operators on values that ask for each element's own precision: a
few large elements beside small ones, columns that the large ones do not reach,
scales of both signs, and every type's largest and smallest numbers."""
import numpy as np
import pytest
import torch

import _fourbit as fb
from _fourbit import GROUP
from test_gpu_fourbit import Ring, TYPES, _append, _dz_type, _np, _stream, _typed

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ products

def product_bound(x, w, group):
    """What the sums of exact products may lose. A scale group's products go
    through group / 16 additions of 16 products to an fp32 accumulator, in which
    each of the 17 terms may be off by 2^-23 = 2 u of the largest, itself at most
    the sum of magnitudes; then one multiplication and K / group + 32 additions
    (warps, 16 blocks, an activation's parts) of half a step each."""
    return (2 * 17 * (group / 16) + x.shape[1] / group + 34) * fb.U * (np.abs(x) @ np.abs(w))


def _product(gpu, q, x, kind):
    xt, xv = _typed(x, kind)
    y = torch.empty(len(x), q.cols, dtype=TYPES[kind], device="cuda")
    q.matmul_async(xt.data_ptr(), y.data_ptr(), len(x), _stream(), type=_dz_type(gpu, kind))
    torch.cuda.synchronize()
    return _np(y), xv


@pytest.mark.parametrize("m,k,n", [(1, 4096, 96), (3, 1000, 40), (8, 2048, 64), (16, 515, 33)])
@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("kind", sorted(TYPES))
def test_products_beside_large_elements(gpu, m, k, n, group, kind):
    """Every 128 activations hold one 2^12 to 2^16 above the rest (fp32 and bf16:
    also 2^30); even columns of W have level 0 there, so that the others alone make
    their results."""
    rng = np.random.RandomState(k + group)
    w = rng.randn(k, n).astype(np.float32)
    large = np.arange(rng.randint(128), k, 128)
    w[large, ::2] = 0
    q = gpu.GroupedWeightMatrix.encode(w, group)
    values = q.unpack().astype(np.float64)
    assert (values[large, ::2] == 0).all()
    for top in (12, 16) if kind == "f16" else (12, 16, 30):
        x = rng.randn(m, k) * (1 / 8 if kind == "f16" else 1)
        x[:, large] = 2.0 ** top * rng.uniform(0.6, 0.95, (m, large.size)) * rng.choice([-1, 1], (m, large.size))
        got, xv = _product(gpu, q, x, kind)
        ref = xv @ values
        bound = product_bound(xv, values, group)
        # results that no value of the type is next to are infinities
        edge = torch.finfo(TYPES[kind]).max * (1 + fb.HALF[kind])
        over, near = np.abs(ref) - bound >= edge, np.abs(ref) + bound >= edge
        assert (got[over] == np.copysign(np.inf, ref[over])).all()
        err = (np.abs(got - ref) - fb.rounding(ref, kind))[~near]
        assert (err <= bound[~near]).all(), (top, (err / bound[~near]).max())
        assert not near[:, ::2].any()
    q.close()


@pytest.mark.parametrize("kind", sorted(TYPES))
def test_product_special_values_of_every_type(gpu, kind):
    rng = np.random.RandomState(21)
    k, n, group = 700, 50, 32
    q = gpu.GroupedWeightMatrix.encode(rng.randn(k, n) * 0.1, group)
    w = q.unpack().astype(np.float64)
    info = torch.finfo(TYPES[kind])
    x = rng.randn(9, k)
    x[0] = 0
    x[1, 5] = np.inf
    x[2, 699] = np.nan
    x[3] = info.smallest_normal * rng.randint(-3, 4, k)       # the smallest, and for 16 bits subnormals
    if kind != "f32":
        x[3] = info.smallest_normal * 2.0 ** rng.randint(-6, 2, k)
    x[4] = 0
    x[4, 300] = -info.max
    x[5] = rng.choice([-1, 1], k) * info.max / 4096
    x[6, ::2] *= 2.0 ** 12
    x[7, 64] = -np.inf
    x[7, 65] = np.inf
    got, xv = _product(gpu, q, x, kind)
    assert (got[0] == 0).all() and np.isnan(got[[1, 2, 7]]).all()
    for r in (3, 4, 5, 6, 8):
        ref = xv[r:r + 1] @ w
        bound = product_bound(xv[r:r + 1], w, group) + 700 * 2.0 ** -133    # bits of fp32 parts below 2^-133
        assert np.abs(ref).max() < info.max and (np.abs(got[r] - ref) <= bound + fb.rounding(ref, kind)).all(), r
    q.close()


def test_synchronous_product_is_the_asynchronous_one(gpu):
    rng = np.random.RandomState(22)
    q = gpu.GroupedWeightMatrix.encode(rng.randn(333, 70), 64)
    x = rng.randn(20, 333).astype(np.float32)
    got, _ = _product(gpu, q, x, "f32")
    np.testing.assert_array_equal(q.matmul(x).astype(np.float64), got)
    q.close()


@pytest.mark.parametrize("kind", sorted(TYPES))
def test_products_whose_rows_go_in_several_passes(gpu, kind):
    """K so large that 16 rows of activations do not fit a block's shared memory together."""
    rng = np.random.RandomState(23)
    m, k, n = 16, 100000, 80
    q = gpu.GroupedWeightMatrix.encode(rng.randn(k, n) * 0.05, 128)
    got, xv = _product(gpu, q, rng.randn(m, k), kind)
    values = q.unpack().astype(np.float64)
    ref = xv @ values
    assert (np.abs(got - ref) <= product_bound(xv, values, 128) + fb.rounding(ref, kind)).all()
    q.close()


def test_products_of_the_longest_rows(gpu):
    """K of 340000: a matrix of that many rows is accepted, and one row's activations take 16 blocks' shared memory."""
    rng = np.random.RandomState(24)
    k, n = 340000, 40
    q = gpu.GroupedWeightMatrix.encode(rng.randn(k, n) * 0.05, 32)
    values = q.unpack().astype(np.float64)
    for kind in TYPES:
        got, xv = _product(gpu, q, rng.randn(2, k), kind)
        ref = xv @ values
        assert (np.abs(got - ref) <= product_bound(xv, values, 32) + fb.rounding(ref, kind)).all(), kind
    q.close()


def test_product_in_several_launches(gpu):
    """K so long and N so wide that a launch takes a range of the columns; strided rows, guard columns."""
    rng = np.random.RandomState(25)
    k, n, m, group = 360000, 20011, 2, 32
    codes = torch.randint(0, 15, (k * n // 2 + 1,), dtype=torch.uint8, device="cuda")
    codes.mul_(16).add_(torch.randint(0, 15, codes.shape, dtype=torch.uint8, device="cuda"))
    scales = torch.rand(-(-k // group), n, device="cuda") * 0.01
    q = gpu.GroupedWeightMatrix.from_device(scales.data_ptr(), codes.data_ptr(), k, n, group)
    x = torch.from_numpy(rng.randn(m, k + 3).astype(np.float32)).cuda()
    y = torch.full((m, n + 5), 9.0, device="cuda")
    q.matmul_async(x.data_ptr(), y.data_ptr(), m, _stream(), lda=k + 3, ldc=n + 5)
    torch.cuda.synchronize()
    assert (y[:, n:] == 9.0).all()
    pick = torch.cat([torch.arange(0, n, 997), torch.arange(n - 40, n)]).cuda()
    at = torch.arange(k, device="cuda")[:, None] * n + pick
    byte = codes[at // 2].long()
    w = (torch.where(at % 2 == 0, byte & 15, byte >> 4).double() - 7) * scales[:, pick].double().repeat_interleave(group, 0)[:k]
    w, xv = w.cpu().numpy(), _np(x[:, :k])
    ref = xv @ w
    assert (np.abs(_np(y[:, pick]) - ref) <= product_bound(xv, w, group) + fb.rounding(ref, "f32")).all()
    q.close()


def test_matrix_from_codes_that_another_device_still_writes(gpu):
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two devices")
    k, n, group = 4096, 4096, 128
    rng = np.random.RandomState(26)
    s, p = gpu.quantize_pack_grouped(rng.randn(k, n).astype(np.float32), group)
    with torch.cuda.device(1):
        ps, pp = torch.from_numpy(s).pin_memory(), torch.from_numpy(p).pin_memory()
        a = torch.randn(8192, 8192, device="cuda:1")
        ds, dp = torch.zeros(s.shape, device="cuda:1"), torch.zeros(p.shape, dtype=torch.uint8, device="cuda:1")
        torch.cuda.synchronize()
        for _ in range(20):
            a = a @ a * 1e-4
        ds.copy_(ps, non_blocking=True)
        dp.copy_(pp, non_blocking=True)
    q = gpu.GroupedWeightMatrix.from_device(ds.data_ptr(), dp.data_ptr(), k, n, group)
    np.testing.assert_array_equal(q.unpack(), fb.dequant(s, p, k, n, group).astype(np.float32))
    q.close()


def test_an_allocation_that_fails_leaves_no_error_behind(gpu):
    """A product whose result no device holds is refused, and the next call does not find its error."""
    L = gpu.lib()
    k, n, m = 1, 100000, 1 << 24
    q = gpu.GroupedWeightMatrix.encode(np.ones((k, n), np.float32), 32)
    a = np.ones((m, k), np.float32)
    assert L.dz_cuda_matmul_grouped(a.ctypes.data, q.handle, a.ctypes.data, m, k) == -5     # a 6 TB result: not enough memory
    again = gpu.GroupedWeightMatrix.encode(np.ones((40, 8), np.float32), 32)
    assert (again.unpack() == 1).all()
    assert np.abs(again.matmul(np.ones((2, 40), np.float32)) - 40).max() < 1e-4
    again.close()
    q.close()


# -------------------------------------------------------------------- append

@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("halves", [False, True])
def test_append_norms_with_gains_of_every_size(gpu, hd, halves):
    """Rows of 1e-12 to 1e17 normed to 1, times gains of 1e-25 to 1e25: neither product leaves fp32's range on the way."""
    rng = np.random.RandomState(27)
    ring = Ring(gpu, 6, 1, hd, 4, 0, rng)
    pos = torch.tensor([0, 1, 2, 3, 100, 7], device="cuda")
    for size in (1e25, 1.0, 1e-25):
        x = (rng.randn(6, 1, hd) * np.array([1e-12, 1e-6, 1.0, 1e6, 1e12, 1e17]).reshape(6, 1, 1)).astype(np.float32)
        gain = (size * (1 + 0.2 * rng.randn(hd))).astype(np.float32)
        t = torch.from_numpy(x).cuda()
        q, k, _ = _append(gpu, ring, "f32", pos, 1, 1, t, t, t, (gain, gain), 1e4, halves, eps=0.0)
        want, mag = fb.norm_rotate(x, gain, 0.0, _np(pos), 1e4, halves)
        got = _np(q).reshape(want.shape)
        # about a dozen fp32 roundings of a norm (its sum is a tree) and three of a rotation
        assert (np.abs(got - want) <= 2.0 ** -20 * mag + fb.rounding(want, "f32")).all(), size
        held = _np(k).reshape(want.shape)
        step = np.abs(want).reshape(6, -1, GROUP).max(2).repeat(GROUP, 1).reshape(want.shape) / 7
        assert (np.abs(held - want) <= step * (0.5 + 2.0 ** -17)).all(), size


# ----------------------------------------------------------------- attention

PAIRS = [(1, 2, 2), (1, 4, 2), (1, 4, 1), (2, 4, 1), (2, 8, 1), (9, 4, 1)]   # tokens, heads, key heads: both kernels


def attend_bound(q, k, v, scale, v_scales, kind, p):
    """What an evaluation with fp32 sums may lose. A query's element is held to
    2^-30 of the largest of its 64, or to 2^-22 = 4 u of its own size; a score is
    the sum of hd / 16 additions of 16 products whose 17 terms may each be off by 2
    u of the largest, and a dozen roundings. A weight is off by twice its score's
    error, by the exponential's 2^-21, by 2^-17 (fp16 and bf16: two bf16 parts) or
    2^-26 of itself or by 2^-30 of the largest in its tile of 32 tokens, all within
    31 places of it, times a level of at most 7. Values add up in at most 6 such
    additions of 16 per 32 tokens, and joins in n / 16 + 64 roundings."""
    n, hd = k.shape
    tops = np.abs(q).reshape(-1, GROUP).max(1)
    held = (np.abs(k).reshape(n, -1, GROUP).sum(2) @ tops).max() * 2.0 ** -30
    score = abs(scale) * ((34 * hd / 16 + 16) * fb.U * (np.abs(k) @ np.abs(q)).max() + held)
    w = np.pad(p * np.abs(v_scales).max(1), 31)
    near = np.lib.stride_tricks.sliding_window_view(w, 63).max(1)
    own = 2.0 ** -26 if kind == "f32" else 2.0 ** -17
    sums = (n / 16 + 64 + 6 * 34 * (n / 32 + 1)) * fb.U
    return (2 * score + 2.0 ** -21 + own + sums) * (p @ np.abs(v)) + 7 * 2.0 ** -30 * near.sum()


def _attend(gpu, ring, kind, n, hq, first, q, scale, window=0):
    """Runs attention and compares every output with the formula; returns the outputs."""
    qt, qv = _typed(q, kind)
    out = torch.full((ring.batch * n, hq * ring.hd), 9.0, dtype=TYPES[kind], device="cuda")
    pos = torch.tensor(first, dtype=torch.int64, device="cuda")
    ring.cache.attention(pos.data_ptr(), n, type=_dz_type(gpu, kind), q_heads=hq, q=qt.data_ptr(), out=out.data_ptr(),
                         scale=scale, window=window, stream_ptr=_stream())
    torch.cuda.synchronize()
    got = _np(out).reshape(ring.batch, n, hq, ring.hd)
    qv = qv.reshape(ring.batch, n, hq, ring.hd)
    for b, f in enumerate(first):
        for h in range(hq):
            kv = [ring.rows(w, b, h * ring.heads // hq, list(range(ring.cap))) for w in range(2)]
            vs = ring.scale_rows(1, b, h * ring.heads // hq, list(range(ring.cap)))
            for j in range(n):
                slots = [fb.slot(p, ring.sinks, ring.cap)
                         for p in fb.visible(f + j, f + n - 1, ring.sinks, ring.cap, window)]
                k, v = (x[slots] for x in kv)
                e = scale * (k @ qv[b, j, h])
                e = np.exp(e - e.max())
                ref = (e / e.sum()) @ v
                bound = attend_bound(qv[b, j, h], k, v, scale, vs[slots], kind, e / e.sum())
                err = np.abs(got[b, j, h] - ref) - 1.001 * fb.rounding(ref, kind)
                assert (err <= bound).all(), (b, j, h, (err / bound).max())
    return got


@pytest.mark.parametrize("n,hq,hk", PAIRS)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("kind", sorted(TYPES))
def test_attention_with_scales_of_both_signs(gpu, n, hq, hk, hd, kind):
    """A scale's sign is the caller's: value = scale * (code - 7) for keys and values."""
    rng = np.random.RandomState(31 + n + hd)
    ring = Ring(gpu, 2, hk, hd, 150, 3, rng)
    for s in ring.scales:
        s.mul_(torch.from_numpy(rng.choice([-1.0, 1.0], s.shape).astype(np.float32)).cuda())
    _attend(gpu, ring, kind, n, hq, [140, 4321], rng.randn(2 * n, hq, hd), hd ** -0.5)
    ring.scales[1].abs_().neg_()
    _attend(gpu, ring, kind, n, hq, [77, 30], rng.randn(2 * n, hq, hd), hd ** -0.5, window=100)


@pytest.mark.parametrize("n,hq,hk", PAIRS)
@pytest.mark.parametrize("kind", sorted(TYPES))
def test_attention_beside_a_token_that_takes_all_weight(gpu, n, hq, hk, kind):
    """The first token takes all weight but 2^-12 or so and holds level 0 in half of the elements: there
    the others alone make the result, most of all those of its own tile."""
    rng = np.random.RandomState(41 + n)
    hd, count = 128, 40
    ring = Ring(gpu, 1, hk, hd, 60, 0, rng)
    q = rng.choice([-1.0, 1.0], hd)
    for h in range(hk):
        at = h * ring.cap
        level = (7 + 7 * q).astype(np.uint8)                  # key: +-7 along the query
        ring.codes[0][at] = torch.from_numpy(level[0::2] | level[1::2] << 4).cuda()
        ring.scales[0][at] = 0.25
        ring.codes[1][at] = ring.codes[1][at] & 0xF0 | 7      # value: even elements level 0
        ring.scales[0][at + 1:at + ring.cap] = 2.0 ** -10
    _attend(gpu, ring, kind, n, hq, [count - n], np.broadcast_to(q, (n, hq, hd)), 0.04)


@pytest.mark.parametrize("n,hq,hk", PAIRS)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("kind", sorted(TYPES))
def test_attention_of_queries_with_large_elements(gpu, n, hq, hk, hd, kind):
    """Every 64 elements of a query hold one 2^12 to 2^15 above the rest, at which all keys hold level 0: the
    others alone make the scores, as precisely with few pairs to a key head as with many."""
    rng = np.random.RandomState(51 + n + hd)
    ring = Ring(gpu, 2, hk, hd, 150, 3, rng)
    large = np.arange(rng.randint(GROUP), hd, GROUP)
    for e in large:
        codes = ring.codes[0][:, e // 2]
        codes.copy_(codes & 0xF0 | 7 if e % 2 == 0 else codes & 0x0F | 0x70)
    for top in (12, 15):
        q = rng.randn(2 * n, hq, hd) * (0.5 if kind == "f16" else 1)
        q[..., large] = 2.0 ** top * rng.uniform(0.6, 0.95, (2 * n, hq, large.size))
        _attend(gpu, ring, kind, n, hq, [140, 4321], q, 0.25)
