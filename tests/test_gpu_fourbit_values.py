"""The 4-bit operators on values that ask for each element's own precision: a
few large elements beside small ones, columns that the large ones do not reach,
scales of both signs, and every type's largest and smallest numbers."""
import numpy as np
import pytest
import torch

import _fourbit as fb
from test_gpu_fourbit import TYPES, _dz_type, _np, _stream, _typed

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
