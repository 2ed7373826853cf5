"""4-bit operators without a GPU: the grouped quantizer, and the refusals of
the C entry points (checked before any device call)."""
import ctypes

import numpy as np
import pytest

import _fourbit as fb

INVALID, UNSUPPORTED = -1, -6


@pytest.mark.parametrize("rows,cols,group", [(1, 1, 32), (31, 5, 32), (33, 7, 32), (128, 3, 64), (200, 9, 64),
                                             (129, 16, 128), (300, 11, 128)])
def test_grouped_quantizer_is_the_framework_quantizer_per_group(dz, rows, cols, group):
    rng = np.random.RandomState(rows + cols)
    w = rng.randn(rows, cols).astype(np.float32)
    w[:, 0] = 0
    s, p = dz.quantize_pack_grouped(w, group)
    codes = fb.unpack(p, rows * cols).reshape(rows, cols)
    for g in range(s.shape[0]):
        part = np.ascontiguousarray(w[g * group:(g + 1) * group])
        s1, p1 = dz.quantize_pack(part, 4, dz.GRAN_COLUMN)
        np.testing.assert_array_equal(s[g].view(np.uint32), s1.view(np.uint32))
        np.testing.assert_array_equal(codes[g * group:(g + 1) * group], fb.unpack(p1, part.size).reshape(part.shape))
    back = dz.quantize_unpack_grouped(s, p, rows, cols, group)
    np.testing.assert_array_equal(back, fb.dequant(s, p, rows, cols, group).astype(np.float32))
    # half a step, plus the roundings of the scaled value and of the product
    step = s.repeat(group, 0)[:rows]
    assert (np.abs(back - w) <= step * (0.5 + 2.0 ** -18)).all()


def test_grouped_quantizer_refuses(dz):
    w = np.ones((40, 3), np.float32)
    for group in (0, 16, 33, 256):
        with pytest.raises(ValueError):
            dz.quantize_pack_grouped(w, group)
    for bad in (np.inf, np.nan):
        v = w.copy()
        v[39, 2] = bad
        with pytest.raises(ValueError):
            dz.quantize_pack_grouped(v, 32)
    s, p = dz.quantize_pack_grouped(w, 32)
    with pytest.raises(ValueError):
        dz.quantize_unpack_grouped(s, p[:-1], 40, 3, 32)
    with pytest.raises(ValueError):
        dz.quantize_unpack_grouped(-s, p, 40, 3, 32)
    with pytest.raises(ValueError):
        dz.quantize_unpack_grouped(s, np.full_like(p, 0xFF), 40, 3, 32)


def _blob(**change):
    from dranzer_b200._native import DzGroupedBlob
    f = dict(rows=64, cols=8, group=32, packed=4096, packed_size=256, scales=4096, scale_count=16, scale_type=0)
    f.update(change)
    return DzGroupedBlob(**f)


@pytest.mark.parametrize("change", [dict(rows=0), dict(cols=0), dict(rows=(1 << 24) + 1), dict(group=0),
                                    dict(group=48), dict(group=256), dict(packed=None), dict(scales=None),
                                    dict(packed_size=255), dict(scale_count=15), dict(scale_type=2),
                                    dict(scale_type=9), dict(rows=65)])
def test_gmatrix_create_refuses(dz, change):
    from dranzer_b200 import _native
    h = ctypes.c_void_p()
    assert _native.lib().dz_cuda_gmatrix_create(0, ctypes.byref(_blob(**change)), ctypes.byref(h)) == INVALID
    assert not h.value and _native.last_error()[1]


def test_matmul_grouped_refuses_nulls(dz):
    from dranzer_b200 import _native
    L = _native.lib()
    assert L.dz_cuda_gmatrix_create(0, None, None) == INVALID
    assert L.dz_cuda_matmul_grouped_async(64, 8, None, 64, 8, 1, 8, 0, None) == INVALID
    assert L.dz_cuda_matmul_grouped(None, None, None, 1, 8) == INVALID
    assert L.dz_cuda_gmatrix_unpack(None, None) == INVALID
    assert L.dz_cuda_gmatrix_bytes(None) == 0
    L.dz_cuda_gmatrix_free(None)


def _cache(**change):
    from dranzer_b200._native import DzKv4
    f = dict(device=0, k_codes=4096, v_codes=8192, k_scales=4096, v_scales=8192, batch=2, kv_heads=2, head_dim=64,
             capacity=32, sinks=4)
    f.update(change)
    return DzKv4(**f)


def _append(**change):
    from dranzer_b200._native import DzKv4Append
    f = dict(type=0, q_heads=4, q=4096, k=4096, v=4096, q_stride=256, k_stride=128, v_stride=128, q_out=4096,
             q_out_stride=256, k_out=None, v_out=None, k_out_stride=0, v_out_stride=0, q_gain=4096, k_gain=4096,
             eps=1e-6, rope_base=1e4, rope_pairing=0)
    f.update(change)
    return DzKv4Append(**f)


def _attention(**change):
    from dranzer_b200._native import DzKv4Attention
    f = dict(type=0, q_heads=4, q=4096, q_stride=256, out=8192, out_stride=256, scale=0.125, window=0)
    f.update(change)
    return DzKv4Attention(**f)


CACHE_REFUSALS = [(dict(k_codes=None), INVALID), (dict(v_scales=None), INVALID), (dict(head_dim=32), UNSUPPORTED),
                  (dict(head_dim=96), UNSUPPORTED), (dict(batch=0), INVALID), (dict(batch=65536), INVALID),
                  (dict(kv_heads=0), INVALID), (dict(capacity=0, sinks=0), INVALID), (dict(sinks=32), INVALID),
                  (dict(capacity=1 << 31), INVALID), (dict(k_codes=4104), INVALID), (dict(v_scales=8196), INVALID)]


@pytest.mark.parametrize("change,status", CACHE_REFUSALS)
def test_kv4_refuses_caches(dz, change, status):
    from dranzer_b200 import _native
    L = _native.lib()
    c = _cache(**change)
    assert L.dz_cuda_kv4_append(ctypes.byref(c), ctypes.byref(_append()), 4096, 1, None) == status
    assert L.dz_cuda_kv4_attention(ctypes.byref(c), ctypes.byref(_attention()), 4096, 1, None) == status


@pytest.mark.parametrize("change", [dict(type=3), dict(type=-1), dict(q=None), dict(k=None), dict(v=None),
                                    dict(q_out=None), dict(q_stride=255), dict(k_stride=127), dict(v_stride=0),
                                    dict(q_out_stride=1), dict(k_out=4096, k_out_stride=127),
                                    dict(v_out=4098, v_out_stride=128), dict(q=4097), dict(eps=-1.0),
                                    dict(eps=float("nan")), dict(rope_base=-2.0), dict(rope_base=float("inf")),
                                    dict(rope_pairing=2), dict(q_gain=4097), dict(q_heads=70000, q_stride=1 << 23,
                                                                                  q_out_stride=1 << 23)])
def test_kv4_append_refuses(dz, change):
    from dranzer_b200 import _native
    st = _native.lib().dz_cuda_kv4_append(ctypes.byref(_cache()), ctypes.byref(_append(**change)), 4096, 1, None)
    assert st == INVALID and _native.last_error()[1]


@pytest.mark.parametrize("change", [dict(type=3), dict(q_heads=0), dict(q_heads=3), dict(q=None), dict(out=None),
                                    dict(q_stride=255), dict(out_stride=255), dict(out=8193),
                                    dict(scale=float("nan")), dict(scale=float("inf")), dict(window=29),
                                    dict(window=(1 << 64) - 1)])
def test_kv4_attention_refuses(dz, change):
    from dranzer_b200 import _native
    L = _native.lib()
    st = L.dz_cuda_kv4_attention(ctypes.byref(_cache()), ctypes.byref(_attention(**change)), 4096, 1, None)
    assert st == INVALID and _native.last_error()[1]


def test_kv4_refuses_capacities_past_32_bit_counts(dz):
    """The kernels count slots in 32 bits up to two tiles of 32 past the last."""
    from dranzer_b200 import _native
    L = _native.lib()
    for capacity in ((1 << 31) - 1, (1 << 31) - 63):
        c = _cache(capacity=capacity)
        assert L.dz_cuda_kv4_append(ctypes.byref(c), ctypes.byref(_append()), 4096, 1, None) == INVALID
        assert L.dz_cuda_kv4_attention(ctypes.byref(c), ctypes.byref(_attention()), 4096, 1, None) == INVALID


def test_kv4_refuses_token_counts(dz):
    from dranzer_b200 import _native
    L = _native.lib()
    for n in (0, 29, 1 << 40):
        assert L.dz_cuda_kv4_append(ctypes.byref(_cache()), ctypes.byref(_append()), 4096, n, None) == INVALID
        assert L.dz_cuda_kv4_attention(ctypes.byref(_cache()), ctypes.byref(_attention()), 4096, n, None) == INVALID
    # a window needs room for the chunk behind it
    a = _attention(window=20)
    assert L.dz_cuda_kv4_attention(ctypes.byref(_cache()), ctypes.byref(a), 4096, 10, None) == INVALID
    assert L.dz_cuda_kv4_attention(ctypes.byref(_cache()), ctypes.byref(a), None, 1, None) == INVALID
    assert L.dz_cuda_kv4_attention(ctypes.byref(_cache()), ctypes.byref(a), 4097, 1, None) == INVALID
    assert L.dz_cuda_kv4_attention(None, ctypes.byref(a), 4096, 1, None) == INVALID
    assert L.dz_cuda_kv4_append(ctypes.byref(_cache()), None, 4096, 1, None) == INVALID
