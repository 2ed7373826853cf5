"""8-bit operators without a GPU: the refusals of the C entry points (checked
before any device call), and the oracle's own arithmetic."""
import ctypes

import numpy as np
import pytest

import _eightbit as eb

INVALID, UNSUPPORTED = -1, -6
AT = 4096     # an address that no refused call reads


def _norm(**change):
    from dranzer_b200._native import DzNormQ8
    f = dict(device=0, type=0, x=AT, x_stride=64, residual=AT, residual_stride=64, sum_out=AT, sum_stride=64, gain=AT,
             norm=1, eps=1e-6, codes=AT, codes_stride=64, scales=AT)
    f.update(change)
    return DzNormQ8(**f)


@pytest.mark.parametrize("change", [dict(x=None), dict(codes=None), dict(scales=None), dict(type=3), dict(type=-1),
                                    dict(x_stride=63), dict(residual_stride=63), dict(sum_stride=63),
                                    dict(codes_stride=63), dict(x=AT + 2), dict(residual=AT + 1), dict(sum_out=AT + 2),
                                    dict(gain=AT + 2), dict(scales=AT + 1), dict(norm=2), dict(norm=-1), dict(eps=-1.0),
                                    dict(eps=float("nan")), dict(eps=float("inf")), dict(x_stride=(1 << 40) + 1),
                                    dict(codes_stride=(1 << 40) + 1)])
def test_norm_q8_refuses(dz, change):
    from dranzer_b200 import _native
    assert _native.lib().dz_cuda_norm_q8(ctypes.byref(_norm(**change)), 4, 64, None) == INVALID
    assert _native.last_error()[1]


@pytest.mark.parametrize("rows,width", [(0, 64), (4, 0), (1 << 31, 64), (4, (1 << 30) + 1)])
def test_norm_q8_refuses_sizes(dz, rows, width):
    from dranzer_b200 import _native
    a = _norm(x_stride=1 << 31, residual_stride=1 << 31, sum_stride=1 << 31, codes_stride=1 << 31)
    assert _native.lib().dz_cuda_norm_q8(ctypes.byref(a), rows, width, None) == INVALID
    assert _native.lib().dz_cuda_norm_q8(None, 4, 64, None) == INVALID


def test_matmul_q8_refuses_nulls(dz):
    from dranzer_b200 import _native
    assert _native.lib().dz_cuda_matmul_q8_async(AT, 64, AT, None, None, AT, 64, 1, 64, 0, None) == INVALID
    assert _native.last_error()[1]


def _cache(**change):
    from dranzer_b200._native import DzKv8
    f = dict(device=0, k_codes=AT, v_codes=AT, k_scales=AT, v_scales=AT, pages=8, page=32, kv_heads=2, head_dim=64,
             table=AT, batch=3, table_pages=4)
    f.update(change)
    return DzKv8(**f)


def _append(**change):
    from dranzer_b200._native import DzKv4Append
    f = dict(type=0, q_heads=4, q=AT, k=AT, v=AT, q_stride=256, k_stride=128, v_stride=128, q_out=AT, q_out_stride=256,
             k_out=None, v_out=None, k_out_stride=128, v_out_stride=128, q_gain=None, k_gain=None, eps=1e-6,
             rope_base=0.0, rope_pairing=0)
    f.update(change)
    return DzKv4Append(**f)


def _attention(**change):
    from dranzer_b200._native import DzKv8Attention
    f = dict(type=0, q_heads=4, q=AT, q_stride=256, out=AT, out_stride=256, scale=0.125, window=0, longest=0)
    f.update(change)
    return DzKv8Attention(**f)


@pytest.mark.parametrize("change,status", [
    (dict(k_codes=None), INVALID), (dict(v_codes=None), INVALID), (dict(k_scales=None), INVALID),
    (dict(v_scales=None), INVALID), (dict(table=None), INVALID), (dict(head_dim=32), UNSUPPORTED),
    (dict(head_dim=0), UNSUPPORTED), (dict(page=16), UNSUPPORTED), (dict(page=0), UNSUPPORTED),
    (dict(page=48), UNSUPPORTED), (dict(batch=0), INVALID), (dict(batch=65536), INVALID), (dict(kv_heads=0), INVALID),
    (dict(kv_heads=65536), INVALID), (dict(pages=0), INVALID), (dict(pages=1 << 31), INVALID),
    (dict(table_pages=0), INVALID), (dict(table_pages=(1 << 31) // 32), INVALID),
    (dict(k_codes=AT + 8), INVALID),
    (dict(v_codes=AT + 1), INVALID), (dict(k_scales=AT + 2), INVALID), (dict(table=AT + 2), INVALID)])
def test_caches_are_refused(dz, change, status):
    from dranzer_b200 import _native
    L, c = _native.lib(), _cache(**change)
    heads = c.kv_heads
    wide = 1 << 23
    a = _append(q_heads=0, k_stride=wide, v_stride=wide)
    assert L.dz_cuda_kv8_append(ctypes.byref(c), ctypes.byref(a), AT, 1, None) == status
    a = _attention(q_heads=max(1, heads), q_stride=wide, out_stride=wide)
    assert L.dz_cuda_kv8_attention(ctypes.byref(c), ctypes.byref(a), AT, 1, None) == status
    assert _native.last_error()[1]


@pytest.mark.parametrize("positions,tokens", [(None, 1), (AT + 4, 1), (AT, 0), (AT, 129)])
def test_positions_and_token_counts_are_refused(dz, positions, tokens):
    from dranzer_b200 import _native
    L, c = _native.lib(), _cache()
    assert L.dz_cuda_kv8_append(ctypes.byref(c), ctypes.byref(_append()), positions, tokens, None) == INVALID
    assert L.dz_cuda_kv8_attention(ctypes.byref(c), ctypes.byref(_attention()), positions, tokens, None) == INVALID


@pytest.mark.parametrize("change", [dict(type=3), dict(q=None), dict(q_out=None), dict(k=None), dict(v=None),
                                    dict(q_stride=255), dict(k_stride=127), dict(v_stride=127), dict(q_out_stride=255),
                                    dict(k=AT + 2), dict(q=AT + 1), dict(k_out=AT, k_out_stride=127),
                                    dict(v_out=AT, v_out_stride=100), dict(v_out=AT + 3), dict(q_gain=AT, eps=-1.0),
                                    dict(k_gain=AT, eps=float("nan")), dict(k_gain=AT + 2), dict(rope_base=-1.0),
                                    dict(rope_base=float("inf")), dict(rope_pairing=2), dict(q_heads=65536),
                                    dict(q_stride=(1 << 40) + 1)])
def test_appends_are_refused(dz, change):
    from dranzer_b200 import _native
    c = _cache()
    assert _native.lib().dz_cuda_kv8_append(ctypes.byref(c), ctypes.byref(_append(**change)), AT, 1, None) == INVALID
    assert _native.lib().dz_cuda_kv8_append(ctypes.byref(c), None, AT, 1, None) == INVALID


@pytest.mark.parametrize("change", [dict(type=3), dict(q_heads=0), dict(q_heads=3), dict(q_heads=65536), dict(q=None),
                                    dict(out=None), dict(q_stride=255), dict(out_stride=255), dict(q=AT + 2),
                                    dict(out=AT + 1), dict(scale=float("nan")), dict(scale=float("inf"))])
def test_attentions_are_refused(dz, change):
    from dranzer_b200 import _native
    c = _cache()
    assert _native.lib().dz_cuda_kv8_attention(ctypes.byref(c), ctypes.byref(_attention(**change)), AT, 1, None) == INVALID
    assert _native.lib().dz_cuda_kv8_attention(ctypes.byref(c), None, AT, 1, None) == INVALID


def test_too_many_rows_and_heads_are_refused(dz):
    from dranzer_b200 import _native
    c = _cache(batch=65535, table_pages=1 << 20, kv_heads=8)
    a = _append(q_heads=64, q_stride=4096, q_out_stride=4096, k_stride=512, v_stride=512)
    assert _native.lib().dz_cuda_kv8_append(ctypes.byref(c), ctypes.byref(a), AT, 1 << 20, None) == INVALID
    a = _attention(q_heads=64, q_stride=4096, out_stride=4096)
    assert _native.lib().dz_cuda_kv8_attention(ctypes.byref(c), ctypes.byref(a), AT, 1 << 20, None) == INVALID


def test_oracle_rows_are_the_framework_quantizer(dz):
    """Without a norm, a row's codes and scale are those of the framework's 8-bit quantizer, one scale a row."""
    rng = np.random.RandomState(0)
    x = (rng.randn(9, 131) * np.exp(rng.randn(9, 1))).astype(np.float32)
    x[4] = 0
    codes, scales = eb.norm_rows(x.astype(np.float64), None, False, 0.0)
    s, p = dz.quantize_pack(x, 8, dz.GRAN_ROW)
    keep = np.arange(9) != 4     # a row of zeros has scale 0 here
    np.testing.assert_array_equal(codes[keep], (p.reshape(x.shape).astype(np.int64) - 127)[keep])
    np.testing.assert_array_equal(scales.astype(np.float32)[keep], s[keep])


def test_oracle_append_keeps_values_within_a_step():
    """Rows that go into a page one by one stay within half a step for each time that the scale grew, and half for themselves."""
    rng = np.random.RandomState(1)
    c = eb.Cache(rng, 4, 32, 1, 64, [[2]])
    y = (rng.randn(32, 1, 64) * np.linspace(0.1, 2, 32)[:, None, None]).astype(np.float32)
    grew, last = 0, 0.0
    for j in range(32):
        c.append("k", 0, j, y[j:j + 1])
        scale = float(c.scales["k"][2, 0])
        grew += scale > last
        last = scale
    got, there = c.values("k", 0, 0, 32, 0)
    assert there.all() and (np.abs(got - y[:, 0]) <= 0.5001 * last * grew).all()
