"""Limits of the 4-bit entry points that keep their index arithmetic in range
(checked before any device call)."""
import ctypes

import pytest

from test_fourbit import INVALID, _append, _attention, _cache


@pytest.mark.parametrize("batch,kv_heads,head_dim", [(4000, 65535, 64), (2000, 65535, 128), (16000, 60000, 128)])
def test_kv4_refuses_buffers_past_62_bit_offsets(dz, batch, kv_heads, head_dim):
    from dranzer_b200 import _native
    L = _native.lib()
    c = _cache(batch=batch, kv_heads=kv_heads, head_dim=head_dim, capacity=(1 << 31) - 64)
    wide = 1 << 23
    a = _append(q_heads=0, k_stride=wide, v_stride=wide)
    assert L.dz_cuda_kv4_append(ctypes.byref(c), ctypes.byref(a), 4096, 1, None) == INVALID
    assert b"2^62" in _native.last_error()[1].encode()
    a = _attention(q_heads=kv_heads, q_stride=wide, out_stride=wide)
    assert L.dz_cuda_kv4_attention(ctypes.byref(c), ctypes.byref(a), 4096, 1, None) == INVALID
    assert b"2^62" in _native.last_error()[1].encode()
