"""A NaN value that a query sees reaches its output also where the token's softmax
weight is zero, and one that it does not see does not, wherever tiles end."""
import numpy as np
import pytest
import torch

from test_gpu_fourbit import Ring, TYPES, _dz_type, _np, _stream

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,hq,hk", [(1, 1, 1), (1, 4, 1), (2, 1, 1), (2, 2, 1), (4, 1, 1), (9, 4, 1)])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("kind", sorted(TYPES))
def test_nan_values_of_tokens_without_weight(gpu, n, hq, hk, hd, kind):
    rng = np.random.RandomState(61 + n)
    count = 75                                                # two tiles of 32 and a part; the last queries end within
    ring = Ring(gpu, 1, hk, hd, 100, 0, rng)
    first = count - n
    sign = rng.choice([-1, 1], hd)
    level = (7 - 7 * sign).astype(np.uint8)
    q = torch.from_numpy(np.broadcast_to(sign, (n, hq, hd)).astype(np.float32).copy()).to(TYPES[kind]).cuda()
    pos = torch.tensor([first], device="cuda")
    out = torch.empty(n, hq * hd, dtype=TYPES[kind], device="cuda")
    ring.scales[0].fill_(2.0 ** -8)
    scales = [s.clone() for s in ring.scales]
    codes = ring.codes[0].clone()
    for token in (0, 40, first, count - 1, count):            # a far score, a NaN value; `count` itself nobody sees
        ring.codes[0][token] = torch.from_numpy(level[0::2] | level[1::2] << 4).cuda()
        ring.scales[0][token] = 8.0
        ring.scales[1][token] = float("nan")
        ring.cache.attention(pos.data_ptr(), n, type=_dz_type(gpu, kind), q_heads=hq, q=q.data_ptr(),
                             out=out.data_ptr(), scale=1.0, stream_ptr=_stream())
        torch.cuda.synchronize()
        nan = np.isnan(_np(out).reshape(n, -1))
        for j in range(n):
            assert nan[j].all() if token <= first + j else not nan[j].any(), (token, j)
        for s, old in zip(ring.scales, scales):
            s.copy_(old)
        ring.codes[0].copy_(codes)
