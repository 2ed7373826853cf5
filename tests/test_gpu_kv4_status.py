"""A 4-bit launch that fails on a model's path reaches the caller. The failing
call is a fake: a library loaded first whose dz_kv4_*_launch return an error
without touching the device takes the place of the product's."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

HERE = os.path.dirname(os.path.abspath(__file__))

FAKE = """
struct CUstream_st;
namespace dz {
struct Kv4AppendArgs;
struct Kv4AttnArgs;
#ifdef APPEND
int dz_kv4_append_launch(const Kv4AppendArgs&, int, int, int, CUstream_st*) { return 9; }   // cudaErrorInvalidConfiguration
#else
int dz_kv4_attn_launch(const Kv4AttnArgs&, int, int, int, CUstream_st*) { return 9; }
#endif
}
"""

CHILD = """
import ctypes, sys
import numpy as np
ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
sys.path[:0] = [sys.argv[2], sys.argv[3]]
import dranzer_b200 as dz
from _models import Spec, quantize_params, synth_params
from _native_oracle import Oracle
spec = Spec(300, 128, 2, 2, 16)
oracle = Oracle()
recs, _ = quantize_params(oracle, spec, synth_params(oracle, spec, 3), 8)
model = dz.Model.from_arrays(spec, [(k, r, c, f, s, p, 8, 2) for (_, k, r, c, f, s, p) in recs])
ids = np.arange(8, dtype=np.uint32).reshape(2, 4)
cache = dz.KVCache(model, 2, 16, kv_bits=4)
greedy = dz.Sampling(dz.GREEDY, masked=())
def generate(mode):
    cache.set_prefill(mode)
    return cache.generate(ids, 3, greedy)
for call in (lambda: cache.forward_tokens(ids[:, 0]), lambda: cache.prefill(ids), lambda: generate(dz.PREFILL_TOKENS),
             lambda: generate(dz.PREFILL_BATCHED)):
    for again in range(2):
        try:
            call()
        except dz.DzError as e:
            assert "configuration" in str(e), e
        else:
            raise SystemExit("a launch that failed was not reported")
# neither the runtime's last error nor the device is touched by it
fp32 = dz.KVCache(model, 2, 16)
assert np.isfinite(fp32.prefill(ids)).all() and np.isfinite(fp32.forward_tokens(ids[:, 0])).all()
assert fp32.generate(ids, 3, greedy).shape == (2, 3)
print("reported")
"""


@pytest.mark.parametrize("which", ["APPEND", "ATTENTION"])
def test_a_failed_launch_is_reported(gpu, oracle, tmp_path, which):
    src, lib = tmp_path / "fake.cpp", tmp_path / "fake.so"
    src.write_text(FAKE)
    subprocess.run(["g++", "-shared", "-fPIC", "-D" + which, str(src), "-o", str(lib)], check=True)
    out = subprocess.run([sys.executable, "-c", CHILD, str(lib), os.path.dirname(HERE), HERE], capture_output=True,
                         text=True, timeout=300)
    assert out.returncode == 0 and "reported" in out.stdout, (out.stdout[-500:], out.stderr[-2000:])
