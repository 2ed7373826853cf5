"""Models on 4-bit caches (dz_cuda_cache_create_kv4): decode steps, batched
prefill and generation against the model's formulas in 64 bits with the same
4-bit keys and values, first tokens kept, windows and ring eviction included.

A key or value next to a border between two codes could fall on either side of
it; the inputs are drawn until none lies within 2e-5 of one (in code steps;
the device's keys and values are within 2^-20 of their group's peak, 7e-6
steps), which depends on the formulas alone. Logits are then compared as
everywhere: max |g - r| / max |r| <= 1e-3."""
import numpy as np
import pytest

import _fourbit as fb
from _models import KIND_PROJECTION, RMSNORM, ROPE, Spec, inventory, quantize_params, synth_params

pytestmark = pytest.mark.gpu

LOGIT_TOL = 1e-3


class Emulated:
    """One sequence of a model with a 4-bit ring cache, in 64 bits."""

    def __init__(self, spec, flat, pe, capacity, sinks, window):
        self.spec, self.pe, self.capacity, self.sinks, self.window = spec, pe, capacity, sinks, window
        self.w, at = {}, 0
        for name, r, c, _ in inventory(spec):
            self.w[name] = flat[at:at + r * c].reshape(r, c).astype(np.float64)
            at += r * c
        self.total, self.margin = 0, 1.0
        self.cache = [dict() for _ in range(spec.layers)]

    def _norm(self, x, gamma, beta):
        if self.spec.architecture_flags & RMSNORM:
            return gamma * x / np.sqrt((x * x).mean() + 1e-6)
        return gamma * (x - x.mean()) / np.sqrt(x.var() + 1e-6) + beta

    def _held(self, x):
        x = x.astype(np.float32)
        codes, scales, scaled = fb.quantize_rows(x)
        self.margin = min(self.margin, np.abs(np.abs(scaled) % 1 - 0.5).min())
        return (codes - 7) * scales.astype(np.float64).repeat(64, -1)

    def forward(self, token):
        s, w, pos = self.spec, self.w, self.total
        d, heads = s.dim, s.heads
        hd = d // heads
        rope = s.architecture_flags & ROPE
        h = w["token_embeddings"][token] + (0 if rope else self.pe[pos])
        seen = fb.visible(pos, pos, self.sinks, self.capacity, self.window)
        for l in range(s.layers):
            p = f"layer{l}."
            q, k, v = ((h @ w[p + n]).reshape(1, heads, hd) for n in ("W_q", "W_k", "W_v"))
            if rope:
                q, k = (fb.norm_rotate(t, None, 0, np.array([pos]), 1e4, False)[0] for t in (q, k))
            self.cache[l][pos] = (self._held(k[0]), self._held(v[0]))
            out = np.empty((heads, hd))
            for i in range(heads):
                kk, vv = (np.stack([self.cache[l][j][n][i] for j in seen]) for n in (0, 1))
                e = kk @ q[0, i] / np.sqrt(hd)
                e = np.exp(e - e.max())
                out[i] = (e / e.sum()) @ vv
            a = self._norm(out.reshape(d) @ w[p + "W_o"] + h, w[p + "ln_gamma_attn"][0],
                           w.get(p + "ln_beta_attn", [0])[0])
            f = np.maximum(a @ w[p + "W_ff1"] + w[p + "b_ff1"][0], 0) @ w[p + "W_ff2"] + w[p + "b_ff2"][0]
            h = self._norm(f + a, w[p + "ln_gamma_ffn"][0], w.get(p + "ln_beta_ffn", [0])[0])
        self.total += 1
        return h @ w["output_projection"] + w["output_bias"][0]


CASES = [  # spec, bits, capacity, sinks, window, tokens
    (Spec(300, 128, 2, 2, 16), 8, 16, 0, 0, 10),
    (Spec(300, 128, 2, 2, 16), 4, 6, 2, 0, 12),
    (Spec(300, 128, 1, 2, 24, ROPE | RMSNORM), 8, 9, 1, 4, 14),
    (Spec(300, 256, 4, 1, 16, ROPE), 4, 12, 0, 5, 9),
]


def _inputs(gpu, oracle, case, batch=2):
    spec, bits, capacity, sinks, window, tokens = case
    pe = gpu.positional_encoding(64, spec.dim)
    for seed in range(50):
        params = synth_params(oracle, spec, 100 + seed)
        for (name, *_), t in zip(inventory(spec), params):
            if name.endswith(("W_q", "W_k")):
                t *= 4          # attention that prefers some tokens
        recs, flat = quantize_params(oracle, spec, params, bits)
        ids = np.random.RandomState(seed).randint(0, 256, (batch, tokens)).astype(np.uint32)
        logits, margin = [], 1.0
        for b in range(batch):
            e = Emulated(spec, flat, pe, capacity, sinks, window)
            logits.append([e.forward(int(t)) for t in ids[b]])
            margin = min(margin, e.margin)
        if margin > 2e-5:
            model = gpu.Model.from_arrays(spec, [(k, r, c, f, s, p, bits, 2) for (_, k, r, c, f, s, p) in recs])
            return model, ids, np.array(logits)
    raise AssertionError("no inputs away from every border")


def _close(got, want):
    err = np.abs(got - want).max(-1) / np.abs(want).max(-1)
    assert (err <= LOGIT_TOL).all(), err


@pytest.mark.parametrize("case", CASES)
def test_decode_steps(gpu, oracle, case):
    model, ids, want = _inputs(gpu, oracle, case)
    cache = gpu.KVCache(model, 2, case[2], kv_bits=4, sinks=case[3], window=case[4])
    assert not cache.uses_fused()
    for rep in range(2):
        for t in range(case[5]):
            _close(cache.forward_tokens(ids[:, t]), want[:, t])
        cache.reset()
    # one sequence restarted on its own: the other goes on
    for t in range(3):
        cache.forward_tokens(ids[:, t])
    cache.reset(np.array([1, 0], np.uint8))
    got = cache.forward_tokens(np.array([ids[0, 0], ids[1, 3]], np.uint32))
    _close(got, np.stack([want[0, 0], want[1, 3]]))
    cache.close()
    model.close()


@pytest.mark.parametrize("case", CASES)
def test_prefill_and_generate(gpu, oracle, case):
    spec, bits, capacity, sinks, window, tokens = case
    model, ids, want = _inputs(gpu, oracle, case)
    cache = gpu.KVCache(model, 2, capacity, kv_bits=4, sinks=sinks, window=window)
    most = min(tokens, capacity - sinks - (window - 1 if window else 0))
    if most >= 3:
        _close(cache.prefill(ids[:, :most]), want[:, most - 1])
        lens = [most, most - 2]
        got = cache.prefill(ids[:, :most], lens)
        _close(got, np.stack([want[b, n - 1] for b, n in enumerate(lens)]))
        if most < tokens:       # the short sequence's padding is overwritten
            got = cache.forward_tokens(np.array([ids[b, n] for b, n in enumerate(lens)], np.uint32))
            _close(got, np.stack([want[b, n] for b, n in enumerate(lens)]))
    if most < tokens:
        with pytest.raises(gpu.DzError) as e:
            cache.prefill(ids[:, :most + 1])
        assert e.value.status == -6
    # the generation loop draws what the steps draw, with either prefill
    greedy = gpu.Sampling(gpu.GREEDY, masked=())
    n_prompt = max(2, min(most, 4))
    streams = []
    for mode in (gpu.PREFILL_TOKENS, gpu.PREFILL_BATCHED):
        cache.set_prefill(mode)
        streams.append(cache.generate(ids[:, :n_prompt], 5, greedy))
    cache.reset()
    for t in range(n_prompt):
        logits = cache.forward_tokens(ids[:, t])
    drawn = []
    for _ in range(5):
        drawn.append(cache.select(greedy))
        logits = cache.forward_tokens(drawn[-1])
    assert np.isfinite(logits).all()
    np.testing.assert_array_equal(streams[0], np.stack(drawn, 1))
    np.testing.assert_array_equal(streams[1], streams[0])
    cache.close()
    model.close()


def test_wide_model_prefills_in_one_pass(gpu, oracle):
    """Wide enough for the tensor-core products: 40 prompt tokens of 5 sequences
    in one pass against token by token. The two round their products apart, so
    a code may differ: logits within 5e-2, the step of a 4-bit code."""
    spec = Spec(300, 512, 4, 2, 64)
    recs, _ = quantize_params(oracle, spec, synth_params(oracle, spec, 3), 8)
    model = gpu.Model.from_arrays(spec, [(k, r, c, f, s, p, 8, 2) for (_, k, r, c, f, s, p) in recs])
    cache = gpu.KVCache(model, 5, 64, kv_bits=4, sinks=4)
    ids = np.random.RandomState(0).randint(0, 256, (5, 40)).astype(np.uint32)
    one = cache.prefill(ids)
    cache.reset()
    for t in range(40):
        each = cache.forward_tokens(ids[:, t])
    err = np.abs(one - each).max(-1) / np.abs(each).max(-1)
    assert (err <= 5e-2).all(), err
    cache.close()
    model.close()


def test_refusals(gpu, oracle):
    spec = Spec(300, 128, 2, 1, 16)
    recs, _ = quantize_params(oracle, spec, synth_params(oracle, spec, 3), 8)
    make = lambda s: gpu.Model.from_arrays(s, [(k, r, c, f, sc, p, 8, 2) for (_, k, r, c, f, sc, p) in recs])  # noqa: E731
    model = make(spec)
    for bad in (dict(sinks=16), dict(window=17), dict(sinks=4, window=13), dict(capacity=17)):
        kw = dict(capacity=16, kv_bits=4)
        kw.update(bad)
        with pytest.raises(gpu.DzError) as e:
            gpu.KVCache(model, 1, **kw)
        assert e.value.status == -1
    for bad in (dict(kv_bits=8), dict(sinks=1), dict(window=4)):
        with pytest.raises(ValueError):
            gpu.KVCache(model, 1, 16, **bad)
    cache = gpu.KVCache(model, 1, 16, kv_bits=4)
    with pytest.raises(gpu.DzError) as e:
        cache.forward_masked(np.zeros((1, 4), np.uint32))
    assert e.value.status == -6
    with pytest.raises(gpu.DzError) as e:
        cache.set_path(cache.PATH_FUSED)
    assert e.value.status == -6
    cache.close()
    model.close()
    narrow = make(Spec(300, 128, 4, 1, 16))
    with pytest.raises(gpu.DzError) as e:
        gpu.KVCache(narrow, 1, 16, kv_bits=4)
    assert e.value.status == -6
    narrow.close()
