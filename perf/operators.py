"""Measured cases of the 4-bit serving operators.

Four operators, each in a plain form (elementary torch operations) and as the
framework's own calls:

  matvec   y = x . W with W in 4-bit codes and one scale per group of rows of
           a column (GroupedWeightMatrix.matmul_async)
  append   norms of queries and keys for each head, the position rotation, and
           the new keys and values quantized into a 4-bit ring cache, in one
           pass (KV4Cache.append)
  attend   attention over the 4-bit ring cache, every retained token visible
           (KV4Cache.attention)
  window   the same with a sliding window and a few first tokens that stay
           visible (KV4Cache.attention with window and sinks)

and `step`, append followed by attend over what was just appended.

Formulas. Codes c are 4-bit, level c - 7 in -7..7, value = scale * level. A
group's scale is fp32(peak / 7), its codes clamp(round_half_away(x * fp32(7 /
peak))) + 7, as the framework's quantizer. Cache rows have one scale per 64
elements. Ring: position p lives in slot p while p < sinks, else in slot
sinks + (p - sinks) mod (capacity - sinks).
"""
import math

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
GROUP = 64   # elements of a cache row that share a scale


# ------------------------------------------------------------------- cases

def listed():
    return [
        # a small projection for one token: the latency of a call
        dict(name="matvec small", op="matvec", m=1, k=2048, n=2048, group=128, type="f32", scales="f32"),
        # the vocabulary head for one token
        dict(name="matvec head", op="matvec", m=1, k=4096, n=32000, group=128, type="f32", scales="f16"),
        # an up-projection for eight sequences in 16 bits
        dict(name="matvec batch", op="matvec", m=8, k=2048, n=8192, group=64, type="bf16", scales="f32"),
        # odd sizes, a short last group, sixteen rows
        dict(name="matvec odd", op="matvec", m=16, k=4099, n=5003, group=32, type="f16", scales="f32"),
        # one decode step of 256 sequences, normed and rotated
        dict(name="append decode", op="append", batch=256, tokens=1, q_heads=16, kv_heads=16, dim=128, capacity=704,
             sinks=0, past=640, norm=True, rope=10000.0, halves=False, type="f32"),
        # a prompt of four sequences, shared key heads, second half of a head rotated against the first
        dict(name="append prompt", op="append", batch=4, tokens=1900, q_heads=32, kv_heads=8, dim=64, capacity=2048,
             sinks=4, past=0, norm=True, rope=500000.0, halves=True, type="bf16"),
        # one sequence, a short context: the latency of a call
        dict(name="attend small", op="attend", batch=1, tokens=1, q_heads=16, kv_heads=16, dim=64, capacity=1024,
             sinks=0, window=0, past=601, type="f32"),
        # one decode step of 256 sequences of different lengths
        dict(name="attend batch", op="attend", batch=256, tokens=1, q_heads=16, kv_heads=16, dim=128, capacity=704,
             sinks=0, window=0, past=640, type="f32"),
        # two long contexts, four query heads to a key head
        dict(name="attend long", op="attend", batch=2, tokens=1, q_heads=32, kv_heads=8, dim=128, capacity=131072,
             sinks=0, window=0, past=130001, type="bf16"),
        # a ring that has wrapped many times, with first tokens kept
        dict(name="window decode", op="window", batch=32, tokens=1, q_heads=16, kv_heads=16, dim=128, capacity=2052,
             sinks=4, window=1024, past=100003, type="f32"),
        # sixteen drafted tokens of each sequence at once
        dict(name="window chunk", op="window", batch=8, tokens=16, q_heads=32, kv_heads=4, dim=64, capacity=4352,
             sinks=64, window=4096, past=9001, type="f16"),
        # append and attend of one small decode step, one after the other
        dict(name="step", op="step", batch=8, tokens=1, q_heads=16, kv_heads=16, dim=128, capacity=2048, sinks=0,
             window=0, past=1500, norm=True, rope=10000.0, halves=False, type="f32"),
    ]


def _spread(rng, lo, hi):
    """A whole number whose logarithm is uniform over lo..hi."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["matvec", "matvec", "append", "attend", "window", "step"])
    if op == "matvec":
        m = _spread(rng, 1, 20)
        k = _spread(rng, 100, 12000)
        n = _spread(rng, 16, min(40000, 120_000_000 // k))
        if rng.random() < 0.5:
            k, n = -(-k // 128) * 128, -(-n // 16) * 16
        return dict(op=op, m=m, k=k, n=n, group=rng.choice([32, 64, 128]), type=rng.choice(sorted(TYPES)),
                    scales=rng.choice(["f16", "f32"]))
    dim = rng.choice([64, 128])
    kv_heads = rng.choice([1, 2, 4, 8, 12, 16])
    q_heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 8])
    kind = rng.choice(sorted(TYPES))
    if op == "append":
        most = 20_000_000 // ((q_heads + 2 * kv_heads) * dim)      # tokens of all sequences
        tokens = rng.choice([1, 1, _spread(rng, 2, min(2000, most))])
        batch = _spread(rng, 1, max(1, min(256, most // tokens)))
        sinks = rng.choice([0, 4, 33])
        return dict(op=op, batch=batch, tokens=tokens, q_heads=q_heads, kv_heads=kv_heads, dim=dim,
                    capacity=tokens + sinks + _spread(rng, 1, 1000), sinks=sinks, past=_spread(rng, 1, 100000) - 1,
                    norm=rng.random() < 0.8, rope=rng.choice([0.0, 10000.0, 1000000.0]), halves=rng.random() < 0.5,
                    type=kind)
    tokens = 1 if op == "step" else rng.choice([1, 1, 1, 2, 5, 24])
    batch = _spread(rng, 1, 64)
    most = max(64, min(100000, 2_000_000 // (batch * kv_heads * tokens)))
    past = _spread(rng, 1, most)
    case = dict(op=op, batch=batch, tokens=tokens, q_heads=q_heads, kv_heads=kv_heads, dim=dim,
                capacity=past + tokens + rng.randrange(40), sinks=0, window=0, past=past, type=kind)
    if op == "step":
        case.update(norm=True, rope=10000.0, halves=rng.random() < 0.5)
    if op == "window":
        sinks, window = rng.choice([0, 1, 4, 64]), _spread(rng, 1, most)
        case.update(sinks=sinks, window=window, capacity=sinks + window + tokens + rng.randrange(300),
                    past=_spread(rng, 1, 200000))
    return case


# ------------------------------------------------------------------ inputs

def _positions(case):
    """Position of each sequence's first new token: sequences differ in length."""
    past, batch = case["past"], case["batch"]
    return [past - (37 * b) % max(1, past // 4) for b in range(batch)]


def _codes(x, dim):
    """(codes, scale) of x quantized in groups along `dim`, whose extent is one group."""
    peak = x.abs().amax(dim, keepdim=True)
    seven = torch.full_like(peak, 7.0)         # a tensor: a division by or of a number rounds twice
    v = x * torch.where(peak > 0, seven / peak, torch.zeros_like(peak))
    level = torch.where(v >= 0, torch.floor(v + 0.5), torch.ceil(v - 0.5)).clamp(-7, 7)
    return (level + 7).to(torch.uint8), peak / seven


def _pack(codes):
    """Codes two to a byte, the first in the low half."""
    flat = codes.reshape(-1)
    if flat.numel() % 2:
        flat = torch.cat([flat, flat.new_zeros(1)])
    return flat[0::2] | (flat[1::2] << 4)


def _weights(case, gen):
    k, n, g = case["k"], case["n"], case["group"]
    groups = -(-k // g)
    w = torch.randn(groups * g, n, device=DEV, generator=gen) * 0.02
    w[k:] = 0
    codes, scale = _codes(w.view(groups, g, n), 1)
    if case["scales"] == "f16":
        scale = scale.half()
    return _pack(codes.view(groups * g, n)[:k]), scale.view(groups, n).contiguous()


def _cache(case, gen):
    """A ring cache that holds `past` tokens of each sequence, every slot written."""
    shape = (case["batch"], case["kv_heads"], case["capacity"], case["dim"])
    out = {}
    channel = torch.exp(0.5 * torch.randn(1, case["kv_heads"], 1, case["dim"], device=DEV, generator=gen))
    for name in ("k", "v"):
        x = torch.randn(shape, device=DEV, generator=gen)
        if name == "k":
            x *= channel / channel.square().mean(-1, keepdim=True).sqrt()
        codes, scale = _codes(x.view(*shape[:3], shape[3] // GROUP, GROUP), -1)
        del x
        out[name + "_codes"] = _pack(codes).view(*shape[:3], shape[3] // 2)
        out[name + "_scales"] = scale.squeeze(-1).contiguous()
    return out


def prepare(case, seed):
    gen = torch.Generator(DEV)
    gen.manual_seed(seed)
    kind = TYPES[case["type"]]
    s = dict(case)
    if case["op"] == "matvec":
        s["packed"], s["w_scales"] = _weights(case, gen)
        x = torch.randn(case["m"], case["k"], device=DEV, generator=gen)
        x *= torch.exp(0.7 * torch.randn(case["k"], device=DEV, generator=gen))   # some channels are large
        s["x"] = x.to(kind)
        if own:
            import dranzer_b200 as dz
            s["w"] = dz.GroupedWeightMatrix.from_device(
                s["w_scales"].data_ptr(), s["packed"].data_ptr(), case["k"], case["n"], case["group"],
                dz.TYPE_F16 if case["scales"] == "f16" else dz.TYPE_F32)
        return s
    rows, dim = case["batch"] * case["tokens"], case["dim"]
    s["positions"] = torch.tensor(_positions(case), dtype=torch.int64, device=DEV)
    s.update(_cache(case, gen))
    if case["op"] in ("append", "step"):
        # one fused row of queries, keys and values for each token, as the projection writes it
        width = (case["q_heads"] + 2 * case["kv_heads"]) * dim
        s["qkv"] = torch.randn(rows, width, device=DEV, generator=gen).to(kind)
        if case["norm"]:
            s["q_gain"] = 1.0 + 0.2 * torch.randn(dim, device=DEV, generator=gen)
            s["k_gain"] = 1.0 + 0.2 * torch.randn(dim, device=DEV, generator=gen)
    else:
        s["q"] = (1.5 * torch.randn(rows, case["q_heads"] * dim, device=DEV, generator=gen)).to(kind)
    if own:
        import dranzer_b200 as dz
        s["cache"] = dz.KV4Cache(s["k_codes"].data_ptr(), s["v_codes"].data_ptr(), s["k_scales"].data_ptr(),
                                 s["v_scales"].data_ptr(), case["batch"], case["kv_heads"], dim, case["capacity"],
                                 case["sinks"])
    return s


# -------------------------------------------------------------- plain forms

def _unpack(packed, shape):
    """Levels -7..7 as fp32 of codes packed two to a byte."""
    count = math.prod(shape)
    pairs = torch.stack([packed & 15, packed >> 4], -1).reshape(-1)[:count]
    return pairs.view(shape).float() - 7.0


def _cached(s, name, used):
    """The first `used` slots of the keys or values, in fp32."""
    batch, hk, dim = s["batch"], s["kv_heads"], s["dim"]
    level = _unpack(s[name + "_codes"][:, :, :used], (batch, hk, used, dim // GROUP, GROUP))
    return (level * s[name + "_scales"][:, :, :used, :, None]).view(batch, hk, 1, used, dim)


def _plain_matvec(s):
    k, n, g = s["k"], s["n"], s["group"]
    scale = s["w_scales"].float().repeat_interleave(g, 0)[:k]
    return (s["x"].float() @ (_unpack(s["packed"], (k, n)) * scale)).to(s["x"].dtype)


def _token_positions(s):
    return s["positions"][:, None] + torch.arange(s["tokens"], device=DEV)


def _norm_rotate(x, gain, s):
    """RMS norm of each head (64 bits: the codes that follow round values next to a border), then the rotation."""
    x = x.double()
    if gain is not None:
        x = gain.double() * x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt()
    if not s["rope"]:
        return x
    half = s["dim"] // 2
    frequency = s["rope"] ** (-2.0 * torch.arange(half, device=DEV, dtype=torch.float64) / s["dim"])
    angle = (_token_positions(s).double()[..., None] * frequency)[:, :, None]
    c, d = angle.cos(), angle.sin()
    if s["halves"]:
        a, b = x[..., :half], x[..., half:]
        return torch.cat([a * c - b * d, a * d + b * c], -1)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * c - b * d, a * d + b * c], -1).flatten(-2)


def _plain_append(s):
    """Rotated queries, and keys and values as the cache now holds them; writes the cache."""
    batch, tokens, hq, hk, dim = s["batch"], s["tokens"], s["q_heads"], s["kv_heads"], s["dim"]
    kind = s["qkv"].dtype
    rows = s["qkv"].view(batch, tokens, hq + 2 * hk, dim)
    q = _norm_rotate(rows[:, :, :hq], s.get("q_gain"), s).to(kind)
    p = _token_positions(s)
    ring = s["capacity"] - s["sinks"]
    slot = torch.where(p < s["sinks"], p, s["sinks"] + (p - s["sinks"]) % ring)
    which = torch.arange(batch, device=DEV)[:, None]
    held = []
    for name, x in (("k", _norm_rotate(rows[:, :, hq:hq + hk], s.get("k_gain"), s).float()),
                    ("v", rows[:, :, hq + hk:].float())):
        codes, scale = _codes(x.reshape(batch, tokens, hk, dim // GROUP, GROUP), -1)
        s[name + "_codes"][which, :, slot] = _pack(codes).view(batch, tokens, hk, dim // 2)
        s[name + "_scales"][which, :, slot] = scale.squeeze(-1)
        held.append(((codes.float() - 7.0) * scale).view(batch * tokens, hk * dim).to(kind))
    return q.reshape(batch * tokens, hq * dim), held[0], held[1]


def _plain_attend(s, q):
    batch, tokens, hq, hk, dim, cap = (s[n] for n in ("batch", "tokens", "q_heads", "kv_heads", "dim", "capacity"))
    used = min(cap, s["past"] + tokens)                        # slots written in the longest sequence
    i = _token_positions(s)                                    # position of each query
    slot = torch.arange(used, device=DEV)
    ring, last = cap - s["sinks"], i[:, -1:]
    held = last - (last - slot) % ring                         # newest position of a ring slot
    held = torch.where(slot < s["sinks"], slot, held)          # what each slot holds
    held = torch.where((slot >= s["sinks"]) & (held < s["sinks"]), torch.full_like(held, -1), held)
    seen = (held[:, None] >= 0) & (held[:, None] <= i[..., None])
    if s["window"]:
        seen &= (held[:, None] > i[..., None] - s["window"]) | (slot < s["sinks"])
    k = _cached(s, "k", used)
    x = q.float().view(batch, tokens, hk, hq // hk, dim).permute(0, 2, 3, 1, 4)
    x = (x @ k.transpose(-1, -2)) / math.sqrt(dim)             # [batch, hk, share, tokens, used]
    del k
    x = x.masked_fill(~seen[:, None, None], -math.inf)
    x = (x - x.amax(-1, keepdim=True)).exp()
    x = x / x.sum(-1, keepdim=True)
    v = _cached(s, "v", used)
    return (x @ v).permute(0, 3, 1, 2, 4).reshape(batch * tokens, hq * dim).to(q.dtype)


# ------------------------------------------------------------------- passes

def _own_type(tensor):
    import dranzer_b200 as dz
    return {torch.float32: dz.TYPE_F32, torch.float16: dz.TYPE_F16, torch.bfloat16: dz.TYPE_BF16}[tensor.dtype]


def _own_append(s):
    x = s["qkv"]
    hq, hk, dim, width = s["q_heads"], s["kv_heads"], s["dim"], x.shape[1]
    size, base = x.element_size(), x.data_ptr()
    q, k, v = (x.new_empty(x.shape[0], h * dim) for h in (hq, hk, hk))
    s["cache"].append(
        s["positions"].data_ptr(), s["tokens"], type=_own_type(x), q_heads=hq, q=base, k=base + hq * dim * size,
        v=base + (hq + hk) * dim * size, q_stride=width, k_stride=width, v_stride=width, q_out=q.data_ptr(),
        k_out=k.data_ptr(), v_out=v.data_ptr(), q_gain=s["q_gain"].data_ptr() if s["norm"] else None,
        k_gain=s["k_gain"].data_ptr() if s["norm"] else None, eps=1e-6, rope_base=s["rope"], halves=s["halves"],
        stream_ptr=torch.cuda.current_stream().cuda_stream)
    return q, k, v


def _own_attend(s, q):
    out = torch.empty_like(q)
    s["cache"].attention(
        s["positions"].data_ptr(), s["tokens"], type=_own_type(q), q_heads=s["q_heads"], q=q.data_ptr(),
        out=out.data_ptr(), window=s["window"], stream_ptr=torch.cuda.current_stream().cuda_stream)
    return out


def run(s):
    op = s["op"]
    if op == "matvec":
        if not own:
            return _plain_matvec(s)
        x = s["x"]
        y = x.new_empty(s["m"], s["n"])
        s["w"].matmul_async(x.data_ptr(), y.data_ptr(), s["m"], torch.cuda.current_stream().cuda_stream,
                            type=_own_type(x))
        return y
    if op == "append":
        return _own_append(s) if own else _plain_append(s)
    if op == "step":
        q, k, v = _own_append(s) if own else _plain_append(s)
        return (_own_attend(s, q) if own else _plain_attend(s, q)), k, v
    return _own_attend(s, s["q"]) if own else _plain_attend(s, s["q"])


# --------------------------------------------------------------------- work

def _visible(case):
    """Over all sequences: cached tokens that a pass has to read, and (query, token) pairs that it scores."""
    rows = pairs = 0
    n, sinks, window = case["tokens"], case["sinks"], case["window"]
    for first in _positions(case):
        last = first + n - 1
        oldest = max(sinks, last - (case["capacity"] - sinks) + 1)
        reach = lambda i: max(oldest, i - window + 1) if window else oldest  # noqa: E731
        rows += min(sinks, last + 1) + max(0, last + 1 - max(sinks, reach(first)))
        pairs += sum(min(sinks, i + 1) + max(0, i + 1 - max(sinks, reach(i))) for i in range(first, last + 1))
    return rows, pairs


def work(case):
    size = 4 if case["type"] == "f32" else 2
    if case["op"] == "matvec":
        m, k, n = case["m"], case["k"], case["n"]
        scales = -(-k // case["group"]) * n * (4 if case["scales"] == "f32" else 2)
        return {"bytes": k * n / 2 + scales + m * (k + n) * size, "flops": 2.0 * m * k * n}
    rows, dim, hq, hk = case["batch"] * case["tokens"], case["dim"], case["q_heads"], case["kv_heads"]
    row = dim / 2 + dim / GROUP * 4          # bytes of one cached row of keys or values
    total = {"bytes": 0.0, "flops": 0.0}
    if case["op"] in ("append", "step"):
        total["bytes"] += rows * dim * size * (2 * hq + 4 * hk) + rows * hk * 2 * row
        total["flops"] += rows * (hq + hk) * dim * 8.0 + rows * hk * dim * 8.0
    if case["op"] != "append":
        tokens, pairs = _visible(case)
        total["bytes"] += tokens * hk * 2 * row + 2 * rows * hq * dim * size
        total["flops"] += pairs * hq * dim * 4.0
    return total


# -------------------------------------------------------------------- exact

def _values(packed, scales, group_axis_len):
    """64-bit values of a [..., bytes] code array with one scale per `group_axis_len` elements of a row."""
    low, high = (packed & 0x0F).double(), torch.div(packed, 16, rounding_mode="floor").double()
    level = torch.empty(*packed.shape[:-1], packed.shape[-1] * 2, dtype=torch.float64, device=packed.device)
    level[..., 0::2], level[..., 1::2] = low - 7, high - 7
    return level * scales.double().repeat_interleave(group_axis_len, -1)


def _exact_matvec(s):
    k, n, g = s["k"], s["n"], s["group"]
    out = torch.zeros(s["m"], n, dtype=torch.float64, device=DEV)
    step = 2 * max(1, 4096 // (2 * g)) * g      # whole groups, and whole bytes at any n
    for r in range(0, k, step):
        rows = min(step, k - r)
        b = s["packed"][r * n // 2: r * n // 2 + -(-rows * n // 2)]
        level = torch.empty(2 * b.numel(), dtype=torch.float64, device=DEV)
        level[0::2], level[1::2] = (b % 16).double() - 7, (b // 16).double() - 7
        scale = s["w_scales"][r // g: r // g + -(-rows // g)].double()
        w = level[:rows * n].view(rows, n) * scale[torch.arange(rows, device=DEV) // g]
        out += s["x"][:, r:r + rows].double() @ w
    return out


def _exact_append(s):
    """Token by token over the batch: complex numbers for the rotation, the quantizer's fp32 steps for the codes."""
    hq, hk, dim, n = s["q_heads"], s["kv_heads"], s["dim"], s["tokens"]
    x = s["qkv"].double().view(s["batch"], n, hq + 2 * hk, dim)
    q, k, v = x[:, :, :hq], x[:, :, hq:hq + hk], x[:, :, hq + hk:]
    where = s["positions"].double().view(-1, 1, 1, 1) + torch.arange(n, dtype=torch.float64, device=DEV).view(1, -1, 1, 1)

    def turned(y, gain):
        if s["norm"]:
            y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / dim + 1e-6) * gain.double()
        if s["rope"]:
            speed = torch.exp(-torch.arange(0, dim, 2, dtype=torch.float64, device=DEV) / dim * math.log(s["rope"]))
            spin = torch.polar(torch.ones((), dtype=torch.float64, device=DEV), where * speed)
            a = y.unflatten(-1, (2, dim // 2)).transpose(-1, -2) if s["halves"] else y.unflatten(-1, (dim // 2, 2))
            z = torch.view_as_real(torch.view_as_complex(a.contiguous()) * spin)
            y = (z.transpose(-1, -2) if s["halves"] else z).flatten(-2)
        return y

    def stored(y):
        y = y.float().unflatten(-1, (dim // GROUP, GROUP))
        top = y.abs().max(-1, keepdim=True).values
        most = torch.full_like(top, 7.0)
        t = y * (most / top)
        level = torch.sign(t) * torch.floor(t.abs() + 0.5)
        level = torch.nan_to_num(level, nan=0.0).clamp(-7, 7)
        return level.to(torch.int8), (top / most).squeeze(-1)

    held = [stored(turned(k, s.get("k_gain"))), stored(v)]
    rows = [(level.double() * scale.double().unsqueeze(-1)).flatten(-2) for level, scale in held]
    return turned(q, s.get("q_gain")), rows[0], rows[1], held


def _exact_attend(s, q, late=None):
    """Sequence by sequence over positions, not slots. `late`: levels and scales of the tokens that this pass appended."""
    hq, hk, dim, n, sinks = s["q_heads"], s["kv_heads"], s["dim"], s["tokens"], s["sinks"]
    ring, share = s["capacity"] - sinks, hq // hk
    out = torch.empty(s["batch"], n, hq, dim, dtype=torch.float64, device=DEV)
    q = q.double().view(s["batch"], n, hk, share, dim)
    for b, first in enumerate(_positions(s)):
        last = first + n - 1
        oldest = max(sinks, last - ring + 1)
        if s["window"]:
            oldest = max(oldest, first - s["window"] + 1)
        p = torch.cat([torch.arange(min(sinks, last + 1)), torch.arange(oldest, max(oldest, last + 1))]).to(DEV)
        slot = torch.where(p < sinks, p, sinks + torch.remainder(p - sinks, ring))
        k, v = (_values(s[x + "_codes"][b, :, slot], s[x + "_scales"][b, :, slot], GROUP) for x in ("k", "v"))
        if late is not None:
            k, v = (torch.cat([old[:, :-n], new[b].double().transpose(0, 1)], 1) for old, new in zip((k, v), late))
        for t in range(n):
            i = first + t
            sees = p <= i
            if s["window"]:
                sees &= (p < sinks) | (i - p < s["window"])
            kt, vt = k[:, sees], v[:, sees]
            e = torch.einsum("hgd,hpd->hgp", q[b, t], kt) * dim ** -0.5
            out[b, t] = torch.einsum("hgp,hpd->hgd", torch.softmax(e, -1), vt).reshape(hq, dim)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    flat = lambda x: x.reshape(case["batch"] * case["tokens"], -1)  # noqa: E731
    if case["op"] == "matvec":
        return _exact_matvec(s)
    if case["op"] == "append":
        q, k, v, _ = _exact_append(s)
        return flat(q), flat(k), flat(v)
    if case["op"] == "step":
        q, k, v, _ = _exact_append(s)
        kind = TYPES[case["type"]]
        return flat(_exact_attend(s, q.to(kind), (k, v))), flat(k), flat(v)
    return flat(_exact_attend(s, s["q"]))
