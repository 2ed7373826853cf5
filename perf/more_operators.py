"""Measured cases of the 8-bit serving operators.

Four operators, each in a plain form (elementary torch operations) and as the
framework's own calls:

  norm     h = x + residual, the root-mean-square norm of h, and the rows in 8
           bits with a scale each; without the norm, rows in 8 bits (norm_q8)
  product  y = (a . w) times a scale for each row and one for each column, with
           a bias: a in 8 bits (what norm leaves), w the levels of a quantized
           matrix (QuantizedWeightMatrix.matmul_q8_async)
  append   norms of queries and keys for each head, the position rotation, and
           the new keys and values quantized into the pages of an 8-bit cache,
           in one pass (KV8Cache.append)
  attend   attention over the pages of an 8-bit cache, causal, with an optional
           window (KV8Cache.attention)

Formulas. An 8-bit code c is -127..127, value = scale * c.
  norm: h is rounded to its type, u = fp32(gain * h), P the largest |u| of a
  row, code = fp32(u * fp32(127 / P)) rounded half away from zero, scale =
  P / sqrt(mean(h^2) + eps) / 127, or P / 127 without the norm. Rows whose P
  lies below 2^-100 take u and P times 2^100 for their codes.
  cache: a page holds `page` consecutive tokens of a sequence, and the keys of
  a page and head have one scale S, the values another. A page whose first
  token is new gets S = fp32(peak / 127) of its new rows; one that holds
  earlier tokens keeps S where that is not below the new rows' peak / 127, and
  else takes the latter, its earlier codes becoming fp32(c * fp32(old S / S))
  rounded half away from zero. New codes are fp32(x * fp32(1 / S)) rounded half
  away from zero and held to -127..127.
"""
import math

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6


# ------------------------------------------------------------------- cases

def listed():
    return [
        # the residual rows of a small decode step: the latency of a call
        dict(name="norm decode", op="norm", rows=8, width=2048, pad=0, residual=True, norm=True, gain=True, type="f32"),
        # the residual stream of a prefill
        dict(name="norm prefill", op="norm", rows=8192, width=4096, pad=0, residual=True, norm=True, gain=True,
             type="bf16"),
        # odd rows of a wider buffer quantized alone, as before a projection that has no norm
        dict(name="norm odd", op="norm", rows=777, width=5003, pad=5, residual=False, norm=False, gain=False, type="f16"),
        # a square projection for eight sequences: the latency of a call
        dict(name="product small", op="product", m=8, k=2048, n=2048, bias=False, type="bf16"),
        # the vocabulary head for one token
        dict(name="product head", op="product", m=1, k=4096, n=32000, bias=True, type="f32"),
        # odd sizes, rows enough for several tiles of rows
        dict(name="product odd", op="product", m=131, k=4099, n=5003, bias=True, type="f16"),
        # an up-projection of a prefill
        dict(name="product prefill", op="product", m=4096, k=4096, n=16384, bias=True, type="bf16"),
        # a decode step of many short sequences
        dict(name="append decode", op="append", batch=256, tokens=1, q_heads=16, kv_heads=16, dim=128, page=32, past=150,
             norm=False, rope=0.0, halves=False, type="f32"),
        # a chunk of a prefill, pages begun and pages gone on with
        dict(name="append chunk", op="append", batch=4, tokens=2000, q_heads=32, kv_heads=8, dim=128, page=64, past=777,
             norm=True, rope=10000.0, halves=True, type="bf16"),
        # one short sequence: the latency of a call
        dict(name="attend small", op="attend", batch=1, tokens=1, q_heads=16, kv_heads=16, dim=64, page=32, past=600,
             window=0, type="f32"),
        # sequences of very different lengths, four query heads to a key head
        dict(name="attend ragged", op="attend", batch=24, tokens=1, q_heads=32, kv_heads=8, dim=128, page=64, past=32001,
             window=0, type="bf16"),
        # sixteen drafted tokens of each sequence at once, within a window
        dict(name="attend drafts", op="attend", batch=8, tokens=16, q_heads=32, kv_heads=4, dim=64, page=32, past=9001,
             window=4096, type="f16"),
    ]


def _spread(rng, lo, hi):
    """A whole number whose logarithm is uniform over lo..hi."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "product", "product", "append", "attend", "attend"])
    kind = rng.choice(sorted(TYPES))
    if op == "norm":
        rows = _spread(rng, 1, 16384)
        width = _spread(rng, 16, min(20000, 33_000_000 // rows))
        if rng.random() < 0.5:
            width = -(-width // 128) * 128
        return dict(op=op, rows=rows, width=width, pad=rng.choice([0, 0, 3, 64]), residual=rng.random() < 0.6,
                    norm=rng.random() < 0.7, gain=rng.random() < 0.7, type=kind)
    if op == "product":
        m = rng.choice([_spread(rng, 1, 64), _spread(rng, 1, 4096)])
        k = _spread(rng, 64, 16384)
        n = _spread(rng, 16, min(32000, 130_000_000 // k, 270_000_000_000 // (m * k)))
        if rng.random() < 0.5:
            k, n = -(-k // 128) * 128, -(-n // 16) * 16
        return dict(op=op, m=m, k=k, n=n, bias=rng.random() < 0.5, type=kind)
    dim, page = rng.choice([64, 128]), rng.choice([32, 64])
    kv_heads = rng.choice([1, 2, 4, 8, 12, 16])
    q_heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 8])
    if op == "append":
        most = 20_000_000 // ((q_heads + 2 * kv_heads) * dim)      # tokens of all sequences
        tokens = rng.choice([1, 1, _spread(rng, 2, min(2000, most))])
        batch = _spread(rng, 1, max(1, min(256, most // tokens)))
        return dict(op=op, batch=batch, tokens=tokens, q_heads=q_heads, kv_heads=kv_heads, dim=dim, page=page,
                    past=_spread(rng, 1, 2000) - 1, norm=rng.random() < 0.7, rope=rng.choice([0.0, 10000.0, 1000000.0]),
                    halves=rng.random() < 0.5, type=kind)
    tokens = rng.choice([1, 1, 1, 2, 5, 24])
    batch = _spread(rng, 1, 64)
    past = _spread(rng, 1, max(64, min(100000, 4_000_000 // (batch * kv_heads * tokens)))) - 1
    return dict(op=op, batch=batch, tokens=tokens, q_heads=q_heads, kv_heads=kv_heads, dim=dim, page=page, past=past,
                window=rng.choice([0, 0, _spread(rng, 1, past + tokens)]), type=kind)


# ------------------------------------------------------------------ inputs

def _positions(case):
    """Position of each sequence's first new token: the last sequence is about a third as long as the first."""
    past, batch = case["past"], case["batch"]
    return [past - past * 2 * b // (3 * batch) for b in range(batch)]


def _pages(case):
    """Pages of the longest sequence."""
    return (case["past"] + case["tokens"] - 1) // case["page"] + 1


def prepare(case, seed):
    gen = torch.Generator(DEV)
    gen.manual_seed(seed)
    randn = lambda *shape: torch.randn(*shape, device=DEV, generator=gen)  # noqa: E731
    kind = TYPES[case["type"]]
    s = dict(case)
    if case["op"] == "norm":
        rows, width, pad = case["rows"], case["width"], case["pad"]
        for name in ("x", "residual"):
            if name == "x" or case["residual"]:
                t = randn(rows, width + pad)
                t *= torch.exp(0.7 * randn(width + pad))           # some channels are large
                s[name + "_rows"] = t.to(kind)[:, :width]
        s["g"] = 1.0 + 0.2 * randn(width) if case["gain"] else None
        return s
    if case["op"] == "product":
        m, k, n = case["m"], case["k"], case["n"]
        lda = -(-k // 16) * 16                                     # rows of codes start on 16-byte boundaries
        s["codes"] = (36.0 * randn(m, lda)).round_().clamp_(-127, 127).to(torch.int8)
        s["a_scales"] = torch.exp(0.5 * randn(m)) / 36.0
        s["levels"] = torch.empty(k, n, dtype=torch.int8, device=DEV)
        for r in range(0, k, 1024):
            level = (32.0 * randn(min(1024, k - r), n)).round_().clamp_(-127, 127)
            s["levels"][r:r + 1024] = level.to(torch.int8)
        s["w_scales"] = 0.02 * torch.exp(0.2 * randn(n)) / 32.0
        s["b"] = 0.1 * randn(n) if case["bias"] else None
        if own:
            import dranzer_b200 as dz
            packed = (s["levels"].view(torch.uint8) + 127).cpu().numpy()       # modulo 256: the stored code
            s["w"] = dz.QuantizedWeightMatrix(s["w_scales"].cpu().numpy(), packed.reshape(-1), k, n, 8)
        return s
    batch, hk, dim, page = (case[name] for name in ("batch", "kv_heads", "dim", "page"))
    per = _pages(case)
    pool = batch * per + 3                                         # pages that no sequence has are in the pool too
    s["positions"] = torch.tensor(_positions(case), dtype=torch.int64, device=DEV)
    s["table"] = torch.randperm(pool, device=DEV, generator=gen)[:batch * per].to(torch.int32).view(batch, per)
    for name in ("k", "v"):
        codes = torch.empty(pool, hk, page, dim, dtype=torch.int8, device=DEV)
        step = max(1, 2 ** 26 // (hk * page * dim))
        for p in range(0, pool, step):
            x = randn(min(step, pool - p), hk, page, dim)
            codes[p:p + step] = (32.0 * x).round_().clamp_(-127, 127).to(torch.int8)
        s[name + "_codes"] = codes
        s[name + "_scales"] = torch.exp(0.2 * randn(pool, hk)) / 32.0
    rows = batch * case["tokens"]
    if case["op"] == "append":
        # one fused row of queries, keys and values for each token, as the projection writes it
        s["qkv"] = randn(rows, (case["q_heads"] + 2 * hk) * dim).to(kind)
        if case["norm"]:
            s["q_gain"] = 1.0 + 0.2 * randn(dim)
            s["k_gain"] = 1.0 + 0.2 * randn(dim)
    else:
        s["q"] = (1.5 * randn(rows, case["q_heads"] * dim)).to(kind)
    if own:
        import dranzer_b200 as dz
        s["cache"] = dz.KV8Cache(s["k_codes"].data_ptr(), s["v_codes"].data_ptr(), s["k_scales"].data_ptr(),
                                 s["v_scales"].data_ptr(), pool, page, hk, dim, s["table"].data_ptr(), batch, per)
    return s


# -------------------------------------------------------------- plain forms

def _half_away(v):
    return torch.where(v >= 0, torch.floor(v + 0.5), torch.ceil(v - 0.5))


def _plain_norm(s):
    x = s["x_rows"]
    h = x.float()
    if s["residual"]:
        total = (h + s["residual_rows"].float()).to(x.dtype)
        h = total.float()
    u = h * s["g"] if s["gain"] else h
    peak = u.abs().amax(-1, keepdim=True)
    raised = torch.where(peak < 2.0 ** -100, 2.0 ** 100, 1.0).to(peak.dtype)
    most = torch.full_like(peak, 127.0)        # a tensor: a division by or of a number rounds twice
    v = (u * raised) * torch.where(peak > 0, most / (peak * raised), torch.zeros_like(peak))
    codes = _half_away(v).to(torch.int8)
    scales = peak / most
    if s["norm"]:
        scales = peak / (h.square().mean(-1, keepdim=True) + EPS).sqrt() / most
    return (codes, scales[:, 0]) + ((total,) if s["residual"] else ())


def _plain_product(s):
    y = s["codes"][:, :s["k"]].float() @ s["levels"].float()
    y = y * s["a_scales"][:, None] * s["w_scales"]
    if s["bias"]:
        y = y + s["b"]
    return y.to(TYPES[s["type"]])


def _token_positions(s):
    return s["positions"][:, None] + torch.arange(s["tokens"], device=DEV)


def _norm_rotate(x, gain, s):
    """RMS norm of each head (64 bits: the codes that follow round values next to a border), then the rotation."""
    x = x.double()
    if gain is not None:
        x = gain.double() * x / (x.square().mean(-1, keepdim=True) + EPS).sqrt()
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
    """Rotated queries, the new keys and values as the cache now holds them, and the cache, which it writes."""
    batch, tokens, hq, hk, dim, page = (s[n] for n in ("batch", "tokens", "q_heads", "kv_heads", "dim", "page"))
    kind = s["qkv"].dtype
    rows = s["qkv"].view(batch, tokens, hq + 2 * hk, dim)
    q = _norm_rotate(rows[:, :, :hq], s.get("q_gain"), s).to(kind)
    p = _token_positions(s)
    where = s["table"].long().gather(1, p // page)                 # page of each new token
    first = s["positions"] % page                                  # rows that the first page holds already
    begun = where[:, 0]
    held = []
    for name, x in (("k", _norm_rotate(rows[:, :, hq:hq + hk], s.get("k_gain"), s).float()),
                    ("v", rows[:, :, hq + hk:].float())):
        codes, scales = s[name + "_codes"], s[name + "_scales"]
        most = torch.full_like(scales, 127.0)
        peak = torch.zeros_like(scales)
        peak.scatter_reduce_(0, where.view(-1, 1).expand(-1, hk), x.abs().amax(-1).view(-1, hk), "amax")
        old = scales[begun]
        new = peak / most
        new[begun] = torch.where(first[:, None] > 0, torch.maximum(old, new[begun]), new[begun])
        ratio = torch.where((first[:, None] > 0) & (new[begun] > old), old / new[begun], torch.ones_like(old))
        was = codes[begun]
        again = _half_away(was.float() * ratio[:, :, None, None]).to(torch.int8)
        early = torch.arange(page, device=DEV) < first[:, None]
        codes[begun] = torch.where(early[:, None, :, None], again, was)
        touched = torch.zeros(scales.shape[0], 1, dtype=torch.bool, device=DEV)
        touched[where.reshape(-1)] = True
        scales.copy_(torch.where(touched, new, scales))
        scale = scales[where][..., None]
        one = torch.ones_like(scale)
        level = _half_away(x * torch.where(scale > 0, one / scale, torch.zeros_like(scale))).clamp(-127, 127)
        codes[where, :, p % page] = level.to(torch.int8)
        held.append((level * scale).view(batch * tokens, hk * dim).to(kind))
    return (q.reshape(batch * tokens, hq * dim), held[0], held[1], s["k_codes"], s["v_codes"], s["k_scales"],
            s["v_scales"])


def _cached(s, name):
    """Keys or values of every sequence in fp32, [batch, kv_heads, 1, positions, dim]."""
    table = s["table"].long()
    x = s[name + "_codes"][table].float() * s[name + "_scales"][table][..., None, None]
    return x.transpose(1, 2).reshape(s["batch"], s["kv_heads"], 1, -1, s["dim"])


def _plain_attend(s):
    batch, tokens, hq, hk, dim = (s[n] for n in ("batch", "tokens", "q_heads", "kv_heads", "dim"))
    q = s["q"]
    i = _token_positions(s)[..., None]
    p = torch.arange(s["table"].shape[1] * s["page"], device=DEV)
    seen = p <= i
    if s["window"]:
        seen &= p > i - s["window"]
    x = q.float().view(batch, tokens, hk, hq // hk, dim).permute(0, 2, 3, 1, 4)
    x = (x @ _cached(s, "k").transpose(-1, -2)) / math.sqrt(dim)   # [batch, hk, share, tokens, positions]
    x = x.masked_fill(~seen[:, None, None], -math.inf)
    x = (x - x.amax(-1, keepdim=True)).exp()
    x = x / x.sum(-1, keepdim=True)
    return (x @ _cached(s, "v")).permute(0, 3, 1, 2, 4).reshape(batch * tokens, hq * dim).to(q.dtype)


# ------------------------------------------------------------------- passes

def _own_type(kind):
    import dranzer_b200 as dz
    return {"f32": dz.TYPE_F32, "f16": dz.TYPE_F16, "bf16": dz.TYPE_BF16}[kind]


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _own_norm(s):
    import dranzer_b200 as dz
    x, rows, width = s["x_rows"], s["rows"], s["width"]
    lda = -(-width // 16) * 16
    codes = torch.empty(rows, lda, dtype=torch.int8, device=DEV)
    scales = torch.empty(rows, dtype=torch.float32, device=DEV)
    total = x.new_empty(rows, width) if s["residual"] else None
    r = s["residual_rows"] if s["residual"] else None
    dz.norm_q8(rows, width, type=_own_type(s["type"]), x=x.data_ptr(), x_stride=x.stride(0),
               residual=r.data_ptr() if s["residual"] else None, residual_stride=r.stride(0) if s["residual"] else None,
               sum_out=total.data_ptr() if s["residual"] else None, gain=s["g"].data_ptr() if s["gain"] else None,
               norm=s["norm"], eps=EPS, codes=codes.data_ptr(), codes_stride=lda, scales=scales.data_ptr(),
               stream_ptr=_stream())
    return (codes[:, :width], scales) + ((total,) if s["residual"] else ())


def _own_product(s):
    y = torch.empty(s["m"], s["n"], dtype=TYPES[s["type"]], device=DEV)
    s["w"].matmul_q8_async(s["codes"].data_ptr(), s["a_scales"].data_ptr(), y.data_ptr(), s["m"], _stream(),
                           type=_own_type(s["type"]), lda=s["codes"].stride(0),
                           bias_ptr=s["b"].data_ptr() if s["bias"] else None)
    return y


def _own_append(s):
    x = s["qkv"]
    hq, hk, dim, width = s["q_heads"], s["kv_heads"], s["dim"], x.shape[1]
    size, base = x.element_size(), x.data_ptr()
    q, k, v = (x.new_empty(x.shape[0], h * dim) for h in (hq, hk, hk))
    s["cache"].append(
        s["positions"].data_ptr(), s["tokens"], type=_own_type(s["type"]), q_heads=hq, q=base, k=base + hq * dim * size,
        v=base + (hq + hk) * dim * size, q_stride=width, k_stride=width, v_stride=width, q_out=q.data_ptr(),
        k_out=k.data_ptr(), v_out=v.data_ptr(), q_gain=s["q_gain"].data_ptr() if s["norm"] else None,
        k_gain=s["k_gain"].data_ptr() if s["norm"] else None, eps=EPS, rope_base=s["rope"], halves=s["halves"],
        stream_ptr=_stream())
    return q, k, v, s["k_codes"], s["v_codes"], s["k_scales"], s["v_scales"]


def _own_attend(s):
    q = s["q"]
    out = torch.empty_like(q)
    s["cache"].attention(s["positions"].data_ptr(), s["tokens"], type=_own_type(s["type"]), q_heads=s["q_heads"],
                         q=q.data_ptr(), out=out.data_ptr(), window=s["window"], stream_ptr=_stream())
    return out


def run(s):
    plain = {"norm": _plain_norm, "product": _plain_product, "append": _plain_append, "attend": _plain_attend}
    mine = {"norm": _own_norm, "product": _own_product, "append": _own_append, "attend": _own_attend}
    return (mine if own else plain)[s["op"]](s)


# --------------------------------------------------------------------- work

def _visible(case):
    """Over all sequences: cached tokens that a pass has to read, and (query, token) pairs that it scores."""
    rows = pairs = 0
    for first in _positions(case):
        last = first + case["tokens"] - 1
        least = lambda i: max(0, i - case["window"] + 1) if case["window"] else 0  # noqa: E731
        rows += last + 1 - least(first)
        pairs += sum(i + 1 - least(i) for i in range(first, last + 1))
    return rows, pairs


def work(case):
    size = 4 if case["type"] == "f32" else 2
    if case["op"] == "norm":
        rows, width = case["rows"], case["width"]
        wide = 3 if case["residual"] else 1
        return {"bytes": rows * width * (wide * size + 1) + rows * 4 + (width * 4 if case["gain"] else 0),
                "flops": rows * width * (4.0 + 2.0 * case["norm"])}
    if case["op"] == "product":
        m, k, n = case["m"], case["k"], case["n"]
        return {"bytes": k * n + m * k + 4 * (m + n + n * case["bias"]) + m * n * size, "flops": 2.0 * m * k * n}
    rows, dim, hq, hk = case["batch"] * case["tokens"], case["dim"], case["q_heads"], case["kv_heads"]
    if case["op"] == "append":
        return {"bytes": rows * dim * (size * (2 * hq + 4 * hk) + 2 * hk), "flops": rows * (hq + 2 * hk) * dim * 8.0}
    tokens, pairs = _visible(case)
    return {"bytes": tokens * hk * 2 * (dim + 4 / case["page"]) + 2 * rows * hq * dim * size,
            "flops": pairs * hq * dim * 4.0}


# -------------------------------------------------------------------- exact

def _nearest(v):
    """To whole numbers, halves away from zero, of fp32 values held in 64 bits."""
    return torch.sign(v) * torch.floor((v.abs() + 0.5).float().double())


def _exact_norm(s):
    h, total = s["x_rows"].double(), ()
    if s["residual"]:
        h = (h + s["residual_rows"].double()).float().to(TYPES[s["type"]])
        total = (h,)
        h = h.double()
    u = (h * s["g"].double()).float().double() if s["gain"] else h
    peak = u.abs().max(-1).values
    inverse = (127.0 / peak).float().double()                      # no peak here is near fp32's smallest numbers
    codes = _nearest((u * inverse[:, None]).float().double())
    scales = peak / 127.0
    if s["norm"]:
        scales = scales * torch.rsqrt((h * h).sum(-1) / s["width"] + EPS)
    return (codes.to(torch.int8), scales) + total


def _exact_product(s):
    a = s["codes"][:, :s["k"]].double()
    y = torch.empty(s["m"], s["n"], dtype=torch.float64, device=DEV)
    for c in range(0, s["n"], 2048):                               # sums of whole numbers below 2^53
        y[:, c:c + 2048] = a @ s["levels"][:, c:c + 2048].double()
    y *= s["a_scales"].double()[:, None]
    y *= s["w_scales"].double()[None, :]
    return y + s["b"].double() if s["bias"] else y


def _exact_append(s):
    """Page by page of each sequence, complex numbers for the rotation."""
    hq, hk, dim, n, page = (s[name] for name in ("q_heads", "kv_heads", "dim", "tokens", "page"))
    x = s["qkv"].double().view(s["batch"], n, hq + 2 * hk, dim)
    where = s["positions"].double().view(-1, 1, 1, 1) + torch.arange(n, dtype=torch.float64, device=DEV).view(1, -1, 1, 1)

    def turned(y, gain):
        if s["norm"]:
            y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / dim + EPS) * gain.double()
        if s["rope"]:
            speed = torch.exp(-torch.arange(0, dim, 2, dtype=torch.float64, device=DEV) / dim * math.log(s["rope"]))
            spin = torch.polar(torch.ones((), dtype=torch.float64, device=DEV), where * speed)
            a = y.unflatten(-1, (2, dim // 2)).transpose(-1, -2) if s["halves"] else y.unflatten(-1, (dim // 2, 2))
            z = torch.view_as_real(torch.view_as_complex(a.contiguous()) * spin)
            y = (z.transpose(-1, -2) if s["halves"] else z).flatten(-2)
        return y

    table = s["table"].tolist()
    out = []
    for name, y in (("k", turned(x[:, :, hq:hq + hk], s.get("k_gain"))), ("v", x[:, :, hq + hk:])):
        y = y.float().double().transpose(1, 2)                     # [batch, hk, tokens, dim]
        codes, scales = s[name + "_codes"].clone(), s[name + "_scales"].clone()
        kept = torch.empty_like(y)
        for b, first in enumerate(_positions(s)):
            for j in range(first // page, (first + n - 1) // page + 1):
                lo, hi = max(first, j * page), min(first + n, (j + 1) * page)
                at, fresh = table[b][j], y[b, :, lo - first:hi - first]
                new = (fresh.abs().amax((1, 2)) / 127.0).float().double()
                if lo > j * page:
                    old = scales[at].double()
                    new = torch.maximum(old, new)
                    shrink = (old / new).float().double()[:, None, None]
                    early = codes[at, :, :lo - j * page].double()
                    codes[at, :, :lo - j * page] = _nearest((early * shrink).float().double()).to(torch.int8)
                scales[at] = new.float()
                c = _nearest((fresh * (1.0 / new).float().double()[:, None, None]).float().double()).clamp(-127, 127)
                codes[at, :, lo - j * page:hi - j * page] = c.to(torch.int8)
                kept[b, :, lo - first:hi - first] = c * new[:, None, None]
        out.append((kept.transpose(1, 2).reshape(s["batch"] * n, -1), codes, scales))
    q = turned(x[:, :, :hq], s.get("q_gain")).reshape(s["batch"] * n, -1)
    return q, out[0][0], out[1][0], out[0][1], out[1][1], out[0][2], out[1][2]


def _exact_attend(s):
    """Sequence by sequence, each query over what it sees."""
    hq, hk, dim, n, page = (s[name] for name in ("q_heads", "kv_heads", "dim", "tokens", "page"))
    out = torch.empty(s["batch"], n, hq, dim, dtype=torch.float64, device=DEV)
    q = s["q"].double().view(s["batch"], n, hk, hq // hk, dim)
    for b, first in enumerate(_positions(s)):
        pages = s["table"][b, :(first + n - 1) // page + 1].long()
        k, v = (torch.einsum("phtd,ph->hptd", s[x + "_codes"][pages].double(), s[x + "_scales"][pages].double())
                .reshape(hk, -1, dim) for x in ("k", "v"))
        for t in range(n):
            hi = first + t + 1
            lo = max(0, hi - s["window"]) if s["window"] else 0
            e = torch.einsum("hgd,hpd->hgp", q[b, t], k[:, lo:hi]) * dim ** -0.5
            out[b, t] = torch.einsum("hgp,hpd->hgd", torch.softmax(e, -1), v[:, lo:hi]).reshape(hq, dim)
    return out.view(s["batch"] * n, hq * dim)


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "product": _exact_product, "append": _exact_append, "attend": _exact_attend}[
        case["op"]](s)
