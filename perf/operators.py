"""Timed calls of the narrow-format operators of a decoder layer: products of
microscaled 4-bit tensors, and attention over a key / value cache held in 8
bits.

`own` false: run() computes them from elementary torch operations in fp32.
`own` true: run() calls ntops_amd.torch.  exact() is the definition in 64 bits.

Formats
  MXFP4   blocks of 32 values along a row share the scale 2^e, e = max(-127,
          floor(log2(max |x|)) - 2), stored as the byte e + 127; each value is
          x / 2^e rounded to the nearest of 0, .5, 1, 1.5, 2, 3, 4, 6 (ties to
          the even code), cut at 6; two codes a byte, the first in the low half.
  cache   a block of tokens of one head shares the scale 2^e, e the least
          integer >= -126 with max |x| <= 448 2^e; values are x / 2^e rounded
          to e4m3.  A block that grows keeps the larger of its scales, and its
          earlier values are rounded again to the new one.
"""

import math

import torch


own = False

DEVICE = "cuda"
_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# ------------------------------------------------------------------ cases --


def listed():
    return [
        # The activations of one token, rounded to MXFP4 and back (latency).
        {"name": "quantize_token", "op": "quantize", "dtype": "bf16", "rows": 1, "cols": 4096},
        # A projection's weight, rounded once when a model is loaded.
        {"name": "quantize_weight", "op": "quantize", "dtype": "bf16", "rows": 14336, "cols": 4096},
        # Single-token decode: a projection of one row; its activations are rounded in the pass.
        {"name": "product_token", "op": "product", "dtype": "bf16", "m": 1, "k": 4096, "n": 14336, "activations": True, "bias": False},
        # A decode batch through the down projection, operands already in MXFP4.
        {"name": "product_decode", "op": "product", "dtype": "f16", "m": 16, "k": 14336, "n": 4096, "activations": False, "bias": True},
        # A short prompt; no size a multiple of a tile, fp32 out.
        {"name": "product_odd", "op": "product", "dtype": "f32", "m": 500, "k": 2080, "n": 1001, "activations": False, "bias": True},
        # A prefill's up projection, activations rounded in the pass.
        {"name": "product_prefill", "op": "product", "dtype": "bf16", "m": 8192, "k": 4096, "n": 14336, "activations": True, "bias": False},
        # One new token of every sequence of a decode batch.
        {"name": "store_token", "op": "store", "dtype": "bf16", "batch": 32, "kv_heads": 8, "tokens": 1, "dim": 128, "capacity": 4096, "block": 64},
        # Prompts of different lengths behind what the cache holds already.
        {"name": "store_prompt", "op": "store", "dtype": "bf16", "batch": 4, "kv_heads": 8, "tokens": 2048, "dim": 128, "capacity": 4096, "block": 64},
        # Decode batch over sequences of half to full length.
        {"name": "attention_decode", "op": "attention", "dtype": "bf16", "batch": 16, "q_heads": 32, "kv_heads": 8, "q_len": 1, "kv_len": 4096, "dim": 128, "block": 64, "causal": False},
        # One sequence with a long context.
        {"name": "attention_long", "op": "attention", "dtype": "f16", "batch": 1, "q_heads": 32, "kv_heads": 8, "q_len": 1, "kv_len": 131072, "dim": 128, "block": 128, "causal": False},
        # Prompts read back from the cache they were stored in.
        {"name": "attention_prefill", "op": "attention", "dtype": "bf16", "batch": 4, "q_heads": 32, "kv_heads": 8, "q_len": 2048, "kv_len": 2048, "dim": 128, "block": 64, "causal": True},
        # A chunk of a prompt behind a longer past; odd sizes.
        {"name": "attention_chunk", "op": "attention", "dtype": "f16", "batch": 3, "q_heads": 24, "kv_heads": 8, "q_len": 101, "kv_len": 5001, "dim": 64, "block": 32, "causal": True},
    ]


def _log(rng, lo, hi):
    """An integer of [lo, hi], uniform over its logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _ragged(rng, n, step):
    """n itself or n moved off a multiple of `step`."""
    return max(1, n + (rng.randrange(-step, step) if rng.random() < 0.5 else 0))


def draw(rng):
    op = rng.choice(["quantize", "product", "product", "store", "attention", "attention"])
    half = rng.choice(["bf16", "f16"])
    if op == "quantize":
        cols = _ragged(rng, _log(rng, 64, 14336), 32)
        dtype = rng.choice(["bf16", "f16", "f32"])
        return {"op": op, "dtype": dtype, "rows": _log(rng, 1, 14336 * 4096 // cols // (2 if dtype == "f32" else 1)), "cols": cols}
    if op == "product":
        k, n = _ragged(rng, _log(rng, 64, 14336), 32), _ragged(rng, _log(rng, 64, 14336), 32)
        m = min(_log(rng, 1, 8192), 8192 * 4096 * 14336 // (k * n))
        return {"op": op, "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]), "m": m, "k": k, "n": n, "activations": rng.random() < 0.5, "bias": rng.random() < 0.5}
    dim = rng.choice([64, 80, 96, 128, 128])
    block = rng.choice([16, 32, 64, 128])
    if op == "store":
        heads = rng.choice([1, 2, 4, 8, 16])
        tokens = 1 if rng.random() < 0.4 else _ragged(rng, _log(rng, 2, 4096), 16)
        batch = max(1, min(_log(rng, 1, 64), 4 * 8 * 2048 * 128 // (heads * tokens * dim)))
        past = _log(rng, 1, max(1, min(4096, 32 * 8 * 4096 * 128 // (batch * heads * dim) - tokens)))
        return {"op": op, "dtype": rng.choice(["bf16", "f16", "f32"]), "batch": batch, "kv_heads": heads, "tokens": tokens, "dim": dim, "capacity": tokens + past, "block": block}
    group = rng.choice([1, 2, 4, 8])
    kv_heads = rng.choice([1, 2, 4, 8])
    kv = _ragged(rng, _log(rng, 16, 131072), 16)
    q = 1 if rng.random() < 0.5 else min(kv, _ragged(rng, _log(rng, 2, 2048), 8))
    batch = max(1, min(_log(rng, 1, 64), 16 * 8 * 4096 * 128 // (kv_heads * kv * dim), 4 * 32 * 2048 * 2048 // (group * kv_heads * q * kv)))
    q = max(1, min(q, 4 * 32 * 2048 * 2048 // (group * kv_heads * batch * kv)))
    return {"op": op, "dtype": half, "batch": batch, "q_heads": group * kv_heads, "kv_heads": kv_heads, "q_len": q, "kv_len": kv, "dim": dim, "block": block, "causal": q > 1 and rng.random() < 0.75}


def _lengths(case):
    """Lengths of a batch's sequences: from half the longest to the longest, evenly."""
    longest, b = case["kv_len"] if case["op"] == "attention" else case["tokens"], case["batch"]
    least = max(1, longest // 2)
    return [longest] if b == 1 else [least + (longest - least) * i // (b - 1) for i in range(b)]


# ---------------------------------------------------------------- formats --


def _quantize(x):
    """MXFP4 of the rows of x: codes (.., 16 a block) and scale bytes (.., 1 a block)."""
    cols = x.shape[-1]
    x = torch.nn.functional.pad(x.float(), (0, -cols % 32)).unflatten(-1, (-1, 32))
    amax = x.abs().amax(-1, keepdim=True)
    e = torch.where(amax > 0, torch.frexp(amax).exponent - 3, -127).clamp(min=-127)
    y = x * torch.exp2(-e.float())
    a = y.abs()
    code = (a > 0.25).to(torch.uint8)
    for over in (a >= 0.75, a > 1.25, a >= 1.75, a > 2.5, a >= 3.5, a > 5):
        code += over
    code |= torch.signbit(y).to(torch.uint8) << 3
    pairs = code.unflatten(-1, (16, 2))
    return (pairs[..., 0] | pairs[..., 1] << 4).flatten(-2), (e + 127).to(torch.uint8).squeeze(-1)


def _values(codes, scales):
    """The fp32 values that MXFP4 codes and scale bytes stand for."""
    table = torch.tensor(_E2M1 + tuple(-v for v in _E2M1), device=codes.device)
    v = table[torch.stack((codes & 15, codes >> 4), -1).flatten(-2).long()]
    return v * torch.exp2(scales.float() - 127).repeat_interleave(32, -1)


def _least_scale(amax):
    """2^e with the least e >= -126 for which amax <= 448 * 2^e."""
    f = torch.frexp(amax)
    e = torch.where(f.mantissa <= 0.875, f.exponent - 9, f.exponent - 8)
    return torch.exp2(torch.where(amax > 0, e, -126).clamp(min=-126).float())


def _cache_of(x, block):
    """A whole cache (batch, heads, capacity, dim) in e4m3 with its scales."""
    c = x.shape[2]
    scale = _least_scale(torch.nn.functional.pad(x.abs().amax(-1), (0, -c % block)).unflatten(-1, (-1, block)).amax(-1))
    return (x / scale.repeat_interleave(block, -1)[..., :c, None]).to(torch.float8_e4m3fn), scale


# ---------------------------------------------------------------- prepare --


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]

    def normal(*shape, std=1.0):
        return torch.empty(shape, device=DEVICE).normal_(0, std, generator=g)

    def activations(*shape):  # a few channels much larger than the others
        return normal(*shape) * torch.exp(normal(shape[-1]))

    st = dict(case)
    if case["op"] == "quantize":
        st["x"] = activations(case["rows"], case["cols"]).to(dtype)
    elif case["op"] == "product":
        m, k, n = case["m"], case["k"], case["n"]
        x = activations(m, k).to(torch.bfloat16 if dtype == torch.float32 else dtype)
        if case["activations"]:
            st["x"] = x
        else:
            st["a"], st["a_scale"] = _quantize(x)
        st["b"], st["b_scale"] = _quantize(normal(n, k, std=1 / math.sqrt(k)))
        st["bias"] = normal(n).to(dtype) if case["bias"] else None
    else:
        b, h, d, block = case["batch"], case["kv_heads"], case["dim"], case["block"]
        capacity = case["capacity"] if case["op"] == "store" else case["kv_len"]
        for name in ("key", "value"):
            held = activations(b, h, capacity, d) * torch.exp(0.5 * normal(b, h, capacity, 1))
            st[name + "_cache"], st[name + "_scale"] = _cache_of(held, block)
        order = torch.randperm(b, generator=g, device=DEVICE)
        st["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device=DEVICE)[order]
        if case["op"] == "store":
            for name in ("key", "value"):
                st[name] = (activations(b, h, case["tokens"], d) * torch.exp(0.5 * normal(b, h, case["tokens"], 1))).to(dtype)
            room = capacity - case["tokens"]
            st["positions"] = torch.randint(0, room + 1, (b,), generator=g, device=DEVICE, dtype=torch.int32)
        else:
            st["query"] = normal(b, case["q_heads"], case["q_len"], d).to(dtype)
            st["scale"] = 1 / math.sqrt(d)
    return st


# -------------------------------------------------------------------- run --


def run(st):
    if own:
        return _run_own(st)
    return {"quantize": _quantize_plain, "product": _product_plain, "store": _store_plain, "attention": _attention_plain}[st["op"]](st)


def _run_own(st):
    import ntops_amd.torch as nt

    if st["op"] == "quantize":
        x = st["x"]
        codes, scales = nt.quantize_mxfp4(x)
        return nt.dequantize_mxfp4(codes, scales, x.shape[-1], dtype=x.dtype)
    if st["op"] == "product":
        dtype = _DTYPES[st["dtype"]]
        if st["activations"]:
            return nt.mxfp4_mm(st["x"], None, st["b"], st["b_scale"], st["bias"], dtype=dtype)
        return nt.mxfp4_mm(st["a"], st["a_scale"], st["b"], st["b_scale"], st["bias"], dtype=dtype)
    cache = (st["key_cache"], st["value_cache"], st["key_scale"], st["value_scale"])
    if st["op"] == "store":
        nt.store_kv_cache(st["key"], st["value"], *cache, st["positions"], st["lengths"], block_size=st["block"])
        return cache
    return nt.kv_cache_attention(st["query"], *cache, st["lengths"], is_causal=st["causal"], scale=st["scale"], block_size=st["block"])


def _quantize_plain(st):
    x = st["x"]
    return _values(*_quantize(x))[..., : x.shape[-1]].to(x.dtype)


def _product_plain(st):
    a = _quantize(st["x"]) if st["activations"] else (st["a"], st["a_scale"])
    y = torch.matmul(_values(*a), _values(st["b"], st["b_scale"]).t())
    if st["bias"] is not None:
        y = y + st["bias"].float()
    return y.to(_DTYPES[st["dtype"]])


def _store_plain(st):
    block = st["block"]
    start, count = st["positions"].long(), st["lengths"].long()
    for new, cache, scale in ((st["key"], st["key_cache"], st["key_scale"]), (st["value"], st["value_cache"], st["value_scale"])):
        (b, h, tokens, d), capacity, blocks = new.shape, cache.shape[2], scale.shape[2]
        # the blocks that the tokens of a sequence can lie in (past the last: the last again, with the same result)
        j = (start[:, None] // block + torch.arange((tokens - 1) // block + 2, device=new.device)).clamp(max=blocks - 1)
        p = (j[..., None] * block + torch.arange(block, device=new.device)).clamp(max=capacity - 1)  # (b, n, block)
        s = p - start[:, None, None]
        is_new = ((s >= 0) & (s < count[:, None, None]))[:, None, :, :, None]
        seq, head = torch.arange(b, device=new.device)[:, None, None, None], torch.arange(h, device=new.device)[None, :, None, None]
        x = new[seq, head, s.clamp(0, tokens - 1)[:, None]].float()  # (b, h, n, block, d)
        old_scale = scale[seq[..., 0], head[..., 0], j[:, None]]
        fits = _least_scale(torch.where(is_new, x.abs(), 0.0).amax((-2, -1)))
        first = is_new[..., 0, 0]  # the block's first token is new: what it held is over
        new_scale = torch.where(is_new.any(-2)[..., 0], torch.where(first, fits, torch.maximum(fits, old_scale)), old_scale)
        held = cache[seq, head, p[:, None]]
        before = (s < 0)[:, None, :, :, None] & is_new.any(-2, keepdim=True) & ~first[..., None, None]
        again = (held.float() * (old_scale / new_scale)[..., None, None]).to(cache.dtype).float()
        codes = torch.where(is_new, x / new_scale[..., None, None], torch.where(before, again, held.float()))
        cache[seq, head, p[:, None]] = codes.to(cache.dtype)
        scale[seq[..., 0], head[..., 0], j[:, None]] = new_scale
    return st["key_cache"], st["value_cache"], st["key_scale"], st["value_scale"]


def _attention_plain(st):
    q, n = st["query"], st["lengths"].long()[:, None, None]
    (b, hq, sq, d), (hkv, c) = q.shape, st["key_cache"].shape[1:3]
    k, v = (st[x + "_cache"].float() * st[x + "_scale"].repeat_interleave(st["block"], -1)[..., :c, None] for x in ("key", "value"))
    s = torch.matmul(q.float().view(b, hkv, -1, d), k.transpose(-1, -2).contiguous()).view(b, hq, sq, c) * st["scale"]
    at = torch.arange(c, device=q.device)
    seen = (at < n).expand(b, sq, c)
    if st["causal"]:
        seen = seen & (at <= n - sq + torch.arange(sq, device=q.device)[:, None])
    s = s.masked_fill_(~seen[:, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s.sub_(torch.where(top == -math.inf, 0.0, top)))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(b, hkv, -1, c), v).view(b, hq, sq, d)
    return torch.where(total > 0, o / total, 0.0).to(q.dtype)


# ------------------------------------------------------------------- work --


def work(case):
    es = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "quantize":
        # read and written in the tensor's type; the codes and scales written, and read back
        n, held = case["rows"] * case["cols"], case["rows"] * -(-case["cols"] // 32) * 17
        return {"bytes": 2 * n * es + 2 * held, "flops": 4 * n}
    if case["op"] == "product":
        m, k, n = case["m"], case["k"], case["n"]
        held = -(-k // 32) * 17
        a = m * k * 2 if case["activations"] else m * held
        return {"bytes": a + n * held + m * n * es + (n * es if case["bias"] else 0), "flops": 2 * m * n * k}
    rows = sum(_lengths(case)) * case["kv_heads"]
    scales = 4 * rows / case["block"]
    if case["op"] == "store":
        return {"bytes": 2 * (rows * case["dim"] * (es + 1) + scales), "flops": 4 * rows * case["dim"]}
    q = case["q_len"]
    pairs = case["q_heads"] * sum(q * n - (min(q, n) * (min(q, n) - 1) // 2 + max(0, q - n) * n if case["causal"] else 0) for n in _lengths(case))
    return {"bytes": 2 * (rows * case["dim"] + scales) + 2 * es * case["batch"] * case["q_heads"] * q * case["dim"], "flops": 4 * case["dim"] * pairs}


# ------------------------------------------------------------------ exact --


def _powers():
    """2^-200 .. 2^200, for exponents found and powers taken without rounding."""
    return torch.tensor([2.0**i for i in range(-200, 201)], dtype=torch.float64, device=DEVICE)


def _floor_log2(x):
    return torch.searchsorted(_powers(), x.contiguous(), right=True) - 201


def _exp2(e):
    return _powers()[e.long() + 200]


def _exact_mxfp4(x):
    """The values that x has in MXFP4, in 64 bits."""
    cols = x.shape[-1]
    x = torch.nn.functional.pad(x.double(), (0, -cols % 32))
    w = x.reshape(*x.shape[:-1], -1, 32)
    top = w.abs().max(-1, keepdim=True).values
    step = _exp2(_floor_log2(top.clamp(min=2.0**-125)) - 2)
    a = (w / step).abs()
    unit = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).double()
    return (torch.sign(w) * torch.clamp(torch.round(a / unit) * unit, max=6) * step).reshape(x.shape)[..., :cols]


def _exact_codes(codes, scales):
    table = torch.tensor(_E2M1, dtype=torch.float64, device=codes.device)
    nibbles = torch.stack((codes % 16, codes // 16), -1).reshape(*codes.shape[:-1], -1).long()
    v = torch.where(nibbles < 8, table[nibbles % 8], -table[nibbles % 8])
    return v * torch.repeat_interleave(_exp2(scales.long() - 127), 32, -1)


def _exact_e4m3(x):
    """x (|x| <= 448) rounded to e4m3."""
    unit = _exp2(_floor_log2(x.abs().clamp(min=2.0**-6)) - 3)
    return torch.round(x / unit) * unit


def _exact_store(st, name):
    new, cache, scale, block = st[name].double(), st[name + "_cache"].double(), st[name + "_scale"].double(), st["block"]
    for i, (start, count) in enumerate(zip(st["positions"].tolist(), st["lengths"].tolist())):
        for j in range(start // block, (start + count - 1) // block + 1):
            lo, hi = max(start, j * block), min(start + count, (j + 1) * block)
            x = new[i, :, lo - start : hi - start]
            top = x.abs().amax((1, 2)).clamp(min=448 * 2.0**-126)
            fits = _exp2(_floor_log2(top / 448))
            fits = torch.where(448 * fits < top, 2 * fits, fits)
            if lo > j * block:
                held = scale[i, :, j].clone()
                fits = torch.maximum(fits, held)
                cache[i, :, j * block : lo] = _exact_e4m3(cache[i, :, j * block : lo] * (held / fits)[:, None, None])
            scale[i, :, j] = fits
            cache[i, :, lo:hi] = _exact_e4m3(x / fits[:, None, None])
    return cache, scale


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "quantize":
        return _exact_mxfp4(st["x"])
    if case["op"] == "product":
        a = _exact_mxfp4(st["x"]) if case["activations"] else _exact_codes(st["a"], st["a_scale"])[:, : case["k"]]
        y = torch.matmul(a, _exact_codes(st["b"], st["b_scale"])[:, : case["k"]].t())
        return y if st["bias"] is None else y + st["bias"].double()
    if case["op"] == "store":
        (kc, ks), (vc, vs) = _exact_store(st, "key"), _exact_store(st, "value")
        return kc, vc, ks, vs
    out = torch.zeros(st["query"].shape, dtype=torch.float64, device=DEVICE)
    group, sq = case["q_heads"] // case["kv_heads"], case["q_len"]
    for i, n in enumerate(st["lengths"].tolist()):
        back = torch.arange(sq, device=DEVICE)[:, None] + (n - sq)  # a row's own place
        open_ = torch.arange(n, device=DEVICE)[None] <= (back if case["causal"] else n)
        for h in range(case["q_heads"]):
            at = torch.arange(n, device=DEVICE) // case["block"]
            k, v = (st[x + "_cache"][i, h // group, :n].double() * st[x + "_scale"][i, h // group].double()[at][:, None] for x in ("key", "value"))
            s = (st["query"][i, h].double() @ k.t() * st["scale"]).masked_fill(~open_, -math.inf)
            p = torch.nan_to_num(torch.softmax(s, -1))
            out[i, h] = p @ v
    return out
