"""Timed calls of the operators with which long, shared and multimodal contexts
are served: attention in a sliding window with sinks, attention of a batch whose
sequences share a prefix, and rotary positions with several axes.

`own` false: run() computes them from elementary torch operations in fp32.
`own` true: run() calls ntops_amd.torch.  exact() is the definition in 64 bits.

Definitions
  window   query row i of a sequence of n tokens is its token p = n - q_len + i.
           It sees the keys j <= p with j > p - window or j < sinks.
  prefix   the sequences of a group share the first tokens' keys and values; row
           i sees all of them, and of its own sequence's n tokens those up to
           n - q_len + i.
  A row that sees no key is 0; query head h reads head h // (heads / kv_heads).
  rotary   pair i of a head is rotated by the angle of table row positions[a],
           column i, where a is the axis of the section that i lies in.
"""

import math

import torch


own = False

DEVICE = "cuda"
_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ------------------------------------------------------------------ cases --


def listed():
    return [
        # One new token of one sequence, in a layer with a short window (latency).
        {"name": "window_token", "op": "window", "dtype": "bf16", "batch": 1, "q_heads": 32, "kv_heads": 8, "q_len": 1, "kv_len": 4096, "least": 4096, "dim": 128, "window": 1024, "sinks": 4},
        # One new token of every sequence of a decode batch, most of them past the window.
        {"name": "window_decode", "op": "window", "dtype": "bf16", "batch": 64, "q_heads": 32, "kv_heads": 8, "q_len": 1, "kv_len": 8192, "least": 2048, "dim": 128, "window": 4096, "sinks": 4},
        # Five drafted tokens of every sequence, checked at once.
        {"name": "window_draft", "op": "window", "dtype": "f16", "batch": 16, "q_heads": 64, "kv_heads": 8, "q_len": 5, "kv_len": 32768, "least": 16384, "dim": 64, "window": 2048, "sinks": 16},
        # A long prompt from its first token on.
        {"name": "window_prefill", "op": "window", "dtype": "bf16", "batch": 1, "q_heads": 32, "kv_heads": 8, "q_len": 16384, "kv_len": 16384, "least": 16384, "dim": 128, "window": 4096, "sinks": 4},
        # Prompts of a padded batch in a layer with a narrow window; no size a multiple of a tile, and short sequences leave rows empty.
        {"name": "window_narrow", "op": "window", "dtype": "f16", "batch": 7, "q_heads": 16, "kv_heads": 16, "q_len": 2001, "kv_len": 2001, "least": 900, "dim": 80, "window": 255, "sinks": 1},
        # A chunk of a prompt behind its past, in 32 bits.
        {"name": "window_f32", "op": "window", "dtype": "f32", "batch": 3, "q_heads": 12, "kv_heads": 4, "q_len": 333, "kv_len": 1501, "least": 700, "dim": 96, "window": 500, "sinks": 8},
        # A few answers to one question, their first tokens (latency).
        {"name": "prefix_token", "op": "prefix", "dtype": "bf16", "groups": 1, "batch": 4, "q_heads": 32, "kv_heads": 8, "q_len": 1, "prefix_len": 1024, "prefix_least": 1024, "kv_len": 64, "least": 16, "dim": 128},
        # A decode batch behind one long system prompt.
        {"name": "prefix_decode", "op": "prefix", "dtype": "bf16", "groups": 1, "batch": 64, "q_heads": 32, "kv_heads": 8, "q_len": 1, "prefix_len": 8192, "prefix_least": 8192, "kv_len": 1024, "least": 256, "dim": 128},
        # Eight samples of each of four prompts of different lengths; every head has its own keys.
        {"name": "prefix_samples", "op": "prefix", "dtype": "f16", "groups": 4, "batch": 32, "q_heads": 16, "kv_heads": 16, "q_len": 1, "prefix_len": 5001, "prefix_least": 1700, "kv_len": 777, "least": 3, "dim": 64},
        # Questions about one document, each prompt behind it.
        {"name": "prefix_prompts", "op": "prefix", "dtype": "bf16", "groups": 1, "batch": 16, "q_heads": 32, "kv_heads": 8, "q_len": 500, "prefix_len": 8192, "prefix_least": 8192, "kv_len": 500, "least": 200, "dim": 128},
        # The queries and keys of one new token of every sequence (latency).
        {"name": "rotary_token", "op": "rotary", "dtype": "bf16", "batch": 16, "tokens": 1, "q_heads": 32, "kv_heads": 8, "dim": 128, "sections": "16 24 24", "interleaved": False},
        # Prompts of text and images.
        {"name": "rotary_prompt", "op": "rotary", "dtype": "bf16", "batch": 4, "tokens": 4096, "q_heads": 32, "kv_heads": 8, "dim": 128, "sections": "16 24 24", "interleaved": False},
    ]


def _log(rng, lo, hi):
    """An integer of [lo, hi], uniform over its logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _ragged(rng, n, step):
    """n itself or n moved off a multiple of `step`."""
    return max(1, n + (rng.randrange(-step, step) if rng.random() < 0.5 else 0))


def _fits(case):
    """True for a case that costs no more than the largest listed ones."""
    w = work(case)
    if case["op"] == "rotary":
        return w["bytes"] <= 350_000_000
    # (products in 32 bits are a sixteenth as fast; the plain form of a window computes the scores of all keys)
    scores = case["batch"] * case["q_heads"] * case["q_len"] * (case["kv_len"] + case.get("prefix_len", 0))
    return w["bytes"] <= 980_000_000 and w["flops"] <= 1e12 / (16 if case["dtype"] == "f32" else 1) and scores <= 32 * 16384 * 16384


def draw(rng):
    op = rng.choice(["window", "window", "window", "prefix", "prefix", "rotary"])
    group, kv_heads = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 2, 4, 8, 16])
    dim = rng.choice([64, 80, 96, 128, 128])
    case = {"op": op, "dtype": rng.choice(["bf16", "bf16", "f16", "f16", "f32"]), "q_heads": group * kv_heads, "kv_heads": kv_heads, "dim": dim, "batch": _log(rng, 1, 64)}
    if op == "rotary":
        axes = rng.choice([1, 2, 3, 3])
        if rng.random() < 0.3:  # the axes in turn, pair by pair
            sections = [1] * (dim // 2)
        else:
            cuts = sorted(rng.randrange(dim // 2 + 1) for _ in range(axes - 1))
            sections = [b - a for a, b in zip([0] + cuts, cuts + [dim // 2])]
        tokens = 1 if rng.random() < 0.3 else _ragged(rng, _log(rng, 2, 8192), 16)
        case.update(tokens=tokens, axes=axes, sections=" ".join(map(str, sections)), interleaved=rng.random() < 0.4)
    else:
        kv = _ragged(rng, _log(rng, 16, 32768 if op == "window" else 4096), 16)
        q = 1 if rng.random() < 0.4 else min(kv, _log(rng, 2, 8) if rng.random() < 0.3 else _ragged(rng, _log(rng, 9, 4096), 8))
        least = kv if rng.random() < 0.3 else max(1, rng.choice([kv // 2, kv // 8, q // 2]))
        case.update(q_len=q, kv_len=kv, least=least)
        if op == "window":
            case.update(window=_ragged(rng, _log(rng, 16, 8192), 16), sinks=rng.choice([0, 1, 4, 16, 100]))
        else:
            prefix = _ragged(rng, _log(rng, 16, 32768), 16)
            case.update(groups=rng.choice([1, 1, 1, 2, 4]), prefix_len=prefix, prefix_least=rng.choice([prefix, max(1, prefix // 3)]))
            case["batch"] = case["groups"] * max(2, case["batch"] // case["groups"])
    while not _fits(case):  # fewer sequences, then shorter ones
        groups = case.get("groups", 1)
        if case["batch"] > groups:
            case["batch"] = groups * (case["batch"] // groups * 3 // 4)
        elif groups > 1:
            case["groups"] = case["batch"] = 1
        else:
            for name in ("tokens", "q_len"):
                if name in case:
                    case[name] = case[name] * 3 // 4
    return case


def _evenly(least, longest, count):
    """Lengths from the least to the longest; one alone has the longest."""
    return [longest] if count == 1 else [least + (longest - least) * i // (count - 1) for i in range(count)]


def _sections(case):
    return [int(n) for n in case["sections"].split()]


# ---------------------------------------------------------------- prepare --


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.empty(shape, device=DEVICE).normal_(generator=g)

    def activations(*shape):  # a few channels much larger than the others
        return (normal(*shape) * torch.exp(0.5 * normal(shape[-1]))).to(dtype)

    def lengths(least, longest, count):
        order = torch.randperm(count, generator=g, device=DEVICE)
        return torch.tensor(_evenly(least, longest, count), dtype=torch.int32, device=DEVICE)[order]

    st = dict(case)
    b, d = case["batch"], case["dim"]
    if case["op"] == "rotary":
        tokens, limit = case["tokens"], 32768
        st["q"], st["k"] = activations(b, tokens, case["q_heads"], d), activations(b, tokens, case["kv_heads"], d)
        rates = 1e6 ** (-torch.arange(d // 2, dtype=torch.float64, device=DEVICE) / (d // 2))
        angles = torch.arange(limit, dtype=torch.float64, device=DEVICE)[:, None] * rates
        st["sin"], st["cos"] = angles.sin().float(), angles.cos().float()
        # text, an image of rows of 32 patches, and text behind the image's larger side
        at = torch.arange(tokens, device=DEVICE)
        first = torch.randint(0, limit - tokens, (b, 1), generator=g, device=DEVICE)
        lo, hi = tokens // 4, tokens - tokens // 4
        row, col = (at - lo) // 32, (at - lo) % 32
        behind = lo + max(32, (hi - lo) // 32) + at - hi
        inside = (at >= lo) & (at < hi)
        axes = [torch.where(inside, lo + x, torch.where(at < lo, at, behind)) for x in (0 * at, row, col)]
        st["positions"] = (torch.stack(axes)[: case.get("axes", 3), None] + first).clamp(max=limit - 1)
        st["sizes"] = _sections(case)
        return st
    hkv, c = case["kv_heads"], case["kv_len"]
    st["query"] = activations(b, case["q_heads"], case["q_len"], d)
    st["key"], st["value"] = activations(b, hkv, c, d), activations(b, hkv, c, d)
    st["lengths"] = lengths(case["least"], c, b)
    if case["op"] == "prefix":
        n = case["groups"]
        st["prefix_key"], st["prefix_value"] = (activations(n, hkv, case["prefix_len"], d) for _ in range(2))
        st["prefix_lengths"] = lengths(case["prefix_least"], case["prefix_len"], n)
    st["scale"] = 1 / math.sqrt(d)
    return st


# -------------------------------------------------------------------- run --


def run(st):
    if own:
        return _run_own(st)
    return {"window": _window_plain, "prefix": _prefix_plain, "rotary": _rotary_plain}[st["op"]](st)


def _run_own(st):
    import ntops_amd.torch as nt

    if st["op"] == "window":
        return nt.sliding_window_attention(
            st["query"], st["key"], st["value"], st["window"], st["sinks"], lengths=st["lengths"], scale=st["scale"])
    if st["op"] == "prefix":
        return nt.shared_prefix_attention(
            st["query"], st["prefix_key"], st["prefix_value"], st["key"], st["value"],
            prefix_lengths=st["prefix_lengths"], lengths=st["lengths"], scale=st["scale"])
    return nt.multi_axis_rotary_position_embedding_qk(
        st["q"], st["k"], st["sin"], st["cos"], st["positions"], st["sizes"], interleaved=st["interleaved"])


def _softmax_plain(s, seen):
    """exp(s - max) of the scores that are seen, in place, and its sums."""
    s = s.masked_fill_(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = s.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    return p, p.sum(-1, keepdim=True)


def _window_plain(st):
    q, n = st["query"], st["lengths"].long()[:, None, None, None]
    (b, hq, sq, d), (hkv, c) = q.shape, st["key"].shape[1:3]
    k, v = st["key"].float(), st["value"].float()
    at = torch.arange(c, device=q.device)
    rows = max(1, (1 << 31) // (b * hq * c))
    out = []
    for i in range(0, sq, rows):  # as many query rows as 8 GiB of scores hold
        part = q[:, :, i : i + rows].float()
        m = part.shape[2]
        s = torch.matmul(part.reshape(b, hkv, -1, d), k.transpose(-1, -2).contiguous()).view(b, hq, m, c) * st["scale"]
        p = n - sq + i + torch.arange(m, device=q.device)[:, None]
        e, total = _softmax_plain(s, (at <= p) & ((at > p - st["window"]) | (at < st["sinks"])))
        o = torch.matmul(e.view(b, hkv, -1, c), v).view(b, hq, m, d)
        out.append(torch.where(total > 0, o / total, 0.0).to(q.dtype))
    return torch.cat(out, 2)


def _prefix_plain(st):
    q = st["query"]
    (b, hq, sq, d), (hkv, c) = q.shape, st["key"].shape[1:3]
    groups, _, prefix, _ = st["prefix_key"].shape
    per, heads = b // groups, hq // hkv
    pk, pv, k, v = (st[name].float() for name in ("prefix_key", "prefix_value", "key", "value"))
    n, pn = st["lengths"].long()[:, None, None, None], st["prefix_lengths"].long().repeat_interleave(per)[:, None, None, None]
    at, pat = torch.arange(c, device=q.device), torch.arange(prefix, device=q.device)
    rows = max(1, (1 << 31) // (b * hq * (c + prefix)))
    out = []
    for i in range(0, sq, rows):
        part = q[:, :, i : i + rows].float()
        m = part.shape[2]
        # the rows of a group's sequences together over their prefix
        together = part.reshape(groups, per, hkv, heads * m, d).transpose(1, 2).reshape(groups, hkv, -1, d)
        s = torch.matmul(together, pk.transpose(-1, -2).contiguous())
        s = s.view(groups, hkv, per, heads * m, prefix).transpose(1, 2).reshape(b, hq, m, prefix)
        t = torch.matmul(part.reshape(b, hkv, -1, d), k.transpose(-1, -2).contiguous()).view(b, hq, m, c)
        p = n - sq + i + torch.arange(m, device=q.device)[:, None]
        seen = torch.cat(((pat < pn).expand(b, 1, m, prefix), (at <= p).expand(b, 1, m, c)), -1)
        e, total = _softmax_plain(torch.cat((s, t), -1) * st["scale"], seen)
        ep = e[..., :prefix].reshape(groups, per, hkv, heads * m, prefix).transpose(1, 2).reshape(groups, hkv, -1, prefix)
        o = torch.matmul(ep, pv).view(groups, hkv, per, heads * m, d).transpose(1, 2).reshape(b, hq, m, d)
        o = o + torch.matmul(e[..., prefix:].reshape(b, hkv, -1, c), v).view(b, hq, m, d)
        out.append(torch.where(total > 0, o / total, 0.0).to(q.dtype))
    return torch.cat(out, 2)


def _rotary_plain(st):
    half = st["dim"] // 2
    axis = torch.arange(len(st["sizes"])).repeat_interleave(torch.tensor(st["sizes"])) % st["positions"].shape[0]
    at = st["positions"][axis.tolist()].movedim(0, -1)  # (batch, tokens, half)
    col = torch.arange(half, device=at.device)
    sin, cos = st["sin"][at, col][:, :, None], st["cos"][at, col][:, :, None]

    def rotated(x):
        y = x.float()
        a, b = (y[..., ::2], y[..., 1::2]) if st["interleaved"] else (y[..., :half], y[..., half:])
        pair = (a * cos - b * sin, b * cos + a * sin)
        return (torch.stack(pair, -1).flatten(-2) if st["interleaved"] else torch.cat(pair, -1)).to(x.dtype)

    return rotated(st["q"]), rotated(st["k"])


# ------------------------------------------------------------------- work --


def _seen(n, q, window, sinks):
    """Pairs of a query row and a key that it sees, and the keys that some row sees."""
    pairs = sum(min(p + 1, window + min(sinks, max(0, p + 1 - window))) for p in range(max(0, n - q), n))
    first = max(0, n - q - window + 1)
    return pairs, n - first + min(sinks, first)


def work(case):
    es = 4 if case["dtype"] == "f32" else 2
    b, d = case["batch"], case["dim"]
    if case["op"] == "rotary":
        tokens, heads = b * case["tokens"], case["q_heads"] + case["kv_heads"]
        return {"bytes": tokens * (2 * heads * d * es + 8 * case.get("axes", 3)) + min(tokens, 32768) * d * 4, "flops": 3 * tokens * heads * d}
    q = case["q_len"]
    pairs = keys = 0
    for n in _evenly(case["least"], case["kv_len"], b):
        p, k = _seen(n, q, case.get("window", n), case.get("sinks", 0))
        pairs, keys = pairs + p, keys + k
    if case["op"] == "prefix":
        prefixes = _evenly(case["prefix_least"], case["prefix_len"], case["groups"])
        keys += sum(prefixes)
        pairs += q * sum(prefixes) * (b // case["groups"])
    return {"bytes": 2 * es * (keys * case["kv_heads"] + b * case["q_heads"] * q) * d, "flops": 4 * d * case["q_heads"] * pairs}


# ------------------------------------------------------------------ exact --


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "rotary":
        return _exact_rotary(st)
    q = st["query"]
    out = torch.zeros(q.shape, dtype=torch.float64, device=DEVICE)
    heads, sq = case["q_heads"] // case["kv_heads"], case["q_len"]
    own_lengths = st["lengths"].tolist()
    prefix_lengths = st["prefix_lengths"].tolist() if case["op"] == "prefix" else None
    for i, n in enumerate(own_lengths):
        for h in range(case["kv_heads"]):
            if case["op"] == "prefix":
                of = i * case["groups"] // case["batch"]
                front_k, front_v = (st[x][of, h, : prefix_lengths[of]].double() for x in ("prefix_key", "prefix_value"))
            for lo in range(0, sq, 1024):
                hi = min(lo + 1024, sq)
                place = torch.arange(n - sq + lo, n - sq + hi, device=DEVICE)[:, None]
                # keys that some row of the block can see
                last = max(0, n - sq + hi)
                if case["op"] == "window":
                    first = max(0, n - sq + lo - case["window"] + 1)
                    sinks = min(case["sinks"], first)
                    where = torch.cat((torch.arange(sinks, device=DEVICE), torch.arange(first, max(first, last), device=DEVICE)))
                    open_ = (where <= place) & ((place - where < case["window"]) | (where < case["sinks"]))
                    k, v = st["key"][i, h].double()[where], st["value"][i, h].double()[where]
                else:
                    where = torch.arange(last, device=DEVICE)
                    open_ = torch.cat((torch.ones(hi - lo, len(front_k), dtype=torch.bool, device=DEVICE), where <= place), 1)
                    k, v = (torch.cat((f, st[x][i, h, :last].double())) for f, x in ((front_k, "key"), (front_v, "value")))
                s = q[i, h * heads : (h + 1) * heads, lo:hi].double() @ k.t() * st["scale"]
                p = torch.nan_to_num(torch.softmax(s.masked_fill(~open_, -math.inf), -1))
                out[i, h * heads : (h + 1) * heads, lo:hi] = p @ v
    return out


def _exact_rotary(st):
    axes, half = st["positions"].shape[0], st["dim"] // 2
    turn = torch.zeros(*st["positions"].shape[1:], half, dtype=torch.complex128, device=DEVICE)
    start = 0
    for j, size in enumerate(st["sizes"]):
        rows = st["positions"][j % axes]
        for c in range(start, start + size):
            turn[:, :, c] = torch.complex(st["cos"][:, c].double()[rows], st["sin"][:, c].double()[rows])
        start += size

    def rotated(x):
        shape = (*x.shape[:-1], half, 2) if st["interleaved"] else (*x.shape[:-1], 2, half)
        dim = -1 if st["interleaved"] else -2
        a, b = x.double().view(shape).unbind(dim)
        z = torch.complex(a, b) * turn[:, :, None]
        return torch.stack((z.real, z.imag), dim).reshape(x.shape)

    return rotated(st["q"]), rotated(st["k"])
