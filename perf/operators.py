"""The operators of the 8-bit key/value cache, as cases that can be timed and checked: keys and values
quantised as they are written into their pages, rows read back from the pages, and the attention of
single tokens and of chunks of new tokens over such pages.

A cached row (a token's key or value of one kv head) is held as e4m3 codes and one byte s that stands
for the power of two 2^(s - 127).  Sizes are those of the decoders that this repository serves (24 or
32 query heads of 128 over 8 kv heads, 32 of 64) and of their neighbours; pages hold 16 to 64 tokens.
"""
import math

import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}
LEAST, MOST = -100, 119          # exponents that a row's scale may have
HEADS = ((24, 8, 128), (32, 8, 128), (32, 8, 64), (16, 4, 128), (16, 16, 64), (40, 8, 128), (28, 4, 128),
         (12, 4, 256), (8, 1, 64))


def listed():
    return [
        # one decode step of a small batch: eight tokens, each at its own place; launches count
        dict(name="write_decode", kind="write", heads=32, kv_heads=8, dim=128, rot=128, requests=8, new=1,
             cached=2047, page=16, dtype="bfloat16"),
        # a whole prompt portion of a long document, far from the first position
        dict(name="write_prompt", kind="write", heads=24, kv_heads=8, dim=128, rot=128, requests=1, new=2048,
             cached=100000, page=64, dtype="bfloat16"),
        # the 32-bit mode, three odd portions, half of a head's features rotated
        dict(name="write_float32", kind="write", heads=32, kv_heads=8, dim=64, rot=32, requests=3, new=333,
             cached=77, page=16, dtype="float32"),
        # the rows of one long request taken out of their pages
        dict(name="read_long", kind="read", heads=32, kv_heads=8, dim=128, requests=1, cached=16000, page=64,
             dtype="bfloat16"),
        # rows of several short requests, in the 32-bit mode
        dict(name="read_float32", kind="read", heads=32, kv_heads=8, dim=64, requests=7, cached=203, page=16,
             dtype="float32"),
        # one user's long conversation: few rows, the keys are the work
        dict(name="decode_one_long", kind="decode", heads=32, kv_heads=8, dim=128, requests=1, cached=16383,
             window=0, keep=0, page=64, dtype="bfloat16"),
        # a small batch of ragged requests, the serving loop's usual step
        dict(name="decode_batch", kind="decode", heads=24, kv_heads=8, dim=128, requests=8, cached=2047,
             window=0, keep=0, page=16, dtype="bfloat16"),
        # many users, each with a window of keys and four first tokens that stay
        dict(name="decode_window", kind="decode", heads=32, kv_heads=8, dim=64, requests=64, cached=8000,
             window=1024, keep=4, page=16, dtype="bfloat16"),
        # a prompt from its start
        dict(name="chunk_prompt", kind="chunk", heads=24, kv_heads=8, dim=128, requests=1, new=2048, cached=0,
             window=0, keep=0, page=64, dtype="bfloat16"),
        # a later portion of a long prompt: the largest case
        dict(name="chunk_long", kind="chunk", heads=32, kv_heads=8, dim=128, requests=1, new=2048, cached=14336,
             window=0, keep=0, page=64, dtype="bfloat16"),
        # a few tokens on a long cache (a question about a document): few rows, long keys
        dict(name="chunk_few", kind="chunk", heads=32, kv_heads=8, dim=128, requests=2, new=17, cached=20000,
             window=0, keep=0, page=16, dtype="bfloat16"),
        # the 32-bit mode, odd portions with a window and kept first tokens
        dict(name="chunk_float32", kind="chunk", heads=32, kv_heads=8, dim=64, requests=2, new=251, cached=300,
             window=200, keep=3, page=16, dtype="float32"),
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], even over its logarithm, odd ones among them."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(("write", "read", "decode", "chunk"))
    heads, kv_heads, dim = rng.choice(HEADS)
    dtype = rng.choice(("bfloat16", "bfloat16", "bfloat16", "float32"))
    case = dict(kind=kind, heads=heads, kv_heads=kv_heads, dim=dim, page=rng.choice((16, 32, 64)), dtype=dtype)
    if kind == "write":
        case.update(rot=rng.choice((dim, dim // 2)), requests=_spread(rng, 1, 8), new=_spread(rng, 1, 512),
                    cached=_spread(rng, 1, 120000))
    elif kind == "read":
        case.update(requests=_spread(rng, 1, 8), cached=_spread(rng, 1, 2048))
    else:
        window = rng.choice((0, 0, _spread(rng, 16, 2000)))
        case.update(window=window, keep=rng.choice((0, 1, 4)) if window else 0)
        small = dtype == "float32"
        if kind == "decode":
            case.update(requests=_spread(rng, 1, 8 if small else 64), cached=_spread(rng, 1, 1000 if small else 8000))
        else:
            case.update(requests=_spread(rng, 1, 4), new=_spread(rng, 2, 128 if small else 512),
                        cached=_spread(rng, 1, 600 if small else 4000))
    return case


# ------------------------------------------------------------------ the rows' format
def _scale_exponent(x):
    """The exponent of each row's scale: the smallest e with max |x| <= 448 * 2^e."""
    most = x.abs().amax(-1, keepdim=True).double()
    mantissa, exponent = torch.frexp(most)                 # most = mantissa * 2^exponent, mantissa in [1/2, 1)
    e = exponent - 9 + (mantissa > 0.875).int()            # 448 = 0.875 * 2^9
    return torch.where(most > 0, e, torch.full_like(e, LEAST)).clamp(LEAST, MOST)


def _power(e):
    """2^e as floats, e whole numbers of [-126, 127]."""
    return ((e + 127) << 23).view(torch.float32)


def _quantise(x):
    """(codes as bytes, scale bytes) of the rows of x (its last dimension)."""
    e = _scale_exponent(x)
    codes = (x.double() * _power(-e).double()).clamp(-448, 448).float().to(torch.float8_e4m3fn)
    return codes.view(torch.uint8), (e + 127).to(torch.uint8).squeeze(-1)


def _values(codes, scales):
    """The float values that codes [..., dim] and scale bytes [...] stand for."""
    return codes.view(torch.float8_e4m3fn).float() * _power(scales.int() - 127).unsqueeze(-1)


# ------------------------------------------------------------------ inputs
def _lengths(case):
    """(new tokens, cached tokens before them) of every request, ragged where there are several."""
    n = case["requests"]
    new, cached = [case.get("new", 1)] * n, [case["cached"]] * n
    for r in range(1, n):
        part = (0.618034 * r) % 1.0
        cached[r] = int(cached[r] * (0.4 + 0.6 * part))
        if new[r] > 1:
            new[r] = max(1, int(new[r] * (1.0 - 0.5 * part)))
    return new, cached


def prepare(case, seed):
    dev, dt = torch.device(DEVICE), DTYPES[case["dtype"]]
    g = torch.Generator(device=dev).manual_seed(seed)
    nq, nkv, dim, page, kind = case["heads"], case["kv_heads"], case["dim"], case["page"], case["kind"]
    new, cached = _lengths(case)
    if kind == "read":
        new, cached = cached, [0] * len(cached)             # every cached row is asked for
    total = [a + b for a, b in zip(new, cached)]
    width = max(-(-t // page) for t in total)
    window, keep = case.get("window", 0), case.get("keep", 0)
    # pages that hold what is written or seen; the others have been given back (-1)
    table = torch.full((len(new), width), -1, dtype=torch.int32)
    held = []
    for r, t in enumerate(total):
        first = cached[r] if kind == "write" else max(0, cached[r] - window + 1) if window else 0
        held += [(r, p) for p in range(-(-t // page)) if p >= first // page or (keep and p <= (keep - 1) // page)]
    order = torch.randperm(len(held) + 3, generator=torch.Generator().manual_seed(seed + 5))
    at = torch.tensor(held)
    table[at[:, 0], at[:, 1]] = order[:len(held)].int()
    pages = len(held) + 3
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    req = [r for r, n in enumerate(new) for _ in range(n)]
    pos = [c + i for n, c in zip(new, cached) for i in range(n)]
    s = dict(case=case, table=table.to(dev), req=i32(req), pos=i32(pos), tokens=len(req),
             start=i32([sum(new[:r]) for r in range(len(new) + 1)]), kv_len=i32(total), max_new=max(new),
             max_len=max(total), scale=dim ** -0.5)
    # a few features of the keys are several times larger than the others, as trained ones are
    bias = 1.0 + 3.0 * (torch.rand(nkv, 1, dim, generator=g, device=dev) > 0.97).float()
    if kind == "write":
        qkv = torch.randn(len(req), (nq + 2 * nkv) * dim, generator=g, device=dev)
        qkv[:, nq * dim:(nq + nkv) * dim] *= bias.reshape(-1)
        s["qkv"] = qkv.to(dt)
        rot = case["rot"]
        s["freq"] = torch.tensor([500000.0 ** (-2.0 * j / rot) for j in range(rot // 2)], dtype=torch.float32, device=dev)
        s["cache"] = torch.zeros(pages, 2, nkv, page, dim, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn)
        s["scales"] = torch.zeros(pages, 2, nkv, page, dtype=torch.uint8, device=dev)
        return s
    rows = torch.randn(pages, 2, nkv, page, dim, generator=g, device=dev)
    rows[:, 0] *= bias
    rows *= torch.exp(0.3 * torch.randn(pages, 2, nkv, page, 1, generator=g, device=dev))   # rows differ in size
    codes, s["scales"] = _quantise(rows)
    s["cache"] = codes.view(torch.float8_e4m3fn)
    if kind != "read":
        s["q"] = (1.5 * torch.randn(len(req), nq * dim, generator=g, device=dev)).to(dt)
    return s


# ------------------------------------------------------------------ the plain forms
def _rotate(x, pos, freq):
    """Rotary encoding of x [tokens, heads, dim] in 64 bits, pairs (j, j + half)."""
    half = freq.numel()
    a = (pos.double()[:, None] * freq.double())[:, None]
    x = x.double()
    lo, hi, rest = x[..., :half], x[..., half:2 * half], x[..., 2 * half:]
    return torch.cat([lo * a.cos() - hi * a.sin(), hi * a.cos() + lo * a.sin(), rest], -1)


def _row_place(s):
    """(page, slot in it) of every token's cached row."""
    page = s["case"]["page"]
    pos = s["pos"].long()
    return s["table"][s["req"].long(), pos // page].long(), pos % page


def _plain_write(s):
    c = s["case"]
    nq, nkv, dim, dt = c["heads"], c["kv_heads"], c["dim"], DTYPES[c["dtype"]]
    x = s["qkv"].view(s["tokens"], nq + 2 * nkv, dim)
    qk = _rotate(x[:, :nq + nkv], s["pos"], s["freq"])
    rows = torch.stack([qk[:, nq:], x[:, nq + nkv:].double()], 1)             # [tokens, 2, kv heads, dim]
    codes, scales = _quantise(rows)
    page, slot = _row_place(s)
    cache = s["cache"].view(torch.uint8)
    cache[page, :, :, slot] = codes
    s["scales"][page, :, :, slot] = scales
    values = _values(cache[page, :, :, slot].contiguous(), s["scales"][page, :, :, slot])
    return {"q": qk[:, :nq].reshape(s["tokens"], nq * dim).to(dt), "rows": values.to(dt)}


def _plain_read(s):
    page, slot = _row_place(s)
    codes = s["cache"].view(torch.uint8)[page, :, :, slot].contiguous()
    return _values(codes, s["scales"][page, :, :, slot]).to(DTYPES[s["case"]["dtype"]])


def _plain_attention(s):
    c = s["case"]
    nq, nkv, dim, dt, page = c["heads"], c["kv_heads"], c["dim"], DTYPES[c["dtype"]], c["page"]
    entries, group, n = c["requests"], nq // nkv, s["max_len"]
    table = s["table"].long().clamp(min=0)
    codes = s["cache"].view(torch.uint8)[table]                               # [entries, width, 2, kv heads, page, dim]
    kv = _values(codes, s["scales"][table]).permute(2, 0, 3, 1, 4, 5).reshape(2, entries, nkv, -1, dim)[:, :, :, :n]
    req, turn = s["req"].long(), torch.arange(s["tokens"], device=s["req"].device) - s["start"].long()[s["req"].long()]
    q = torch.zeros(entries, s["max_new"], nq, dim, device=s["q"].device)
    q[req, turn] = s["q"].view(-1, nq, dim).float()
    q = q.view(entries, s["max_new"], nkv, group, dim).permute(0, 2, 1, 3, 4).reshape(entries, nkv, -1, dim)
    scores = (q * s["scale"]) @ kv[0].transpose(-1, -2)                       # [entries, kv heads, new * group, keys]
    place = torch.zeros(entries, s["max_new"], dtype=torch.long, device=q.device)
    place[req, turn] = s["pos"].long()
    place, key = place[:, :, None], torch.arange(n, device=q.device)[None, None]
    seen = key <= place
    if c["window"]:
        seen = seen & ((key > place - c["window"]) | (key < c["keep"]))
    seen = seen[:, None, :, None].expand(-1, 1, -1, group, -1).reshape(entries, 1, -1, n)
    scores = scores.masked_fill(~seen, float("-inf"))
    scores = (scores - scores.amax(-1, keepdim=True)).exp_()
    total = scores.sum(-1, keepdim=True)
    out = (scores @ kv[1]) / total
    out = out.view(entries, nkv, s["max_new"], group, dim).permute(0, 2, 1, 3, 4)[req, turn]
    return out.reshape(s["tokens"], nq * dim).to(dt)


def _own_run(s):
    from mstar_b200 import ops

    c = s["case"]
    nq, nkv, dim, page, kind = c["heads"], c["kv_heads"], c["dim"], c["page"], c["kind"]
    if kind == "write":
        q = ops.rope_kv8_write(s["qkv"], s["pos"], s["pos"], s["req"], s["table"], s["freq"], s["cache"], s["scales"],
                               nq, nkv, dim, c["rot"], False, page)
        return {"q": q, "rows": ops.kv8_read_rows(s["cache"], s["scales"], s["table"], s["req"], s["pos"],
                                                  DTYPES[c["dtype"]])}
    if kind == "read":
        return ops.kv8_read_rows(s["cache"], s["scales"], s["table"], s["req"], s["pos"], DTYPES[c["dtype"]])
    out = torch.empty_like(s["q"])
    if kind == "decode":
        ops.paged_decode_attention_kv8(s["q"], out, s["cache"], s["scales"], s["table"], s["req"], s["pos"],
                                       s["tokens"], nq, nkv, dim, page, c["window"], c["keep"], s["scale"], s["max_len"])
    else:
        ops.paged_prefill_attention_kv8(s["q"], out, s["cache"], s["scales"], s["table"], s["start"], s["kv_len"], 0,
                                        c["requests"], s["max_new"], nq, nkv, dim, page, c["window"], c["keep"],
                                        s["scale"], s["max_len"])
    return out


def run(state):
    if own:
        return _own_run(state)
    kind = state["case"]["kind"]
    if kind == "write":
        return _plain_write(state)
    if kind == "read":
        return _plain_read(state)
    return _plain_attention(state)


def _visible(case, place):
    window, keep = case.get("window", 0), case.get("keep", 0)
    if not window or place + 1 <= window:
        return place + 1
    return window + min(keep, place + 1 - window)


def work(case):
    nq, nkv, dim = case["heads"], case["kv_heads"], case["dim"]
    item = 2 if case["dtype"] == "bfloat16" else 4
    new, cached = _lengths(case)
    if case["kind"] == "read":
        new, cached = cached, [0] * len(cached)
    tokens, row = sum(new), 2 * nkv * (dim + 1)
    if case["kind"] == "write":         # in, rotated queries out, rows written, and read back as values
        return {"bytes": tokens * ((2 * nq + 4 * nkv) * dim * item + 2 * row), "flops": tokens * (6.0 * nq + 10.0 * nkv) * dim}
    if case["kind"] == "read":
        return {"bytes": tokens * (row + 2 * nkv * dim * item), "flops": tokens * 2.0 * nkv * dim}
    pairs = sum(_visible(case, c + i) for n, c in zip(new, cached) for i in range(n))
    keys = 0
    for n, c in zip(new, cached):       # the keys that some token of the request sees
        window = case["window"]
        first = max(0, c - window + 1) if window else 0
        keys += c + n - first + min(case["keep"], first)
    return {"bytes": keys * row + 2 * tokens * nq * dim * item, "flops": 4.0 * dim * nq * pairs}


# ------------------------------------------------------------------ the definition in 64 bits
def _row_values(s, request, first, last):
    """Keys and values [rows, 2, kv heads, dim] of positions first .. last - 1 of a request, in 64 bits."""
    page = s["case"]["page"]
    place = torch.arange(first, last, device=s["table"].device)
    pages = s["table"][request].long()[place // page]
    byte = s["cache"].view(torch.uint8)[pages, :, :, place % page].int()
    sign, expo, man = 1.0 - 2.0 * (byte >> 7).double(), (byte >> 3) & 15, (byte & 7).double()
    value = torch.where(expo > 0, (1.0 + man / 8.0) * torch.exp2(expo.double() - 7.0), man * 2.0 ** -9)
    return sign * value * torch.exp2(s["scales"][pages, :, :, place % page].double() - 127.0)[..., None]


def _exact_rows(x):
    """Each row of x rounded to the nearest number that its format can hold (ties to even), in 64 bits."""
    most = x.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(most / 448.0))
    e = torch.where(448.0 * torch.exp2(e - 1) >= most, e - 1, torch.where(448.0 * torch.exp2(e) < most, e + 1, e))
    y = x / torch.exp2(e)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step * torch.exp2(e)


def exact(case, seed):
    s = prepare(case, seed)
    nq, nkv, dim, kind = case["heads"], case["kv_heads"], case["dim"], case["kind"]
    new, cached = _lengths(case)
    if kind == "write":
        x = s["qkv"].double().view(s["tokens"], nq + 2 * nkv, dim)
        half = case["rot"] // 2
        turn = torch.polar(torch.ones(1, dtype=torch.float64, device=x.device), s["pos"].double()[:, None] * s["freq"].double())
        pair = torch.complex(x[:, :nq + nkv, :half].contiguous(), x[:, :nq + nkv, half:2 * half].contiguous()) * turn[:, None]
        x[:, :nq + nkv, :half], x[:, :nq + nkv, half:2 * half] = pair.real, pair.imag
        return {"q": x[:, :nq].reshape(s["tokens"], nq * dim),
                "rows": torch.stack([_exact_rows(x[:, nq:nq + nkv]), _exact_rows(x[:, nq + nkv:])], 1)}
    if kind == "read":
        return torch.cat([_row_values(s, r, 0, n) for r, n in enumerate(cached)])
    out = torch.empty(s["tokens"], nkv, nq // nkv, dim, dtype=torch.float64, device=s["q"].device)
    q = s["q"].double().view(s["tokens"], nkv, nq // nkv, dim)
    at = 0
    for r, (n, c) in enumerate(zip(new, cached)):
        first = max(0, c - case["window"] + 1) if case["window"] else 0
        kept = min(case["keep"], first)
        rows = torch.cat([_row_values(s, r, 0, kept), _row_values(s, r, first, c + n)])
        place = torch.cat([torch.arange(kept), torch.arange(first, c + n)]).to(rows.device)
        newest = torch.arange(c, c + n, device=rows.device)[:, None]
        hidden = place > newest
        if case["window"]:
            hidden = hidden | ((place <= newest - case["window"]) & (place >= case["keep"]))
        for h in range(nkv):
            scores = torch.einsum("tgd,kd->gtk", q[at:at + n, h], rows[:, 0, h]) * s["scale"]
            weights = torch.softmax(scores.masked_fill(hidden, float("-inf")), -1)
            out[at:at + n, h] = torch.einsum("gtk,kd->tgd", weights, rows[:, 1, h])
        at += n
    return out.reshape(s["tokens"], nq * dim)
