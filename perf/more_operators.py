"""Timing cases of the softmax-attention operators: the per-head norm with rotary positions of
several axes (`norm_rope_axes`), the paged 8-bit cache (`cache_write`, `cache_read`), and attention
over it (`attention_decode`, `attention_prefill`).

`prepare` makes what a layer has in hand before the call, `run` is one call: the plain torch form
where `own` is false, the framework's operator where it is true.  `exact` is the definition in 64
bits.

A case is a dict of plain values; `op` names the operator.  Heads have 128 elements, `heads` query
heads share `kv_heads` key heads.  Request r of a batch has the rows cu[r] .. cu[r+1]-1, which are
the last of its lengths[r] tokens; token t of it lies in page pages[r, t // page].  Pages are handed
out in no order, page 0 is padding, and tables are wider than the longest request, as a server's
are.  Keys and values of a page and head are e4m3 with one power of two as their scale:

  k_cache [pages, kv_heads, 8, page, 16]      element d of a token at [d // 16, token, d % 16]
  v_cache [pages, kv_heads, page / 16, 128, 16]   element d at [token // 16, d, token % 16]
  k_scale, v_scale [pages, kv_heads]  e8m0

Queries, keys and values are about unit size, as they are behind a per-head norm.
"""

from __future__ import annotations

import math

import torch

own = False

DIM = 128
EPS = 1e-6
SCALE = DIM**-0.5
LOW, HIGH = -100, 119  # exponents of a scale
MOST = 448.0  # e4m3's largest value


def listed():
    return [
        # The decode step of an ordinary batch behind the projection: three axes (time, height,
        # width), frequencies shared out in runs.
        _norm_rope("norm_rope_axes_32", tokens=32, heads=16, kv_heads=2),
        # Prompts with images: axes in turn over the frequencies, a quarter of the head rotated.
        _norm_rope("norm_rope_axes_16384", tokens=16384, heads=32, kv_heads=8, rotary=64,
                   runs=False, bf16=True, interleaved=True),
        # One new token of each of 64 running requests, pages filled to any offset.
        _cache("cache_write_b64", "cache_write", requests=64, low=1, high=1, before=3000),
        # The keys and values of a full prefill batch, from the first token on.
        _cache("cache_write_32x1024", "cache_write", requests=32, low=1024, high=1024),
        # One short prefix back in 16 bits, small pages.
        _cache("cache_read_1x300", "cache_read", requests=1, low=300, high=300, kv_heads=2,
               page=16),
        # Whole contexts back in 16 bits, to be moved to a cache of another kind.
        _cache("cache_read_19x1to8000", "cache_read", requests=19, low=1, high=8000),
        # One request early in its answer: the latency of a single call.
        _attention("attention_decode_b1", "attention_decode", requests=1, low=1, high=1,
                   before=500),
        # A running batch of unequal contexts with an output gate and a padding request.
        _attention("attention_decode_b33_8000", "attention_decode", requests=33, low=1, high=1,
                   before=8000, heads=32, kv_heads=8, gated=True, padding=1),
        # Speculative verify of up to 4 tokens a request.
        _attention("attention_verify_b64_t4", "attention_decode", requests=64, low=1, high=4,
                   before=4000),
        # One long new prompt: what time to first token waits for.
        _attention("attention_prefill_1x8192", "attention_prefill", requests=1, low=8192,
                   high=8192, gated=True),
        # A mixed batch: prompts from one token on, some behind a cached prefix, small pages.
        _attention("attention_prefill_13x1to1500", "attention_prefill", requests=13, low=1,
                   high=1500, before=1000, heads=32, kv_heads=8, page=16),
        # A few short questions about long documents.
        _attention("attention_prefill_3x20to90_30000", "attention_prefill", requests=3, low=20,
                   high=90, before=30000, page=128),
    ]


def _norm_rope(name, tokens, heads, kv_heads, rotary=DIM, runs=True, bf16=False,
               interleaved=False):
    return dict(name=name, op="norm_rope_axes", tokens=tokens, heads=heads, kv_heads=kv_heads,
                rotary=rotary, runs=runs, bf16=bf16, interleaved=interleaved)


def _cache(name, op, requests, low, high, before=0, kv_heads=8, page=64, padding=0):
    return dict(name=name, op=op, requests=requests, low=low, high=high, before=before,
                heads=kv_heads, kv_heads=kv_heads, page=page, padding=padding, gated=False)


def _attention(name, op, requests, low, high, before=0, heads=16, kv_heads=2, page=64,
               gated=False, padding=0):
    return dict(name=name, op=op, requests=requests, low=low, high=high, before=before,
                heads=heads, kv_heads=kv_heads, page=page, padding=padding, gated=gated)


def draw(rng):
    def log_int(low, high):
        return int(round(math.exp(rng.uniform(math.log(low), math.log(max(low, high))))))

    op = rng.choice(["norm_rope_axes", "cache_write", "cache_read", "attention_decode",
                     "attention_decode", "attention_prefill", "attention_prefill"])
    heads, kv_heads = rng.choice([(16, 2), (16, 2), (32, 8), (16, 16), (5, 1), (12, 4), (16, 1)])
    page = rng.choice([16, 32, 64, 64, 128])
    gated = rng.random() < 0.5
    if op == "norm_rope_axes":
        case = _norm_rope("", log_int(1, 16384), heads, kv_heads,
                          rng.choice([16, 32, 64, 96, 128, 128]), rng.random() < 0.5,
                          rng.random() < 0.5, rng.random() < 0.5)
    elif op in ("cache_write", "cache_read"):
        requests = log_int(1, 200)
        high = log_int(1, max(1, 200000 // (requests * kv_heads)))
        case = _cache("", op, requests, rng.choice([1, high]), high,
                      rng.choice([0, log_int(1, 100)]), kv_heads, page,
                      1 if requests > 4 and rng.random() < 0.3 else 0)
    elif op == "attention_decode":
        width = rng.choice([1, 1, 1, 2, 3, 4])
        requests = log_int(1, 128 // width)
        before = log_int(1, min(100000, 800000 // (requests * kv_heads)))
        case = _attention("", op, requests, 1, width, before, heads, kv_heads, page, gated,
                          1 if requests > 4 and rng.random() < 0.3 else 0)
    else:
        # prompts of all lengths; pairs of queries and keys at most a few hundred million
        requests = log_int(1, 40)
        high = log_int(2, min(6000, 12000 // requests))
        before = rng.choice([0, log_int(1, min(60000, 400000000 // (requests * high * heads)))])
        case = _attention("", op, requests, rng.choice([1, (high + 1) // 2, high]), high, before,
                          heads, kv_heads, page, gated)
    case.pop("name")
    return case


# ---- inputs ------------------------------------------------------------------------------


def _spread(n, low, high, seed):
    """n whole numbers spread evenly from low to high (in the logarithm over a wide range), in an
    order that is the same for every seed."""
    if high < 8 * low:
        values = [round(low + (high - low) * (i + 0.5) / n) for i in range(n)]
    else:
        values = [round(math.exp(math.log(low) + math.log(high / low) * (i + 0.5) / n))
                  for i in range(n)]
    gen = torch.Generator().manual_seed(seed)
    return [values[i] for i in torch.randperm(n, generator=gen).tolist()]


def _lengths(case):
    """Of each request: its new tokens, and all of them with those of before."""
    n = case["requests"]
    new = _spread(n, case["low"], case["high"], n)
    before = [0] * n
    if case["before"]:
        before = _spread(n, max(1, case["before"] // 8), case["before"], n + 1)
    live = n - case["padding"]
    return new, [a + b if r < live else 0 for r, (a, b) in enumerate(zip(new, before))]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0):
        return torch.empty(shape, device="cuda").normal_(0.0, std, generator=gen)

    heads, kv_heads = case["heads"], case["kv_heads"]
    if case["op"] == "norm_rope_axes":
        tokens, rotary = case["tokens"], case["rotary"]
        param = torch.bfloat16 if case["bf16"] else torch.float32
        half = torch.arange(rotary // 2, device="cuda", dtype=torch.int32)
        at = torch.arange(tokens, device="cuda")
        # text, then a grid of 40 x 40 places a frame: time, height, width
        start = int(torch.randint(0, 30000, (), generator=gen, device="cuda"))
        positions = torch.stack([start + at // 1600, start + at // 40 % 40, start + at % 40])
        return dict(
            case=case, qkv=normal(tokens, (heads + 2 * kv_heads) * DIM, std=2.0).bfloat16(),
            q_weight=(1 + normal(DIM, std=0.1)).to(param),
            k_weight=(1 + normal(DIM, std=0.1)).to(param), positions=positions,
            axes=(half * 3) // max(1, rotary // 2) if case["runs"] else half % 3,
            inv_freq=10000.0 ** (-torch.arange(0, rotary, 2, device="cuda") / rotary))

    page = case["page"]
    new, lengths = _lengths(case)
    n, tokens = len(new), sum(new)
    held = [-(-x // page) for x in lengths]
    cu = torch.zeros(n + 1, dtype=torch.int32)
    cu[1:] = torch.cumsum(torch.tensor(new), 0)
    # each request's pages, out of a pool a little larger than all of them
    count = sum(held) + 3
    ids = (torch.randperm(count - 1, generator=gen, device="cuda") + 1).int().cpu()
    pages = torch.zeros(n, 2 * max(held) + 1, dtype=torch.int32)
    at = 0
    for r, h in enumerate(held):
        pages[r, :h] = ids[at:at + h]
        at += h
    rows = normal(tokens, (heads + 2 * kv_heads) * DIM).bfloat16()
    q, k, v = (x.view(tokens, -1, DIM) for x in
               rows.split([heads * DIM, kv_heads * DIM, kv_heads * DIM], 1))

    # the cache: blocks whose loudness differs by a few powers of two, quantised as a whole
    def cache(*shape):
        x = normal(count, kv_heads, *shape)
        x = x * normal(count, kv_heads, 1, 1, 1).exp2()
        scale = _exponent(x.abs().amax((2, 3, 4)).bfloat16().float())
        return ((x * _power(-scale)[:, :, None, None, None]).clamp(-MOST, MOST)
                .to(torch.float8_e4m3fn), (scale + 127).to(torch.uint8))

    k_cache, k_scale = cache(8, page, 16)
    v_cache, v_scale = cache(page // 16, DIM, 16)
    state = dict(
        case=case, cu=cu.cuda(), lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"),
        pages=pages.cuda(), k_cache=k_cache, v_cache=v_cache,
        k_scale=k_scale.view(torch.float8_e8m0fnu), v_scale=v_scale.view(torch.float8_e8m0fnu),
        longest=max(lengths), most=max(new))
    if case["op"] == "cache_write":
        state.update(k=k, v=v)
    elif case["op"] == "cache_read":
        state.update(k=torch.zeros(tokens, kv_heads, DIM, dtype=torch.bfloat16, device="cuda"),
                     v=torch.zeros(tokens, kv_heads, DIM, dtype=torch.bfloat16, device="cuda"))
    else:
        gate = normal(tokens, heads, DIM).bfloat16() if case["gated"] else None
        state.update(q=q, gate=gate, out=torch.zeros(tokens, heads, DIM, dtype=torch.bfloat16,
                                                     device="cuda"))
    return state


def _exponent(most):
    """The least e with most <= 448 * 2^e, within a scale's range."""
    fraction, e = torch.frexp(most.double() / MOST)
    e = torch.where(fraction == 0.5, e - 1, e)
    return torch.where(most > 0, e, LOW).clamp(LOW, HIGH).int()


def _power(e):
    """2^e in 32 bits, every bit of it; 2^-126 below that."""
    return ((e.clamp(min=-126) + 127) << 23).view(torch.float32)


# ---- one pass ----------------------------------------------------------------------------


def run(state):
    op = state["case"]["op"]
    if own:
        _own(state)
    elif op == "norm_rope_axes":
        _plain_norm_rope(state)
    elif op == "cache_write":
        _plain_write(state)
    elif op == "cache_read":
        _plain_read(state)
    else:
        _plain_attention(state)
    if op == "norm_rope_axes":
        return {"qkv": state["qkv"]}
    if op == "cache_write":
        return {"k": state["k_cache"], "v": state["v_cache"],
                "k_scale": state["k_scale"].view(torch.uint8),
                "v_scale": state["v_scale"].view(torch.uint8)}
    if op == "cache_read":
        return {"k": state["k"], "v": state["v"]}
    return {"out": state["out"]}


def _own(s):
    from lightdelta_amd import ops  # noqa: F401  -- registers torch.ops.lightdelta

    case, op = s["case"], torch.ops.lightdelta
    if case["op"] == "norm_rope_axes":
        op.norm_rope_axes(s["qkv"], s["q_weight"], s["k_weight"], s["positions"], s["axes"],
                          s["inv_freq"], case["heads"], case["kv_heads"], EPS,
                          case["interleaved"])
        return
    where = (s["pages"], s["cu"], s["lengths"])
    cache = (s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"])
    if case["op"] == "cache_write":
        op.cache_write(s["k"], s["v"], *where, *cache)
    elif case["op"] == "cache_read":
        op.cache_read(*where, *cache, s["k"], s["v"])
    elif case["op"] == "attention_decode":
        op.attention_decode(s["q"], *where, *cache, s["gate"], s["out"], case["high"], SCALE)
    else:
        op.attention_prefill(s["q"], *where, *cache, s["gate"], s["out"], SCALE)


# ---- the plain forms ---------------------------------------------------------------------


def _plain_norm_rope(s):
    case = s["case"]
    heads, kv_heads, rotary = case["heads"], case["kv_heads"], case["rotary"]
    width = (heads + kv_heads) * DIM
    x = s["qkv"][:, :width].float().view(-1, heads + kv_heads, DIM)
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    x = x * torch.cat([s["q_weight"].float().expand(heads, DIM),
                       s["k_weight"].float().expand(kv_heads, DIM)])
    angle = s["positions"].double()[s["axes"].long()].t() * s["inv_freq"].double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    turned, rest = x[..., :rotary], x[..., rotary:]
    if case["interleaved"]:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = turned[..., :rotary // 2], turned[..., rotary // 2:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    s["qkv"][:, :width].copy_(torch.cat([turned, rest], -1).flatten(1))


def _plain_write(s):
    cu, lengths, pages, size = s["cu"], s["lengths"], s["pages"], s["case"]["page"]
    n, width = pages.shape
    # the pages that each request may write, and the tokens in them
    start = lengths - (cu[1:] - cu[:-1])
    at = start.clamp(min=0)[:, None] // size + torch.arange((s["most"] + 2 * size - 2) // size,
                                                            device=cu.device)
    position = at[..., None] * size + torch.arange(size, device=cu.device)
    page = pages.gather(1, at.clamp(max=width - 1).long())
    fresh = (position >= start[:, None, None]) & (position < lengths[:, None, None])
    used = fresh.any(-1) & (at < width) & (page > 0) & (page < s["k_cache"].shape[0])
    page = torch.where(used, page, 0).long().flatten()
    fresh = (fresh & used[..., None]).flatten(0, 1)[..., None, None]
    kept = ((position < start[:, None, None]) & used[..., None]).flatten(0, 1)[..., None, None]
    row = (position + (cu[1:] - lengths)[:, None, None]).flatten(0, 1)
    row = row.clamp(0, s["k"].shape[0] - 1).long()
    for name in ("k", "v"):
        cache, scale = s[name + "_cache"].view(torch.uint8), s[name + "_scale"].view(torch.uint8)
        new = torch.where(fresh, s[name][row].float(), 0.0)  # [pages, tokens, heads, 128]
        e = _exponent(torch.where(new.isfinite(), new.abs(), 0.0).amax((1, 3)))
        old = scale[page].int() - 127
        e = torch.where(kept[:, 0, 0], torch.maximum(e, old.clamp(LOW, HIGH)), e)
        code = _by_token(cache[page], name)
        held = code.view(torch.float8_e4m3fn).float() * _power(old - e)[:, None, :, None]
        value = (new * _power(-e)[:, None, :, None]).clamp(-MOST, MOST)
        value = torch.where(new.isfinite(), value, math.nan)
        value = torch.where(fresh, value, held).to(torch.float8_e4m3fn).view(torch.uint8)
        code = torch.where(fresh | kept, value, code)
        if name == "k":
            code = code.view(len(page), size, -1, 8, 16).permute(0, 2, 3, 1, 4)
        else:
            code = code.view(len(page), size // 16, 16, -1, DIM).permute(0, 3, 1, 4, 2)
        # (what is not used writes page 0 as it was)
        cache.index_copy_(0, page, code.contiguous())
        scale.index_copy_(0, page, torch.where(used.flatten()[:, None], e + 127, old + 127)
                          .to(torch.uint8))


def _by_token(x, name):
    """Pages of the k or v cache [pages, ...] as [pages, tokens, heads, 128], contiguous."""
    x = x.permute(0, 3, 1, 2, 4) if name == "k" else x.permute(0, 2, 4, 1, 3)
    return x.flatten(3, 4).contiguous() if name == "k" else x.flatten(1, 2).contiguous()


def _values(s, name, page, offset):
    """The values of the tokens at `offset` of `page`: [..., heads, 128], in 32 bits."""
    code = s[name + "_cache"].view(torch.uint8)
    if name == "k":
        code = code[page, :, :, offset].flatten(-2)
    else:
        code = code[page, :, offset // 16, :, offset % 16]
    e = s[name + "_scale"].view(torch.uint8)[page].int() - 127
    return code.view(torch.float8_e4m3fn).float() * _power(e)[..., None]


def _plain_read(s):
    cu, lengths, pages, size = s["cu"].long(), s["lengths"].long(), s["pages"], s["case"]["page"]
    row = torch.arange(s["k"].shape[0], device=cu.device)
    request = (torch.searchsorted(cu, row, right=True) - 1).clamp(0, len(lengths) - 1)
    position = lengths[request] - cu[request + 1] + row
    held = (position >= 0) & (position < pages.shape[1] * size)
    at = position.clamp(0, pages.shape[1] * size - 1)
    page = torch.where(held, pages[request, at // size], 0).long()
    page = torch.where((page > 0) & (page < s["k_cache"].shape[0]), page, 0)
    mine = (row < cu[-1])[:, None, None]
    for name in ("k", "v"):
        value = torch.where((page > 0)[:, None, None], _values(s, name, page, at % size), 0.0)
        s[name].copy_(torch.where(mine, value, s[name].float()))


def _plain_attention(s):
    case, cu, lengths, pages, q = s["case"], s["cu"], s["lengths"], s["pages"], s["q"]
    heads, kv_heads, size = case["heads"], case["kv_heads"], case["page"]
    tokens, group, n = q.shape[0], heads // kv_heads, cu.numel() - 1
    at = torch.arange(s["longest"], device=q.device)
    page = pages[:, at // size]
    live = (page > 0) & (page < s["k_cache"].shape[0]) & (at < lengths[:, None])
    page, offset = torch.where(live, page, 0).long(), (at % size).expand(n, -1)
    k, v = (torch.where(live[..., None, None],
                        _values(s, x, page, offset), 0.0)
            for x in ("k", "v"))
    row = cu[:-1, None] + torch.arange(s["most"], device=q.device)
    real = row < cu[1:, None]
    row = row.clamp(max=tokens - 1).long()
    x = q[row].float().view(n, -1, kv_heads, group, DIM).transpose(1, 2).flatten(2, 3)
    scores = SCALE * (x @ k.permute(0, 2, 3, 1).contiguous())  # [n, kv_heads, rows, keys]
    position = lengths[:, None] - cu[1:, None] + row
    sees = live[:, None] & (at <= position[..., None])
    sees = sees.repeat_interleave(group, 1)[:, None]
    scores = scores.masked_fill_(~sees, -math.inf)
    top = scores.amax(-1, keepdim=True)
    scores = scores.sub_(torch.where(sees.any(-1, keepdim=True), top, 0.0)).exp_()
    total = scores.sum(-1, keepdim=True)
    o = (scores @ v.transpose(1, 2).contiguous()) / torch.where(total > 0, total, 1.0)
    o = o.view(n, kv_heads, -1, group, DIM).transpose(1, 2).flatten(2, 3).flatten(0, 1)
    result = torch.cat([s["out"].float(), torch.zeros_like(o[:1])])
    result = result.index_copy(0, torch.where(real, row, tokens).flatten(), o)[:tokens]
    if s["gate"] is not None:
        mine = (torch.arange(tokens, device=q.device) < cu[-1])[:, None, None]
        result = torch.where(mine, result * torch.sigmoid(s["gate"].float()), result)
    s["out"].copy_(result)


# ---- what a pass cannot do without ---------------------------------------------------------


def work(case):
    if case["op"] == "norm_rope_axes":
        elements = case["tokens"] * (case["heads"] + case["kv_heads"]) * DIM
        return {"bytes": 4 * elements + 24 * case["tokens"], "flops": 8 * elements}
    new, lengths = _lengths(case)
    live = [(a, b) for a, b in zip(new, lengths) if b]
    tokens, row = sum(a for a, _ in live), case["kv_heads"] * DIM
    if case["op"] in ("cache_write", "cache_read"):
        return {"bytes": 6 * tokens * row, "flops": 4 * tokens * row}
    out = tokens * case["heads"] * DIM * (6 if case["gated"] else 4)
    pairs = sum(a * b - a * (a - 1) // 2 for a, b in live)
    return {"bytes": 2 * row * sum(b for _, b in live) + out,
            "flops": 4 * DIM * case["heads"] * pairs}


# ---- the definition in 64 bits -------------------------------------------------------------


def _double_power(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _round8(x):
    """To the nearest e4m3 value, ties to even, of numbers within its range."""
    e = torch.frexp(x)[1] - 1
    step = _double_power(e.clamp(min=-6) - 3)
    return torch.round(x / step) * step


def _decoded(s, name):
    """Codes' values and scales of a whole cache: [pages, tokens, heads, 128], [pages, heads]."""
    x, page = s[name + "_cache"].float().double(), s["case"]["page"]
    x = x.permute(*((0, 3, 1, 2, 4) if name == "k" else (0, 2, 4, 1, 3)))
    return (x.reshape(x.shape[0], page, -1, DIM),
            _double_power(s[name + "_scale"].view(torch.uint8).long() - 127))


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm_rope_axes":
        qkv = s["qkv"].double()
        half = case["rotary"] // 2
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), torch.stack(
            [s["positions"][a].double() * s["inv_freq"][i].double()
             for i, a in enumerate(s["axes"].tolist())], 1))
        for h in range(case["heads"] + case["kv_heads"]):
            x = qkv[:, h * DIM:(h + 1) * DIM]
            w = s["q_weight" if h < case["heads"] else "k_weight"].double()
            y = x / (x.square().mean(1, keepdim=True) + EPS).sqrt() * w
            first = torch.arange(half, device="cuda") * (2 if case["interleaved"] else 1)
            second = first + (1 if case["interleaved"] else half)
            z = torch.complex(y[:, first], y[:, second]) * turn
            x.copy_(y)
            x[:, first], x[:, second] = z.real, z.imag
        return {"qkv": qkv}
    page, cu, lengths = case["page"], s["cu"].tolist(), s["lengths"].tolist()
    table = s["pages"].tolist()
    if case["op"] == "cache_write":
        return _exact_write(s, page, cu, lengths, table)
    keys, k_scale = _decoded(s, "k")
    values, v_scale = _decoded(s, "v")
    heads, kv_heads = case["heads"], case["kv_heads"]
    result = (dict(k=s["k"].double(), v=s["v"].double()) if case["op"] == "cache_read"
              else dict(out=s["out"].double()))
    for r, length in enumerate(lengths):
        if not length:
            continue
        ids = table[r][:-(-length // page)]
        k = (keys[ids] * k_scale[ids][:, None, :, None]).flatten(0, 1)[:length]
        v = (values[ids] * v_scale[ids][:, None, :, None]).flatten(0, 1)[:length]
        n = cu[r + 1] - cu[r]
        if case["op"] == "cache_read":
            result["k"][cu[r]:cu[r + 1]], result["v"][cu[r]:cu[r + 1]] = k[-n:], v[-n:]
            continue
        future = torch.ones(n, length, dtype=torch.bool, device="cuda").triu(length - n + 1)
        for h in range(heads):
            j = h // (heads // kv_heads)
            a = s["q"][cu[r]:cu[r + 1], h].double() @ k[:, j].t().contiguous() * SCALE
            a = torch.softmax(a.masked_fill(future, -math.inf), -1)
            result["out"][cu[r]:cu[r + 1], h] = a @ v[:, j].contiguous()
        if case["gated"]:
            rows = result["out"][cu[r]:cu[r + 1]]
            rows /= 1 + torch.exp(-s["gate"][cu[r]:cu[r + 1]].double())
    return result


def _exact_write(s, page, cu, lengths, table):
    """Page by page over the pages that the call writes."""
    found = {}
    for name in ("k", "v"):
        held, scale = _decoded(s, name)
        for r, length in enumerate(lengths):
            if not length:
                continue
            start = length - (cu[r + 1] - cu[r])
            for first in range(start // page * page, length, page):
                low, high = max(first, start), min(first + page, length)
                x = s[name][cu[r] + low - start:cu[r] + high - start].double()
                p = table[r][first // page]
                most = x.abs().amax((0, 2)).clamp(min=1e-300)
                need = _double_power(torch.ceil(torch.log2(most / MOST) - 1e-9).clamp(LOW, HIGH))
                if low > first:
                    need = torch.maximum(need, scale[p])
                    before = held[p, :low - first]
                    before.copy_(_round8(before * (scale[p] / need)[:, None]))
                held[p, low - first:high - first] = _round8(
                    (x / need[:, None]).clamp(-MOST, MOST))
                scale[p] = need
        if name == "k":
            held = held.view(*held.shape[:3], 8, 16).permute(0, 2, 3, 1, 4)
        else:
            held = held.view(held.shape[0], page // 16, 16, -1, DIM).permute(0, 3, 1, 4, 2)
        found[name] = held.contiguous()
        found[name + "_scale"] = (torch.frexp(scale)[1] + 126).to(torch.uint8)
    return found
