"""Timing cases of the linear-attention operators: a decay for each head over the state pool
(`linear_decode`, `linear_prefill`), and the per-head norm with position rotation that goes
ahead of them (`norm_rope`).

`prepare` makes what a layer has in hand before the call, `run` is one call: the plain torch form
where `own` is false, the framework's operator where it is true.  `exact` is the definition in 64
bits, token by token.

A case is a dict of plain values; `op` names the operator.  Activations come as a layer hands them
over: bf16 rows of q, k and v columns (and the output gate beside them), heads of 128.  q and k are
about unit size, as they are behind a per-head norm; v ~ N(0, 1).  Decays are a constant slope per
head (2^(-8 (h + 1) / HV), from short to long memory) or per token
(-softplus(N(0, 1)) * U(0.01, 1) of the head).  Batches hold a padding request now and then, as a
captured batch size does.
"""

from __future__ import annotations

import math

import torch

own = False

DIM = 128
EPS = 1e-6
SCALE = DIM**-0.5


def listed():
    return [
        # One token of one request: the latency of a single call between two projections.
        _norm_rope("norm_rope_1", tokens=1),
        # A verify step of 37 requests, positions far into long contexts, interleaved pairs, a
        # quarter of the head rotated, grouped key heads, parameters in bf16.
        _norm_rope("norm_rope_111_partial", tokens=111, q_heads=32, k_heads=8, v_heads=8, rotary=32,
                   interleaved=True, bf16=True, far=4_000_000),
        # The prompts of a full prefill batch.
        _norm_rope("norm_rope_32768", tokens=32768),
        # One request of a small model (4/8 heads): the latency of a single call.
        _decode("linear_decode_b1_small", batch=1, heads=4, v_heads=8),
        # The decode step of an ordinary batch with the gated norm.
        _decode("linear_decode_b32", batch=32, gated=True),
        # A full odd batch, 16/48 heads, decays per token, a padding request, bf16 parameters.
        _decode("linear_decode_b119_hv48", batch=119, v_heads=48, gated=True, bf16=True, padding=1,
                per_token=True),
        # Speculative verify of up to 4 tokens a request.
        _decode("linear_verify_b64_t4", batch=64, width=4, gated=True),
        # One long new prompt: what time to first token waits for.
        _prefill("linear_prefill_1x4096", prompts=1, low=4096, high=4096, initial=0.0, gated=True),
        # A full batch of equal prompts that continue from a state.
        _prefill("linear_prefill_32x1024", prompts=32, low=1024, high=1024, gated=True),
        # Many short prompts of unequal length, decays per token.
        _prefill("linear_prefill_512x8to56", prompts=512, low=8, high=56, initial=0.5,
                 per_token=True),
        # A mixed batch: lengths from one token to thousands, 16/48 heads, bf16 parameters.
        _prefill("linear_prefill_13x1to3000_hv48", prompts=13, low=1, high=3000, v_heads=48,
                 initial=0.5, gated=True, bf16=True, per_token=True),
        # A few short extensions of running requests on one GPU's share of the heads.
        _prefill("linear_prefill_7x1to90_hv16", prompts=7, low=1, high=90, heads=8, v_heads=16),
    ]


def _norm_rope(name, tokens, q_heads=16, k_heads=16, v_heads=32, rotary=DIM, interleaved=False,
               bf16=False, far=0):
    return dict(name=name, op="norm_rope", tokens=tokens, q_heads=q_heads, k_heads=k_heads,
                v_heads=v_heads, rotary=rotary, interleaved=interleaved, bf16=bf16, far=far)


def _decode(name, batch, heads=16, v_heads=32, width=1, gated=False, bf16=False, per_token=False,
            padding=0):
    return dict(name=name, op="linear_decode", batch=batch, heads=heads, v_heads=v_heads,
                width=width, gated=gated, bf16=bf16, per_token=per_token, padding=padding)


def _prefill(name, prompts, low, high, heads=16, v_heads=32, initial=1.0, gated=False, bf16=False,
             per_token=False):
    return dict(name=name, op="linear_prefill", prompts=prompts, low=low, high=high, heads=heads,
                v_heads=v_heads, initial=initial, gated=gated, bf16=bf16, per_token=per_token)


def draw(rng):
    def log_int(low, high):
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    op = rng.choice(["norm_rope", "linear_decode", "linear_decode", "linear_prefill",
                     "linear_prefill", "linear_prefill"])
    heads, v_heads = rng.choice([(4, 8), (16, 32), (16, 32), (16, 48), (8, 16), (16, 16)])
    bf16, gated, per_token = (rng.random() < 0.5 for _ in range(3))
    if op == "norm_rope":
        q_heads, k_heads = rng.choice([(heads, heads), (heads, heads), (32, 8), (16, 2), (5, 1)])
        case = _norm_rope("", log_int(1, 32768), q_heads, k_heads, rng.choice([k_heads, 32]),
                          rng.choice([16, 32, 64, 96, 128, 128]), rng.random() < 0.5, bf16,
                          rng.choice([0, 0, 100_000, 8_000_000]))
    elif op == "linear_decode":
        width = rng.choice([1, 1, 1, 2, 3, 4])
        batch = log_int(1, 128 // width)
        case = _decode("", batch, heads, v_heads, width, gated, bf16, per_token,
                       1 if batch > 4 and rng.random() < 0.3 else 0)
    else:
        # tokens over three decades, prompts from one to as many as that allows
        tokens = log_int(16, 20000)
        prompts = min(log_int(1, 300), max(1, tokens // 4))
        mean = max(1, tokens // prompts)
        spread = rng.choice([0, mean // 2, mean - 1])
        case = _prefill("", prompts, mean - spread, mean + spread, heads, v_heads,
                        rng.choice([0.0, 0.5, 1.0]), gated, bf16, per_token)
    case.pop("name")
    return case


# ---- inputs ------------------------------------------------------------------------------


def _lengths(case):
    """Prompt lengths, spread evenly in the logarithm from `low` to `high` and shuffled (the
    same for every seed)."""
    n, low, high = case["prompts"], case["low"], case["high"]
    if low == high:
        return [low] * n
    if high < 8 * low:
        values = [round(low + (high - low) * (i + 0.5) / n) for i in range(n)]
    else:
        values = [round(math.exp(math.log(low) + math.log(high / low) * (i + 0.5) / n))
                  for i in range(n)]
    gen = torch.Generator().manual_seed(n)
    return [values[i] for i in torch.randperm(n, generator=gen).tolist()]


class _Source:
    """Random tensors on the GPU from one seed."""

    def __init__(self, seed):
        self.gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(self, *shape, std=1.0, dtype=torch.float32):
        x = torch.empty(shape, dtype=torch.float32, device="cuda").normal_(0.0, std,
                                                                          generator=self.gen)
        return x if dtype == torch.float32 else x.to(dtype)

    def uniform(self, *shape):
        return torch.rand(shape, generator=self.gen, device="cuda")

    def perm(self, n):
        return torch.randperm(n, generator=self.gen, device="cuda")


def prepare(case, seed):
    src = _Source(seed)
    if case["op"] == "norm_rope":
        tokens, rotary = case["tokens"], case["rotary"]
        cols = (case["q_heads"] + case["k_heads"] + case["v_heads"]) * DIM
        param = torch.bfloat16 if case["bf16"] else torch.float32
        start = src.uniform(tokens).mul(case["far"]).long()
        return dict(
            case=case, qkv=src.normal(tokens, cols, std=2.0, dtype=torch.bfloat16),
            q_weight=(1 + src.normal(DIM, std=0.1)).to(param),
            k_weight=(1 + src.normal(DIM, std=0.1)).to(param),
            positions=start + torch.arange(tokens, device="cuda"),
            inv_freq=10000.0 ** (-torch.arange(0, rotary, 2, device="cuda") / rotary))
    state = _layer(src, case)
    if case["op"] == "linear_prefill":
        lengths = _lengths(case)
        n = len(lengths)
        cu = torch.zeros(n + 1, dtype=torch.int32)
        cu[1:] = torch.cumsum(torch.tensor(lengths), 0)
        state.update(cu=cu.to("cuda"), slots=(src.perm(n) + 1).int(),
                     has_initial=src.uniform(n) < case["initial"], longest=max(lengths))
        return state
    batch, width = case["batch"], case["width"]
    # each request: 1 .. width tokens, its accepted length, and slots of its own
    lengths = src.uniform(batch).mul(width).int().clamp_(max=width - 1) + 1
    cu = torch.zeros(batch + 1, dtype=torch.int32, device="cuda")
    cu[1:] = torch.cumsum(lengths, 0)
    indices = (src.perm(batch * width) + 1).int().view(batch, width)
    if case["padding"]:
        indices[-case["padding"]:] = 0
    accepted = (src.uniform(batch) * width).int().clamp_(max=width - 1) + 1
    state.update(cu=cu, indices=indices, accepted=accepted)
    return state


def _layer(src, case):
    """One layer's activations, decays, parameters and state pool."""
    heads, v_heads = case["heads"], case["v_heads"]
    if case["op"] == "linear_prefill":
        tokens, slots = sum(_lengths(case)), case["prompts"] + 1
    else:  # a captured batch has rows for every token it may hold
        tokens = case["batch"] * case["width"]
        slots = tokens + 1
    cols, gate_cols = (2 * heads + v_heads) * DIM, v_heads * DIM
    rows = src.normal(tokens, cols + gate_cols, dtype=torch.bfloat16)
    slope = 2.0 ** (-8.0 * torch.arange(1, v_heads + 1, device="cuda") / v_heads)
    if case["per_token"]:
        rate = 0.01 + 0.99 * src.uniform(v_heads)
        log_decay = -torch.nn.functional.softplus(src.normal(tokens, v_heads)) * rate
    else:
        log_decay = -slope
    param = torch.bfloat16 if case["bf16"] else torch.float32
    return dict(
        case=case, qkv=rows[:, :cols], log_decay=log_decay,
        gate=rows[:, cols:].view(tokens, v_heads, DIM) if case["gated"] else None,
        weight=(1 + src.normal(DIM, std=0.1)).to(param) if case["gated"] else None,
        pool=src.normal(slots, v_heads, DIM, DIM),
        out=torch.zeros(tokens, v_heads, DIM, dtype=torch.bfloat16, device="cuda"))


# ---- one pass ----------------------------------------------------------------------------


def run(state):
    op = state["case"]["op"]
    if op == "norm_rope":
        (_own_norm_rope if own else _plain_norm_rope)(state)
        return {"qkv": state["qkv"]}
    if own:
        (_own_prefill if op == "linear_prefill" else _own_decode)(state)
    else:
        (_plain_prefill if op == "linear_prefill" else _plain_decode)(state)
    return {"out": state["out"], "pool": state["pool"]}


def _own_norm_rope(s):
    from lightdelta_amd import ops  # noqa: F401  -- registers torch.ops.lightdelta

    case = s["case"]
    torch.ops.lightdelta.norm_rope(s["qkv"], s["q_weight"], s["k_weight"], s["positions"],
                                   s["inv_freq"], case["q_heads"], case["k_heads"], EPS,
                                   case["interleaved"])


def _own_decode(s):
    from lightdelta_amd import ops  # noqa: F401

    torch.ops.lightdelta.linear_decode(s["qkv"], s["log_decay"], s["indices"], s["cu"],
                                       s["accepted"], s["pool"], s["gate"], s["weight"], s["out"],
                                       SCALE, EPS)


def _own_prefill(s):
    from lightdelta_amd import ops  # noqa: F401

    torch.ops.lightdelta.linear_prefill(s["qkv"], s["log_decay"], s["slots"], s["has_initial"],
                                        s["cu"], s["pool"], s["gate"], s["weight"], s["out"], SCALE,
                                        EPS)


# ---- the plain forms ---------------------------------------------------------------------


def _plain_norm_rope(s):
    case = s["case"]
    q_heads, k_heads, rotary = case["q_heads"], case["k_heads"], case["rotary"]
    width = (q_heads + k_heads) * DIM
    x = s["qkv"][:, :width].float().view(-1, q_heads + k_heads, DIM)
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    weight = torch.cat([s["q_weight"].float().expand(q_heads, DIM),
                        s["k_weight"].float().expand(k_heads, DIM)])
    x = x * weight
    angle = s["positions"].double()[:, None] * s["inv_freq"].double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    turned, rest = x[..., :rotary], x[..., rotary:]
    if case["interleaved"]:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = turned[..., :rotary // 2], turned[..., rotary // 2:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    s["qkv"][:, :width].copy_(torch.cat([turned, rest], -1).flatten(1))


def _finish(s, o):
    """Outputs [.., v_heads, 128] in 32 bits, gated norm over each head where the layer has one;
    `o` holds one row per row of the activations."""
    if s["gate"] is None:
        return o
    gate = s["gate"].float()
    o = o * torch.rsqrt((o * o).mean(-1, keepdim=True) + EPS) * s["weight"].float()
    return o * (gate * torch.sigmoid(gate))


def _plain_decode(s):
    case, pool, indices, cu = s["case"], s["pool"], s["indices"], s["cu"]
    heads, v_heads, width = case["heads"], case["v_heads"], case["width"]
    tokens, group = s["qkv"].shape[0], v_heads // heads
    accepted = s["accepted"]
    source = indices.gather(1, (accepted.clamp(1, width) - 1)[:, None].long()).flatten()
    lengths = cu[1:] - cu[:-1]
    valid = (accepted >= 1) & (accepted <= width) & (source > 0) & (lengths <= width)
    x = s["qkv"].float()
    q, k = (x[:, i * heads * DIM:(i + 1) * heads * DIM].view(tokens, heads, DIM)
            .repeat_interleave(group, 1) for i in range(2))
    v = x[:, 2 * heads * DIM:].view(tokens, v_heads, DIM)
    decay = s["log_decay"].exp().expand(tokens, v_heads)
    state = pool[source.clamp(min=0).long()]
    # one row more than the tokens: where rows that no request has go
    o = torch.zeros(tokens + 1, v_heads, DIM, device=pool.device)
    held, first = [], pool[:1].clone()
    for t in range(width):
        live = valid & (lengths > t)
        at = (cu[:-1] + t).clamp(max=tokens - 1).long()
        state = state * decay[at][:, :, None, None] + v[at][..., None] * k[at][:, :, None]
        value = SCALE * (state * q[at][:, :, None]).sum(-1)
        o.index_copy_(0, torch.where(live, at, tokens), value)
        held.append((torch.where(live & (indices[:, t] > 0), indices[:, t], 0).long(), state))
    for slot, value in held:
        pool.index_copy_(0, slot, torch.where((slot > 0)[:, None, None, None], value, first))
    o = _finish(s, o[:tokens])
    # rows of requests that are not valid are zeros; rows behind the last request stay
    row = torch.arange(tokens, device=pool.device)
    request = (row[:, None] >= cu[None, 1:]).sum(1)
    mine = (request < len(lengths))[:, None, None]
    good = valid[request.clamp(max=len(lengths) - 1)][:, None, None]
    s["out"].copy_(torch.where(mine, torch.where(good, o, 0.0), s["out"].float()))


def _plain_prefill(s, chunk=128):
    case, pool, slots, cu = s["case"], s["pool"], s["slots"], s["cu"]
    heads, v_heads = case["heads"], case["v_heads"]
    tokens, group = s["qkv"].shape[0], v_heads // heads
    n = slots.numel()
    from_slot = (slots > 0) & s["has_initial"]
    state = pool[slots.clamp(min=0).long()]
    state = torch.where(from_slot[:, None, None, None], state, 0.0)
    log_decay = s["log_decay"].expand(tokens, v_heads)
    o = torch.zeros(tokens + 1, v_heads, DIM, device=pool.device)
    for c0 in range(0, s["longest"], chunk):
        size = min(chunk, s["longest"] - c0)
        at = cu[:-1, None] + torch.arange(c0, c0 + size, device=pool.device)
        live = at < cu[1:, None]
        at = at.clamp(max=tokens - 1).long()
        x = torch.where(live[..., None], s["qkv"][at].float(), 0.0)
        q, k = (x[..., i * heads * DIM:(i + 1) * heads * DIM].view(n, size, heads, DIM)
                .transpose(1, 2).repeat_interleave(group, 1) for i in range(2))
        v = x[..., 2 * heads * DIM:].view(n, size, v_heads, DIM).transpose(1, 2).contiguous()
        g = torch.where(live[..., None], log_decay[at], 0.0).transpose(1, 2).double()
        c = g.cumsum(-1)
        past = torch.ones(size, size, dtype=torch.bool, device=pool.device).tril()
        between = torch.where(past, c[..., :, None] - c[..., None, :], -math.inf).exp().float()
        value = ((q @ k.transpose(-1, -2).contiguous()) * between) @ v
        value = value + (q @ state.transpose(-1, -2).contiguous()) * c.exp().float()[..., None]
        left = (c[..., -1:] - c).exp().float()
        state = (state * c[..., -1].exp().float()[..., None, None]
                 + (v * left[..., None]).transpose(-1, -2).contiguous() @ k.contiguous())
        value = (SCALE * value).transpose(1, 2).reshape(n * size, v_heads, DIM)
        o.index_copy_(0, torch.where(live, at, tokens).flatten(), value)
    s["out"].copy_(_finish(s, o[:tokens]))
    keep = slots > 0
    pool.index_copy_(0, torch.where(keep, slots, 0).long(),
                     torch.where(keep[:, None, None, None], state, pool[:1]))


# ---- what a pass cannot do without ---------------------------------------------------------


def work(case):
    if case["op"] == "norm_rope":
        elements = case["tokens"] * (case["q_heads"] + case["k_heads"]) * DIM
        return {"bytes": 4 * elements + 8 * case["tokens"], "flops": 8 * elements}
    heads, v_heads = case["heads"], case["v_heads"]
    tile = v_heads * DIM * DIM * 4
    token = 2 * DIM * (2 * heads + (3 if case["gated"] else 2) * v_heads)
    token += 4 * v_heads if case["per_token"] else 0
    step = 4 * v_heads * DIM * DIM  # the update and S q
    if case["op"] == "linear_prefill":
        tokens, n = sum(_lengths(case)), case["prompts"]
        return {"bytes": int(tokens * token + n * (1 + case["initial"]) * tile),
                "flops": tokens * step}
    batch, width = case["batch"] - case["padding"], case["width"]
    tokens = batch * (width + 1) / 2
    return {"bytes": int(tokens * token + (batch + tokens) * tile), "flops": int(tokens * step)}


# ---- the definition in 64 bits -------------------------------------------------------------


def exact(case, seed):
    """norm_rope by complex products; linear attention by its recurrence, token by token over
    the sequences that still have one (sorted by length, so that they are a prefix)."""
    s = prepare(case, seed)
    if case["op"] == "norm_rope":
        qkv = s["qkv"].double()
        heads = case["q_heads"] + case["k_heads"]
        half = case["rotary"] // 2
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                           s["positions"].double()[:, None] * s["inv_freq"].double())
        for h in range(heads):
            x = qkv[:, h * DIM:(h + 1) * DIM]
            w = s["q_weight" if h < case["q_heads"] else "k_weight"].double()
            y = x / (x.square().mean(1, keepdim=True) + EPS).sqrt() * w
            first = torch.arange(half, device="cuda") * (2 if case["interleaved"] else 1)
            second = first + (1 if case["interleaved"] else half)
            z = torch.complex(y[:, first], y[:, second]) * turn
            x.copy_(y)
            x[:, first], x[:, second] = z.real, z.imag
        return {"qkv": qkv}
    heads, v_heads = case["heads"], case["v_heads"]
    cu = s["cu"].tolist()
    pool, out = s["pool"].double(), s["out"].double()
    if case["op"] == "linear_prefill":
        order = sorted(range(case["prompts"]), key=lambda r: cu[r] - cu[r + 1])
        homes = s["slots"].long()[order]
        state = pool[homes] * s["has_initial"].double()[order, None, None, None]
    else:
        indices, accepted = s["indices"].tolist(), s["accepted"].tolist()
        order = [r for r in range(case["batch"]) if indices[r][0] > 0]
        order.sort(key=lambda r: cu[r] - cu[r + 1])
        state = pool[[indices[r][accepted[r] - 1] for r in order]]
    q_at, k_at = (torch.arange(v_heads, device="cuda") // (v_heads // heads) + i * heads
                  for i in range(2))
    for t in range(cu[order[0] + 1] - cu[order[0]] if order else 0):
        rows = [r for r in order if cu[r + 1] - cu[r] > t]
        at = torch.tensor([cu[r] + t for r in rows], device="cuda")
        x = s["qkv"][at].double().view(len(rows), -1, DIM)
        q, k, v = x[:, q_at], x[:, k_at], x[:, 2 * heads:]
        g = (s["log_decay"][at] if case["per_token"] else s["log_decay"]).double()
        now = state[:len(rows)]
        now.mul_(g.exp()[..., None, None]).add_(v[..., None] * k[:, :, None])
        o = torch.matmul(now, q[..., None])[..., 0] * SCALE
        if case["gated"]:
            gate = s["gate"][at].double()
            o = o / (o.square().mean(-1, keepdim=True) + EPS).sqrt() * s["weight"].double()
            o = o * gate * torch.sigmoid(gate)
        out[at] = o
        if case["op"] == "linear_decode":
            pool[[indices[r][t] for r in rows]] = now
    if case["op"] == "linear_prefill":
        pool[homes] = state
    return {"out": out, "pool": pool}
