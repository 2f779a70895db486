"""The softmax-attention operators by their definitions, in 64 bits: the paged 8-bit cache
(cache_write, cache_read), attention over it (attention_decode, attention_prefill) and norm_rope
with several axes.  No counterpart in the reference.

Everything here runs on the CPU, request by request and page by page; tensors may be anywhere.  The
cache's layout and the requests are include/lightdelta_attention_hip.h's.

How far a correct implementation may be off (attention): the output's rounding to bf16 (2^-8 of the
value, half a step), the weights' to bf16 (each 2^-8 of itself, once as a numerator), and the scores'
errors, which are relative errors of the weights and their sum.  A score is a sum of 128 products in
32 bits, at most 2^-24 of the running magnitude an addition (128 of them, in any order), scaled by
log2(e) * scale and moved by the maximum (two roundings of at most 2^-23 of the score and of the
maximum); exp2 and the division are good to 2^-21.  The sum of n weights and the products with the
values, in 32 bits, are off by at most n 2^-24 of the sum of magnitudes.
"""

from __future__ import annotations

import math

import torch

DIM = 128
LOW, HIGH = -100, 119
LARGEST = 448.0


def e4m3_values() -> torch.Tensor:
    """The value of each of the 256 codes, from the format: sign, 4 bits of exponent (bias 7), 3 of
    fraction; exponent 0 is subnormal; all ones but the sign is NaN."""
    out = torch.empty(256, dtype=torch.float64)
    for code in range(256):
        e, m = code >> 3 & 15, code & 7
        x = m / 8 * 2.0**-6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
        if code & 127 == 127:
            x = math.nan
        out[code] = -x if code & 128 else x
    return out


_VALUES = e4m3_values()
_MAGNITUDES = _VALUES[:127]  # 0 .. 448, rising


def round_e4m3(x: torch.Tensor) -> torch.Tensor:
    """Codes (uint8) of the nearest values; of two equally near the one with an even fraction;
    magnitudes over 448 as 448, NaN as NaN."""
    m = x.abs().clamp(max=LARGEST).nan_to_num(0.0)
    above = torch.searchsorted(_MAGNITUDES, m).clamp(max=126)
    below = (above - 1).clamp(min=0)
    up, down = _MAGNITUDES[above] - m, m - _MAGNITUDES[below]
    code = torch.where((up < down) | ((up == down) & (above % 2 == 0)), above, below)
    code = torch.where(x.signbit(), code + 128, code)
    return torch.where(x.isnan(), 127, code).to(torch.uint8)


def scale_exponent(largest: float) -> int:
    """The least e with largest <= 448 * 2^e, within the scales' range."""
    e = LOW
    while e < HIGH and largest > LARGEST * 2.0**e:
        e += 1
    return e


def _k_index(page_size, token):
    """Flat places of a token's elements within a page and head of the k cache, then the v cache's."""
    d = torch.arange(DIM)
    return (d // 16 * page_size + token) * 16 + d % 16


def _v_index(page_size, token):
    d = torch.arange(DIM)
    return (token // 16 * DIM + d) * 16 + token % 16


INDEX = {"k": _k_index, "v": _v_index}


def _codes(cache):
    return cache.cpu().view(torch.uint8).contiguous().flatten(2)


def _scales(scale):
    return scale.cpu().view(torch.uint8)


def _places(pages, cu, lengths, rows, num_pages, page_size):
    """(row, request, page or 0, offset, position) of every row that a request has."""
    pages, cu, lengths = pages.cpu().tolist(), cu.cpu().tolist(), lengths.cpu().tolist()
    for r, length in enumerate(lengths):
        for row in range(max(cu[r], 0), min(cu[r + 1], rows)):
            position = length - cu[r + 1] + row
            page = 0
            if 0 <= position < len(pages[r]) * page_size:
                page = pages[r][position // page_size]
                page = page if 0 < page < num_pages else 0
            yield row, r, page, position % page_size, position


def expected_write(k, v, pages, cu, lengths, k_cache, v_cache, k_scale, v_scale):
    """(k codes, v codes, k scales, v scales) after the call, as uint8, in the caches' shapes."""
    page_size, num_pages = k_cache.shape[3], k_cache.shape[0]
    places = {}
    for row, _, page, offset, _ in _places(pages, cu, lengths, k.shape[0], num_pages, page_size):
        if page:
            places.setdefault(page, {})[offset] = row
    out = []
    for name, x, cache, scale in (("k", k, k_cache, k_scale), ("v", v, v_cache, v_scale)):
        codes, scales, x = _codes(cache).clone(), _scales(scale).clone(), x.cpu().double()
        for page, rows in places.items():
            first = min(rows)
            for h in range(x.shape[1]):
                new = x[list(rows.values()), h]
                finite = new[new.isfinite()].abs()
                e = scale_exponent(finite.max().item() if finite.numel() else 0.0)
                old = min(max(int(scales[page, h]) - 127, LOW), HIGH)
                if first > 0:
                    e = max(e, old)
                    for t in range(first):
                        at = INDEX[name](page_size, t)
                        codes[page, h, at] = round_e4m3(_VALUES[codes[page, h, at].long()]
                                                        * 2.0 ** (old - e))
                for offset, row in rows.items():
                    y = torch.where(x[row, h].isfinite(), x[row, h] * 2.0**-e, math.nan)
                    codes[page, h, INDEX[name](page_size, offset)] = round_e4m3(y)
                scales[page, h] = e + 127
        out.append((codes.view(cache.shape), scales))
    (kc, ks), (vc, vs) = out
    return kc, vc, ks, vs


def canonical(codes):
    """Codes with both NaNs as one and without the sign of zero."""
    codes = codes.cpu().view(torch.uint8)
    return torch.where(codes & 127 == 127, 127, torch.where(codes & 127 == 0, 0, codes))


def _token(codes, scales, name, page_size, page, head, offset):
    e = min(max(int(scales[page, head]) - 127, LOW), HIGH)
    return _VALUES[codes[page, head, INDEX[name](page_size, offset)].long()] * 2.0**e


def expected_read(pages, cu, lengths, k_cache, v_cache, k_scale, v_scale, k, v):
    """(k, v) after the call, in 64 bits."""
    page_size, num_pages = k_cache.shape[3], k_cache.shape[0]
    out = []
    for name, x, cache, scale in (("k", k, k_cache, k_scale), ("v", v, v_cache, v_scale)):
        codes, scales, x = _codes(cache), _scales(scale), x.cpu().double().clone()
        for row, _, page, offset, _ in _places(pages, cu, lengths, x.shape[0], num_pages,
                                               page_size):
            for h in range(x.shape[1]):
                x[row, h] = (_token(codes, scales, name, page_size, page, h, offset)
                             if page else 0.0)
        out.append(x)
    return out


def _context(codes, scales, name, page_size, table, length, num_pages):
    """A request's tokens [tokens, heads, 128] and which of them have a page."""
    n = min(max(length, 0), len(table) * page_size)
    order = torch.stack([INDEX[name](page_size, t) for t in range(page_size)])
    x = torch.zeros(n, codes.shape[1], DIM, dtype=torch.float64)
    live = torch.zeros(n, dtype=torch.bool)
    for i in range(-(-n // page_size)):
        page = table[i]
        if 0 < page < num_pages:
            low, high = i * page_size, min((i + 1) * page_size, n)
            e = (scales[page].double() - 127).clamp(LOW, HIGH)
            tokens = _VALUES[codes[page].long()][:, order] * (2.0**e)[:, None, None]
            x[low:high] = tokens.transpose(0, 1)[:high - low]
            live[low:high] = True
    return x, live


def expected_attention(q, pages, cu, lengths, k_cache, v_cache, k_scale, v_scale, gate, out, scale,
                       width=None):
    """(out, bound): the outputs in 64 bits, and how far each may be off."""
    page_size, num_pages = k_cache.shape[3], k_cache.shape[0]
    kc, vc, ks, vs = _codes(k_cache), _codes(v_cache), _scales(k_scale), _scales(v_scale)
    heads, kv_heads = q.shape[1], k_cache.shape[1]
    q, result = q.cpu().double(), out.cpu().double().clone()
    gate = None if gate is None else gate.cpu().double()
    bound = torch.zeros_like(result)
    table, cu, lengths = pages.cpu().tolist(), cu.cpu().tolist(), lengths.cpu().tolist()
    for r, length in enumerate(lengths):
        rows = range(max(cu[r], 0), min(cu[r + 1], q.shape[0]))
        if not len(rows):
            continue
        keys, live = _context(kc, ks, "k", page_size, table[r], length, num_pages)
        values, _ = _context(vc, vs, "v", page_size, table[r], length, num_pages)
        at = slice(rows[0], rows[-1] + 1)
        position = torch.tensor([length - cu[r + 1] + row for row in rows])
        sees = live & (torch.arange(len(keys)) <= position[:, None])
        if width is not None and len(rows) > width:
            sees = torch.zeros_like(sees)
        some = sees.any(1)
        for h in range(heads):
            j = h // (heads // kv_heads)
            x = q[at, h]
            s = scale * (x @ keys[:, j].t())
            size = scale * (x.abs() @ keys[:, j].abs().t())
            s = torch.where(sees, s, -math.inf)
            top = torch.where(some, s.amax(1) if len(keys) else 0.0, 0.0)[:, None]
            p = torch.exp(s - top)
            total = torch.where(some, p.sum(1), 1.0)[:, None]
            p = p / total
            # (a weight of zero keeps what is not finite in a value out only where it is not seen)
            o = torch.stack([p[i, sees[i]] @ values[sees[i], j] for i in range(len(rows))])
            big = torch.stack([p[i, sees[i]] @ values[sees[i], j].abs()
                               for i in range(len(rows))])
            off = torch.where(sees, 128 * 2.0**-24 * size + 2.0**-22 * (s.abs() + top.abs()),
                              0.0)
            off = off.amax(1, keepdim=True) if len(keys) else torch.zeros(len(rows), 1)
            error = big * (2.0**-8 + 2 * off + 2.0**-20 + 2 * len(keys) * 2.0**-24)
            if gate is not None:
                turn = torch.sigmoid(gate[at, h])
                turn = torch.where(some[:, None], turn, 0.0)
                o, error = o * turn, (error + 2.0**-20 * o.abs()) * turn
            result[at, h] = o
            bound[at, h] = error + 2.0**-8 * (o.abs() + error) + 2.0**-133
    return result, bound


def expected_norm_rope_axes(qkv, q_weight, k_weight, positions, axes, inv_freq, q_heads, k_heads,
                            eps, interleaved):
    """qkv after the call, in 64 bits (angles of the exact products while these hold in 64 bits)."""
    x = qkv.cpu().double().clone()
    rotary = 2 * inv_freq.numel()
    axes, positions = axes.cpu().tolist(), positions.cpu().double()
    angle = torch.zeros(x.shape[0], rotary // 2, dtype=torch.float64)
    for i, axis in enumerate(axes):
        if 0 <= axis < positions.shape[0]:
            angle[:, i] = positions[axis] * inv_freq.cpu().double()[i]
    first = [2 * i if interleaved else i for i in range(rotary // 2)]
    second = [2 * i + 1 if interleaved else i + rotary // 2 for i in range(rotary // 2)]
    for h in range(q_heads + k_heads):
        w = (q_weight if h < q_heads else k_weight).cpu().double()
        at = x[:, h * DIM:(h + 1) * DIM]
        y = at / torch.sqrt((at * at).mean(1, keepdim=True) + eps) * w
        at.copy_(y)
        a, b = y[:, first], y[:, second]
        at[:, first] = a * torch.cos(angle) - b * torch.sin(angle)
        at[:, second] = b * torch.cos(angle) + a * torch.sin(angle)
    return x
