"""The linear-attention operators' definitions in 64 bits, token by token, and how far an
implementation in 32 bits may be off.

  S <- exp(g) S + v k^T ;  o = scale * S q ;  out = o, or o * rsqrt(mean(o^2) + eps) * w * silu(gate)

Every function returns values and, for computed numbers, a bound on the error of a correct
implementation that holds states and sums in fp32 and rounds outputs to bf16 once.  With `A` the
same recurrence over absolute values (what a term's rounding is relative to):
  state   A * (n + 64) * 2^-22: an entry's term is decayed over up to n tokens, each decay within
          2^-22 (an exponential's and a product's rounding), and is one of up to 128 summed terms
          of a chunk or an update, a few roundings of 2^-24 each
  o       A * (n + 64) * 2^-22 + A * 2^-16: the state's, and sums over 128 keys and 64 tokens
          (192 * 2^-24)
  out     half a bf16 step (2^-8 of the value), and what o's bound comes to behind the norm:
          its own element's, and through the root mean square at most the row's
"""

from __future__ import annotations

import torch

DIM = 128


def geometry(qkv, pool):
    hv = pool.shape[1]
    return (qkv.shape[1] // DIM - hv) // 2, hv


def _recur(qkv, log_decay, heads, v_heads, rows, state, scale, visit):
    """Steps one sequence's `state` [2, HV, V, K] (values, magnitudes) through `rows`; visit(t,
    row, o, magnitude, state) after each."""
    group = v_heads // heads
    which = torch.arange(v_heads, device=qkv.device) // group
    for t, row in enumerate(rows):
        x = qkv[row].double().view(-1, DIM)
        q, k, v = x[which], x[heads + which], x[2 * heads:]
        g = (log_decay[row] if log_decay.dim() == 2 else log_decay).double()
        term = v[:, :, None] * k[:, None, :]
        state = state * g.exp()[None, :, None, None] + torch.stack([term, term.abs()])
        o = scale * (state[0] * q[:, None, :]).sum(-1)
        magnitude = abs(scale) * (state[1] * q.abs()[:, None, :]).sum(-1)
        visit(t, row, o, magnitude, state)
    return state


def _finish(o, o_bound, gate, weight, eps):
    """(out, bound) of one token's o [HV, 128]."""
    if gate is not None:
        gate, weight = gate.double(), weight.double()
        mean = o.square().mean(-1, keepdim=True) + eps
        factor = weight * gate * torch.sigmoid(gate) * mean.rsqrt()
        row = (o_bound.square().mean(-1, keepdim=True) / mean).sqrt()
        o_bound = factor.abs() * (o_bound + o.abs() * (row + 2.0**-20))
        o = o * factor
    return o, o_bound + o.abs() * 2.0**-8 + 1e-30


def _bounds(n, magnitude, state):
    held = (n + 64) * 2.0**-22
    return magnitude * (held + 2.0**-16), state[1] * held


def expected_linear_decode(qkv, log_decay, indices, cu, accepted, pool, gate, weight, out, scale,
                           eps):
    """(out, out bound, pool, pool bound) of one decode or verify step."""
    heads, v_heads = geometry(qkv, pool)
    out, new_pool = out.double(), pool.double()
    out_bound, pool_bound = torch.zeros_like(out), torch.zeros_like(new_pool)
    width = indices.shape[1]
    live = lambda s: 0 < s < pool.shape[0]  # noqa: E731
    for r, slots in enumerate(indices.tolist()):
        first, last, taken = int(cu[r]), int(cu[r + 1]), int(accepted[r])
        if last <= first:
            continue
        if not 1 <= taken <= width or not live(slots[taken - 1]) or last - first > width:
            out[first:last] = 0
            continue
        start = pool[slots[taken - 1]].double()

        def visit(t, row, o, magnitude, state):
            o_bound, state_bound = _bounds(t + 1, magnitude, state)
            out[row], out_bound[row] = _finish(o, o_bound, None if gate is None else gate[row],
                                               weight, eps)
            if live(slots[t]):
                new_pool[slots[t]], pool_bound[slots[t]] = state[0], state_bound

        _recur(qkv, log_decay, heads, v_heads, range(first, last),
               torch.stack([start, start.abs()]), scale, visit)
    return out, out_bound, new_pool, pool_bound


def expected_linear_prefill(qkv, log_decay, slots, has_initial, cu_seqlens, pool, gate, weight, out,
                            scale, eps):
    """(out, out bound, pool, pool bound) of a prefill; rows outside every sequence keep theirs."""
    heads, v_heads = geometry(qkv, pool)
    out, new_pool = out.double(), pool.double()
    out_bound, pool_bound = torch.zeros_like(out), torch.zeros_like(new_pool)
    for n, slot in enumerate(slots.tolist()):
        first, last = int(cu_seqlens[n]), int(cu_seqlens[n + 1])
        live = 0 < slot < pool.shape[0]
        start = pool[slot].double() if live and bool(has_initial[n]) else torch.zeros(
            pool.shape[1:], dtype=torch.float64, device=pool.device)

        def visit(t, row, o, magnitude, state):
            o_bound, _ = _bounds(t + 1, magnitude, state)
            out[row], out_bound[row] = _finish(o, o_bound, None if gate is None else gate[row],
                                               weight, eps)

        state = _recur(qkv, log_decay, heads, v_heads, range(first, last),
                       torch.stack([start, start.abs()]), scale, visit)
        if live:
            new_pool[slot] = state[0]
            pool_bound[slot] = _bounds(last - first, state[1], state)[1]
    return out, out_bound, new_pool, pool_bound


def exact_angles(positions, inv_freq):
    """positions x inv_freq.  From 2^29 on a product with an fp32 frequency has more than a double's
    53 bits: there by whole numbers, in units of 2^-320, less the whole turns."""
    if positions.numel() == 0 or -(2**29) < int(positions.min()) <= int(positions.max()) < 2**29:
        return positions.double()[:, None] * inv_freq.double()
    unit = 1 << 320

    def arctan(n):   # of 1 / n
        term = total = unit // n
        k = 1
        while term:
            term //= -n * n
            k += 2
            total += term // k
        return total

    turn = 8 * (4 * arctan(5) - arctan(239))
    angles = []
    for position in positions.tolist():
        for frequency in inv_freq.tolist():
            above, below = frequency.as_integer_ratio()
            angles.append(position * above * unit // below % turn / unit)
    return torch.tensor(angles, dtype=torch.float64, device=positions.device).view(
        len(positions), -1)


def expected_norm_rope(qkv, q_weight, k_weight, positions, inv_freq, q_heads, k_heads, eps,
                       interleaved):
    """(qkv, bound) of norm_rope.  The bound: half a bf16 step, and 2^-20 of the normalised pair
    (2^-23.3 for an angle that is an fp32 fraction of a turn, below 2^-22 each for its sine and
    cosine, and for the norm's root and the products)."""
    result = qkv.double()
    bound = torch.zeros_like(result)
    half = inv_freq.numel()
    angle = exact_angles(positions, inv_freq)
    cos, sin = angle.cos(), angle.sin()
    lower = torch.arange(half, device=qkv.device) * (2 if interleaved else 1)
    upper = lower + (1 if interleaved else half)
    for h in range(q_heads + k_heads):
        columns = slice(h * DIM, (h + 1) * DIM)
        x = qkv[:, columns].double()
        weight = (q_weight if h < q_heads else k_weight).double()
        y = x * (x.square().mean(-1, keepdim=True) + eps).rsqrt() * weight
        z = y.clone()
        z[:, lower] = y[:, lower] * cos - y[:, upper] * sin
        z[:, upper] = y[:, upper] * cos + y[:, lower] * sin
        size = y.abs()
        pair = size[:, lower] + size[:, upper]
        size[:, lower] = pair
        size[:, upper] = pair
        result[:, columns] = z
        bound[:, columns] = z.abs() * 2.0**-8 + size * 2.0**-20 + 1e-30
    return result, bound
