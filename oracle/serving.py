"""CPU restatement of the serving operators around the paged cache, in plain
loops and 64 bits: block tables and slot mappings from request lengths, the
per-head norm with rotation, the 4-bit cache rows and attention over them."""

from __future__ import annotations

import numpy as np
import torch

HALF_MAX = 65504.0


def build_slot_mapping(ctx, new, table, free, block_size, num_tokens):
    """(table, slots, positions, query_start, seq_lens, used) as a host
    allocator would make them, request by request."""
    table = np.array(table, dtype=np.int64)
    cols = table.shape[1]
    slots = np.full(num_tokens, -1, np.int64)
    positions = np.zeros(num_tokens, np.int64)
    starts, lens = [0], []
    used = at = 0
    for b in range(len(ctx)):
        c, n = max(0, int(ctx[b])), max(0, int(new[b]))
        for page in range(-(-c // block_size), min(cols, -(-(c + n) // block_size))):
            table[b, page] = free[used] if used < len(free) else -1
            used += 1
        for i in range(n):
            if at >= num_tokens:
                break
            pos = c + i
            page = table[b, pos // block_size] if pos // block_size < cols else -1
            slots[at] = page * block_size + pos % block_size if page >= 0 else -1
            positions[at] = pos
            at += 1
        starts.append(at)
        lens.append(c + n)
    return table, slots, positions, np.array(starts), np.array(lens), used


def qk_norm_rope(x, weight, positions, cache, eps, is_neox):
    """x [T, H, D] in float64: normed, weighted, rotated."""
    x = x.double()
    y = x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt()
    if weight is not None:
        y = y * weight.double()
    half = cache.shape[1] // 2
    cs = cache.double()[positions.long()]
    out = y.clone()
    for i in range(half):
        a, b = (i, i + half) if is_neox else (2 * i, 2 * i + 1)
        cos, sin = cs[:, None, i], cs[:, None, half + i]
        out[..., a] = y[..., a] * cos - y[..., b] * sin
        out[..., b] = y[..., b] * cos + y[..., a] * sin
    return out


def kv4_row_words(heads, head_size):
    return -(-heads * (head_size // 8 + 1) // 4) * 4


def kv4_quantise(x):
    """(codes, scale, zero) of x [..., D] as int64 and float64."""
    x = x.double()
    x = torch.where(x.isnan(), torch.zeros_like(x), x).clamp(-HALF_MAX, HALF_MAX)
    lo, hi = x.min(-1).values, x.max(-1).values
    span = (hi - lo).float()                       # fp32 difference and product,
    fifteenth = torch.tensor(1.0 / 15.0, dtype=torch.float32).double()
    scale = (span.double() * fifteenth).float().half().double()   # each rounded once
    zero = lo.float().half().double() + 0.0        # never -0
    q = (x - zero[..., None]) / torch.where(scale > 0, scale, torch.ones_like(scale))[..., None]
    codes = torch.where(scale[..., None] > 0, q.round().clamp(0, 15), torch.zeros_like(q))
    return codes.long(), scale, zero


def kv4_values(codes, scale, zero):
    return zero[..., None] + scale[..., None] * codes.double()


def kv4_words(codes, scale, zero):
    """The words a row occupies [T, H * D / 8 + H] (no padding), int32."""
    t, h, d = codes.shape
    words = (codes.reshape(t, h * d // 8, 8) << (4 * torch.arange(8))).sum(-1)
    s = scale.half().view(torch.int16).long() & 0xFFFF
    z = zero.half().view(torch.int16).long() & 0xFFFF
    row = torch.cat([words, s | (z << 16)], 1)
    return torch.where(row >= 1 << 31, row - (1 << 32), row).int()


def visible(pos, keys, window, sinks):
    seen = keys <= pos
    if window > 0:
        seen &= (keys > pos - window) | (keys < sinks)
    return seen


def kv4_attention(q, codes, params, scale, pos, window, sinks, num_kv_heads):
    """One request: q [n, Hq, D]; codes [2][len, H, D]; params [2] of (scale,
    zero) [len, H]; pos [n] query positions. Returns the output in float64 and
    a bound on what 16-bit operands and fp32 sums may add to it:
      products p s_v c are rounded to fp16 once (2^-11 of sum p s_v c);
      a logit is an fp32 sum of D exact products, taken in steps of 16, off by
      at most 2^-19 of its terms' absolute sum M, which moves the output by at
      most 4 of that times the largest |v|; exp2 and the fp32 sums over the keys
      add (n_keys / 16 + 8) 2^-22 of the largest |v|."""
    n, hq, d = q.shape
    group = hq // num_kv_heads
    out = torch.zeros(n, hq, d, dtype=torch.float64)
    slack = torch.zeros(n, hq, d, dtype=torch.float64)
    length = codes[0].shape[0]
    keys = torch.arange(length)
    k = kv4_values(codes[0], *params[0])
    v = kv4_values(codes[1], *params[1])
    kabs = params[0][0][..., None] * codes[0] + params[0][1].abs()[..., None]
    vspan = params[1][0][..., None] * codes[1]
    for i in range(n):
        seen = visible(int(pos[i]), keys, window, sinks)
        if not bool(seen.any()):
            continue
        for h in range(hq):
            kv = h // group
            row = q[i, h].double()
            logit = (k[seen, kv] @ row) * scale
            p = torch.softmax(logit, 0)
            out[i, h] = p @ v[seen, kv]
            mass = float((kabs[seen, kv] @ row.abs()).max()) * abs(scale)
            big = float(v[seen, kv].abs().max() + vspan[seen, kv].abs().max())
            steps = int(seen.sum()) / 16 + 8
            slack[i, h] = (2.0**-11 * (p @ vspan[seen, kv])
                           + big * (4 * mass * 2.0**-19 + steps * 2.0**-22))
    return out, slack
