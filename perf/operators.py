"""The serving operators around the paged KV cache, as they are measured.

Four operators that a serving step runs one after the other: the slot mapping
of a batch from its request lengths, the per-head norm and rotation of queries
and keys, the paged cache held in 4 bits (stored to and loaded from), and
attention over that cache.

``run`` computes a case in plain torch operations when ``own`` is false, and
calls the framework's operators when it is true.
"""

import os
import sys

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32,
          "int64": torch.int64, "int32": torch.int32}
FP16_MAX = 65504.0


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # One decode step of a small batch: every request adds one token. Latency.
        dict(name="slots_decode_8", op="slots", batch=8, ctx_max=4096, new_max=1,
             prefill_share=1.0, block=16, slot_dtype="int64", pad=0, layout=1),
        # A long-prompt batch: every request of a large queue brings its prompt.
        dict(name="slots_prompts_1021", op="slots", batch=1021, ctx_max=2048, new_max=1500,
             prefill_share=1.0, block=16, slot_dtype="int64", pad=37, layout=2),
        # One token of a 32 + 8 head model: the smallest decode step.
        dict(name="qk_one_token", op="qk", tokens=1, q_heads=32, k_heads=8, head=128, rot=128,
             neox=True, dtype="bf16", packed=True, layout=3),
        # A decode batch, adjacent pairs and partly rotated heads, an odd token count.
        dict(name="qk_decode_259", op="qk", tokens=259, q_heads=64, k_heads=8, head=128, rot=64,
             neox=False, dtype="fp16", packed=False, layout=4),
        # A prefill batch of the 64 + 8 head model, q and k views of one packed projection.
        dict(name="qk_prefill_16k", op="qk", tokens=16384, q_heads=64, k_heads=8, head=128,
             rot=128, neox=True, dtype="bf16", packed=True, layout=5),
        # A decode batch's new rows into the 4-bit cache and back.
        dict(name="kv4_rows_96", op="kv4", tokens=96, heads=8, head=128, block=16, dtype="bf16",
             skipped=3, layout=6),
        # A prefill batch's rows into the 4-bit cache and back, with skipped slots.
        dict(name="kv4_rows_40k", op="kv4", tokens=40001, heads=8, head=128, block=16,
             dtype="bf16", skipped=500, layout=7),
        # One long request on a tensor-parallel shard with one KV head: latency, split over the cache.
        dict(name="attn_one_16k", op="attn", batch=1, query=1, ctx_min=16001, ctx_max=16001,
             kv_heads=1, group=8, head=128, block=16, dtype="bf16", window=0, sinks=0, pad=0,
             layout=8),
        # A decode batch of ragged contexts over 8 KV heads.
        dict(name="attn_decode_96", op="attn", batch=96, query=1, ctx_min=1, ctx_max=16384,
             kv_heads=8, group=4, head=128, block=16, dtype="bf16", window=0, sinks=0, pad=0,
             layout=9),
        # A decode batch with a sliding window and four first tokens, rows of padding behind it.
        dict(name="attn_window_61", op="attn", batch=61, query=1, ctx_min=1, ctx_max=32768,
             kv_heads=8, group=8, head=64, block=32, dtype="fp16", window=1024, sinks=4, pad=3,
             layout=10),
        # Suffixes computed over retrieved prefixes (prefix reuse), ragged.
        dict(name="attn_suffix_4", op="attn", batch=4, query=1024, ctx_min=4096, ctx_max=16384,
             kv_heads=8, group=8, head=128, block=16, dtype="bf16", window=0, sinks=0, pad=0,
             layout=11),
        # The same with a window, where most of the prefix is out of sight.
        dict(name="attn_suffix_window", op="attn", batch=3, query=2000, ctx_min=2000,
             ctx_max=20000, kv_heads=4, group=4, head=128, block=64, dtype="fp16", window=2048,
             sinks=16, pad=5, layout=12),
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    v = int(round(float(np.exp(rng.uniform(np.log(lo), np.log(hi))))))
    return max(lo, min(hi, v))


def _cost(case):
    w = work(case)
    return w["bytes"] / 6.5e12 + w["flops"] / 1.6e15


def draw(rng):
    op = rng.choice(["slots", "qk", "kv4", "attn", "attn"])
    layout = rng.randrange(1 << 30)
    if op == "slots":
        case = dict(op=op, batch=_log(rng, 1, 1021), ctx_max=_log(rng, 1, 32768),
                    new_max=_log(rng, 1, 1500), prefill_share=rng.choice([0.0, 0.2, 1.0]),
                    block=rng.choice([8, 16, 32, 64, 128]),
                    slot_dtype=rng.choice(["int64", "int64", "int32"]),
                    pad=rng.choice([0, rng.randrange(1, 200)]), layout=layout)
        shrink = "batch"
    elif op == "qk":
        k_heads = rng.choice([1, 2, 4, 5, 8])
        head = rng.choice([64, 80, 128, 128, 256])
        case = dict(op=op, tokens=_log(rng, 1, 16384), q_heads=k_heads * rng.choice([1, 4, 7, 8]),
                    k_heads=k_heads, head=head, rot=rng.choice([head, head // 2]),
                    neox=rng.random() < 0.6, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                    packed=rng.random() < 0.5, layout=layout)
        shrink = "tokens"
    elif op == "kv4":
        tokens = _log(rng, 1, 40001)
        case = dict(op=op, tokens=tokens, heads=rng.choice([1, 2, 4, 5, 8, 16]),
                    head=rng.choice([64, 128, 128, 256]), block=rng.choice([8, 16, 32, 64]),
                    dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                    skipped=rng.choice([0, tokens // 7]), layout=layout)
        shrink = "tokens"
    else:
        query = rng.choice([1, 1, rng.randrange(2, 9), _log(rng, 9, 2000)])
        ctx_max = _log(rng, query, 32768)
        case = dict(op=op, batch=_log(rng, 1, 96), query=query,
                    ctx_min=rng.choice([query, ctx_max]), ctx_max=ctx_max,
                    kv_heads=rng.choice([1, 2, 3, 4, 8]), group=rng.choice([1, 2, 4, 5, 7, 8, 16]),
                    head=rng.choice([64, 128, 128, 256]), block=rng.choice([8, 16, 24, 32, 64]),
                    dtype=rng.choice(["bf16", "fp16"]),
                    window=rng.choice([0, 0, _log(rng, 1, 4096)]),
                    sinks=rng.choice([0, 4, 16]), pad=rng.choice([0, rng.randrange(1, 9)]),
                    layout=layout)
        shrink = "batch"
    largest = max(_cost(c) for c in listed() if c["op"] == op)
    while _cost(case) > largest:
        if case[shrink] > 1:
            case[shrink] = max(1, case[shrink] * 3 // 4)
        else:
            case["query"] = max(1, case["query"] // 2)
    if op == "kv4":
        case["skipped"] = min(case["skipped"], case["tokens"] // 7)
    return case


# ---------------------------------------------------------------------------
# What a case's layout is: lengths, which the host program knows
# ---------------------------------------------------------------------------

def _slot_lens(case):
    rs = np.random.RandomState(case["layout"])
    b = case["batch"]
    new = rs.randint(1, case["new_max"] + 1, b)
    ctx = rs.randint(0, case["ctx_max"] + 1, b)
    # requests that are not prefilling decode one token
    new = np.where(rs.rand(b) < case["prefill_share"], new, 1)
    return ctx, new


def _attn_lens(case):
    rs = np.random.RandomState(case["layout"])
    b, q = case["batch"], case["query"]
    qlens = np.ones(b, np.int64) if q == 1 else rs.randint(max(1, q // 2), q + 1, b)
    lens = rs.randint(case["ctx_min"], case["ctx_max"] + 1, b)
    return qlens, np.maximum(lens, qlens)


def _row_words(heads, head):
    """int32 words of one token's K (or V) row in the 4-bit cache: heads x
    head / 8 words of codes, heads words of (scale, zero), padded to 16 bytes."""
    return (heads * (head // 8 + 1) + 3) // 4 * 4


def _visible(case):
    """(pairs, keys): visible (query, key) pairs of one head over the batch, and keys read."""
    pairs = keys = 0
    w, s = case["window"], case["sinks"]
    for n, length in zip(*_attn_lens(case)):
        p = np.arange(length - n, length, dtype=np.int64)
        if w == 0:
            pairs += int((p + 1).sum())
            keys += int(length)
        else:
            lo = np.maximum(0, p - w + 1)
            pairs += int((p + 1 - lo + np.minimum(lo, s)).sum())
            first = int(lo[0])
            keys += int(length) - first + min(first, s)
    return pairs, keys


def work(case):
    if case["op"] == "slots":
        ctx, new = _slot_lens(case)
        bs, isz = case["block"], 8 if case["slot_dtype"] == "int64" else 4
        need = (ctx + new + bs - 1) // bs - (ctx + bs - 1) // bs
        tokens = int(new.sum()) + case["pad"]
        # lengths and the partly filled pages' table entries in, free pages in, table entries,
        # slots, positions, starts and lengths out
        return {"bytes": int(case["batch"] * (8 + 4 + 8) + need.sum() * 8 + tokens * 2 * isz),
                "flops": 0}
    if case["op"] == "qk":
        esz = 4 if case["dtype"] == "fp32" else 2
        rows = case["tokens"] * (case["q_heads"] + case["k_heads"])
        return {"bytes": rows * case["head"] * 2 * esz + case["tokens"] * (case["rot"] * 4 + 8),
                "flops": rows * case["head"] * 7}
    if case["op"] == "kv4":
        esz = 4 if case["dtype"] == "fp32" else 2
        rows = (case["tokens"] - case["skipped"]) * case["heads"] * 2
        # 16/32-bit rows in, 4-bit rows out and in again, 16/32-bit rows out
        return {"bytes": rows * 2 * (case["head"] * esz + case["head"] // 2 + 4)
                + case["tokens"] * 16,
                "flops": rows * case["head"] * 6}
    pairs, keys = _visible(case)
    qlens, _ = _attn_lens(case)
    q_rows = int(qlens.sum()) * case["kv_heads"] * case["group"]
    return {"bytes": keys * case["kv_heads"] * (case["head"] + 8) + q_rows * case["head"] * 4
            + keys // case["block"] * 4,
            "flops": 4 * pairs * case["kv_heads"] * case["group"] * case["head"]}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def _quantise(x):
    """(codes, scale, zero) of head rows x [..., D]: a row's minimum and a
    fifteenth of its span, both rounded to 16 bits, and the nearest code, ties
    to even. NaN counts as 0; values beyond the 16-bit range as its ends."""
    x = torch.nan_to_num(x.float(), nan=0.0, posinf=FP16_MAX, neginf=-FP16_MAX)
    x = x.clamp(-FP16_MAX, FP16_MAX)
    lo, hi = x.amin(-1), x.amax(-1)
    scale = ((hi - lo) / 15.0).half().float()
    zero = lo.half().float()
    # in 64 bits: a quotient next to a border falls to the right side of it
    q = (x.double() - zero.double()[..., None]) / scale.double()[..., None]
    q = torch.where(scale[..., None] > 0, q, torch.zeros_like(q))
    return q.round().clamp(0, 15).to(torch.int64), scale, zero


def _pack(codes, scale, zero):
    """int32 words [T, W] of codes [T, H, D], scale and zero [T, H]."""
    t, h, d = codes.shape
    shifts = torch.arange(8, device=codes.device) * 4
    words = (codes.view(t, h * d // 8, 8) << shifts).sum(-1)
    s = scale.half().view(torch.int16).long() & 0xFFFF
    z = zero.half().view(torch.int16).long() & 0xFFFF
    row = torch.zeros(t, _row_words(h, d), dtype=torch.int64, device=codes.device)
    row[:, : h * d // 8] = words
    row[:, h * d // 8 : h * d // 8 + h] = s | (z << 16)
    return torch.where(row >= 1 << 31, row - (1 << 32), row).int()


def _unpack(rows, heads, head, dtype=torch.float32):
    """Values [T, H, D] of int32 rows [T, W]."""
    t = rows.shape[0]
    n = heads * head // 8
    shifts = torch.arange(8, device=rows.device, dtype=torch.int32) * 4
    codes = ((rows[:, :n, None] >> shifts) & 15).view(t, heads, head)
    par = rows[:, n : n + heads].contiguous().view(torch.float16).view(t, heads, 2).to(dtype)
    return codes.to(dtype) * par[..., 0:1] + par[..., 1:2]


def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, shape, dtype):
    return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32).to(dtype)


def prepare(case, seed):
    g = _generator(seed)
    state = {"case": case}
    if case["op"] == "slots":
        ctx, new = _slot_lens(case)
        bs, b = case["block"], case["batch"]
        has = (ctx + bs - 1) // bs
        total = (ctx + new + bs - 1) // bs
        cols = int(total.max()) + 2
        pages = torch.randperm(int(total.sum()) + 17, generator=g, device=DEV).int()
        col = torch.arange(cols, device=DEV)[None]
        has_t = torch.from_numpy(has).to(DEV)
        first = has_t.cumsum(0) - has_t
        held = pages[(first[:, None] + col).clamp(max=pages.numel() - 1)]
        table = torch.where(col < has_t[:, None], held, torch.full_like(held, -1))
        n = int(new.sum()) + case["pad"]
        dt = DTYPES[case["slot_dtype"]]
        state.update(
            ctx=torch.from_numpy(ctx).int().to(DEV), new=torch.from_numpy(new).int().to(DEV),
            table=table.contiguous(), free=pages[int(has.sum()):].contiguous(), block=bs,
            slots=torch.empty(n, dtype=dt, device=DEV),
            positions=torch.empty(n, dtype=dt, device=DEV),
            starts=torch.empty(b + 1, dtype=torch.int32, device=DEV),
            lens=torch.empty(b, dtype=torch.int32, device=DEV),
            used=torch.empty(1, dtype=torch.int32, device=DEV))
        return state
    if case["op"] == "qk":
        t, hq, hk, d = case["tokens"], case["q_heads"], case["k_heads"], case["head"]
        dt = DTYPES[case["dtype"]]
        if case["packed"]:  # q and k as a fused projection leaves them: [q | k | v]
            qkv = _randn(g, (t, (hq + 2 * hk) * d), dt)
            q = qkv[:, : hq * d].view(t, hq, d)
            k = qkv[:, hq * d : (hq + hk) * d].view(t, hk, d)
        else:
            q, k = _randn(g, (t, hq, d), dt), _randn(g, (t, hk, d), dt)
        rot, limit = case["rot"], 40960
        inv = 1e6 ** (-torch.arange(0, rot, 2, device=DEV, dtype=torch.float64) / rot)
        ang = torch.arange(limit, device=DEV, dtype=torch.float64)[:, None] * inv
        state.update(
            q=q, k=k, qw=(1 + 0.1 * _randn(g, (d,), torch.float32)).to(dt),
            kw=(1 + 0.1 * _randn(g, (d,), torch.float32)).to(dt),
            positions=torch.randint(0, limit, (t,), generator=g, device=DEV),
            cos_sin=torch.cat([ang.cos(), ang.sin()], -1).float(), eps=1e-6,
            q_out=torch.empty(t, hq, d, dtype=dt, device=DEV),
            k_out=torch.empty(t, hk, d, dtype=dt, device=DEV))
        return state
    if case["op"] == "kv4":
        t, h, d, bs = case["tokens"], case["heads"], case["head"], case["block"]
        dt = DTYPES[case["dtype"]]
        blocks = (t + bs - 1) // bs + 5
        page = torch.randperm(blocks, generator=g, device=DEV)
        tok = torch.arange(t, device=DEV)
        slots = page[tok // bs] * bs + tok % bs
        slots[torch.randperm(t, generator=g, device=DEV)[: case["skipped"]]] = -1
        key = _randn(g, (t, h, d), torch.float32)
        key = key * (1 + 3 * torch.rand(h, d, generator=g, device=DEV))  # channels differ
        state.update(
            key=key.to(dt), value=_randn(g, (t, h, d), dt), slots=slots,
            cache=torch.zeros(2, blocks, bs, 1, _row_words(h, d), dtype=torch.int32, device=DEV),
            k_out=torch.zeros(t, h, d, dtype=dt, device=DEV),
            v_out=torch.zeros(t, h, d, dtype=dt, device=DEV))
        return state
    qlens, lens = _attn_lens(case)
    h, d, bs, b = case["kv_heads"], case["head"], case["block"], case["batch"]
    dt = DTYPES[case["dtype"]]
    pages = (lens + bs - 1) // bs
    blocks = int(pages.sum()) + 3
    perm = torch.randperm(blocks, generator=g, device=DEV).int()
    table = torch.full((b, int(pages.max()) + 1), -1, dtype=torch.int32, device=DEV)
    # pages and page ends that no token fills hold what memory held before: here NaN scales
    cache = torch.full((2, blocks, bs, 1, _row_words(h, d)), -1, dtype=torch.int32, device=DEV)
    flat = cache.view(2, blocks * bs, -1)
    at = 0
    for i in range(b):
        n = int(pages[i])
        table[i, :n] = perm[at : at + n]
        at += n
    channel = 1 + 2 * torch.rand(h, d, generator=g, device=DEV)
    for i in range(b):
        tok = torch.arange(int(lens[i]), device=DEV)
        slot = table[i].long()[tok // bs] * bs + tok % bs
        for half in range(2):
            x = _randn(g, (int(lens[i]), h, d), torch.float32)
            flat[half, slot] = _pack(*_quantise(x * channel if half == 0 else x))
    n = int(qlens.sum())
    starts = np.concatenate([[0], np.cumsum(qlens)])
    state.update(
        q=_randn(g, (n + case["pad"], h * case["group"], d), dt), cache=cache, table=table,
        lens=torch.from_numpy(lens).int().to(DEV),
        starts=None if case["query"] == 1 and case["pad"] == 0
        else torch.from_numpy(starts).int().to(DEV),
        host_lens=[int(v) for v in lens], host_starts=[int(v) for v in starts],
        max_query=int(qlens.max()), max_len=int(lens.max()), scale=float(d) ** -0.5,
        out=torch.zeros(n + case["pad"], h * case["group"], d, dtype=dt, device=DEV))
    return state


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------

def _c_ops():
    root = os.path.join(os.getcwd(), "lmcache-ascend_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from lmcache_b200 import c_ops

    return c_ops


def run(state):
    return (_run_own if own else _run_plain)[state["case"]["op"]](state)


def _own_slots(s):
    _c_ops().build_slot_mapping(s["ctx"], s["new"], s["table"], s["free"], s["block"], s["slots"],
                                s["positions"], s["starts"], s["lens"], s["used"])
    return s["table"], s["slots"], s["positions"], s["starts"], s["lens"], s["used"]


def _plain_slots(s):
    bs, table, free = s["block"], s["table"], s["free"]
    b, cols = table.shape
    ctx, new = s["ctx"].long(), s["new"].long()
    has = (ctx + bs - 1) // bs
    need = (ctx + new + bs - 1) // bs - has
    first = need.cumsum(0) - need
    j = torch.arange(cols, device=DEV)[None] - has[:, None]
    src = first[:, None] + j
    fresh = torch.where(src < free.numel(), free[src.clamp(0, free.numel() - 1)].long(), -1)
    table = torch.where((j >= 0) & (j < need[:, None]), fresh, table.long())
    ends = new.cumsum(0)
    tok = torch.arange(s["slots"].numel(), device=DEV)
    req = torch.searchsorted(ends, tok, right=True)
    real = req < b
    req = req.clamp(max=b - 1)
    pos = ctx[req] + tok - (ends - new)[req]
    page = table[req, (pos // bs).clamp(max=cols - 1)]
    slot = torch.where(real & (page >= 0), page * bs + pos % bs, -1)
    starts = torch.cat([torch.zeros_like(ends[:1]), ends])
    dt = s["slots"].dtype
    return (table.int(), slot.to(dt), torch.where(real, pos, 0).to(dt), starts.int(),
            (ctx + new).int(), need.sum().view(1).int())


def _own_qk(s):
    c = s["case"]
    _c_ops().qk_norm_rope(s["q"], s["k"], s["qw"], s["kw"], s["positions"], s["cos_sin"],
                          s["eps"], c["neox"], s["q_out"], s["k_out"])
    return s["q_out"], s["k_out"]


def _plain_qk(s):
    c = s["case"]
    rot = c["rot"]
    cs = s["cos_sin"][s["positions"]][:, None]
    cos, sin = cs[..., : rot // 2], cs[..., rot // 2 :]
    outs = []
    for x, w in ((s["q"], s["qw"]), (s["k"], s["kw"])):
        y = x.float()
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + s["eps"]) * w.float()
        if c["neox"]:
            a, b = y[..., : rot // 2], y[..., rot // 2 : rot]
            turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        else:
            a, b = y[..., :rot:2], y[..., 1:rot:2]
            turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        outs.append(torch.cat([turned, y[..., rot:]], -1).to(x.dtype))
    return tuple(outs)


def _own_kv4(s):
    ops = _c_ops()
    ops.kv4_store(s["key"], s["value"], s["cache"], s["slots"])
    ops.kv4_load(s["cache"], s["slots"], s["k_out"], s["v_out"])
    return s["k_out"], s["v_out"]


def _plain_kv4(s):
    h, d = s["key"].shape[1:]
    flat = s["cache"].view(2, -1, s["cache"].shape[-1])
    # skipped rows go to and come from a row behind the cache
    spare = torch.cat([flat, torch.zeros_like(flat[:, :1])], 1)
    slot = torch.where(s["slots"] >= 0, s["slots"], flat.shape[1])
    outs = []
    for half, (x, prior) in enumerate(((s["key"], s["k_out"]), (s["value"], s["v_out"]))):
        spare[half, slot] = _pack(*_quantise(x))
        flat[half] = spare[half, :-1]
        got = _unpack(spare[half, slot], h, d).to(x.dtype)
        outs.append(torch.where((s["slots"] >= 0)[:, None, None], got, prior))
    return tuple(outs)


def _own_attn(s):
    c = s["case"]
    _c_ops().kv4_attention(s["q"], s["cache"], s["table"], s["lens"], s["starts"], s["max_query"],
                           s["max_len"], c["kv_heads"], s["scale"], c["window"], c["sinks"],
                           s["out"])
    return s["out"]


def _plain_attn(s):
    c = s["case"]
    h, d, grp, bs = c["kv_heads"], c["head"], c["group"], c["block"]
    w, sinks = c["window"], c["sinks"]
    flat = s["cache"].view(2, -1, s["cache"].shape[-1])
    out = s["out"].clone()
    for i, length in enumerate(s["host_lens"]):
        a, e = s["host_starts"][i], s["host_starts"][i + 1]
        n = e - a
        keys = torch.arange(length, device=DEV)
        if w:
            lo = max(0, length - n - w + 1)
            keys = torch.cat([keys[: min(lo, sinks)], keys[lo:]])
        slot = s["table"][i].long()[keys // bs] * bs + keys % bs
        k = _unpack(flat[0, slot], h, d)
        v = _unpack(flat[1, slot], h, d)
        pos = torch.arange(length - n, length, device=DEV)[:, None]
        seen = keys[None] <= pos
        if w:
            seen = seen & ((keys[None] > pos - w) | (keys[None] < sinks))
        q = s["q"][a:e].float().view(n, h, grp, d) * s["scale"]
        res = torch.empty(n, h, grp, d, device=DEV)
        step = h if n == 1 else 1
        for j in range(0, h, step):
            m = slice(j, j + step)
            qj = q[:, m].permute(1, 0, 2, 3).reshape(step, n * grp, d)
            sc = qj @ k[:, m].permute(1, 2, 0)
            sc = sc.view(step, n, grp, -1).masked_fill(~seen[None, :, None], float("-inf"))
            sc = (sc - sc.amax(-1, keepdim=True)).exp()
            sc = sc / sc.sum(-1, keepdim=True)
            o = sc.view(step, n * grp, -1) @ v[:, m].transpose(0, 1)
            res[:, m] = o.view(step, n, grp, d).transpose(0, 1)
        out[a:e] = res.view(n, h * grp, d).to(out.dtype)
    return out


_run_own = {"slots": _own_slots, "qk": _own_qk, "kv4": _own_kv4, "attn": _own_attn}
_run_plain = {"slots": _plain_slots, "qk": _plain_qk, "kv4": _plain_kv4, "attn": _plain_attn}


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    return _exact[case["op"]](prepare(case, seed))


def _exact_slots(s):
    """Request by request, token by token, as a host allocator does it."""
    bs = s["block"]
    table, free = s["table"].cpu().numpy().copy(), s["free"].cpu().numpy()
    ctx, new = s["ctx"].cpu().numpy(), s["new"].cpu().numpy()
    slots = np.full(s["slots"].numel(), -1, np.int64)
    positions = np.zeros(s["slots"].numel(), np.int64)
    starts, at, used = [0], 0, 0
    for b in range(len(ctx)):
        for page in range(-(-int(ctx[b]) // bs), -(-int(ctx[b] + new[b]) // bs)):
            table[b, page] = free[used] if used < len(free) else -1
            used += 1
        pos = np.arange(ctx[b], ctx[b] + new[b], dtype=np.int64)
        page = table[b, pos // bs].astype(np.int64)
        slots[at : at + len(pos)] = np.where(page >= 0, page * bs + pos % bs, -1)
        positions[at : at + len(pos)] = pos
        at += len(pos)
        starts.append(at)
    dt = s["slots"].dtype
    return (torch.from_numpy(table).to(DEV), torch.from_numpy(slots).to(DEV, dt),
            torch.from_numpy(positions).to(DEV, dt),
            torch.tensor(starts, dtype=torch.int32, device=DEV),
            torch.from_numpy(ctx + new).int().to(DEV),
            torch.tensor([used], dtype=torch.int32, device=DEV))


def _exact_qk(s):
    c = s["case"]
    rot = c["rot"]
    outs = []
    for x, w in ((s["q"], s["qw"]), (s["k"], s["kw"])):
        y = x.double()
        y /= (y.square().mean(-1, keepdim=True) + s["eps"]).sqrt()
        y *= w.double()
        i = torch.arange(rot // 2, device=DEV)
        one, two = (i, i + rot // 2) if c["neox"] else (2 * i, 2 * i + 1)
        cos = s["cos_sin"][s["positions"], : rot // 2].double()[:, None]
        sin = s["cos_sin"][s["positions"], rot // 2 :].double()[:, None]
        z = y.clone()
        z[..., one] = y[..., one] * cos - y[..., two] * sin
        z[..., two] = y[..., one] * sin + y[..., two] * cos
        outs.append(z)
    return tuple(outs)


def _exact_kv4(s):
    outs = []
    for x, prior in ((s["key"], s["k_out"]), (s["value"], s["v_out"])):
        y = x.double()
        y = torch.where(y.isnan(), torch.zeros_like(y), y).clamp(-FP16_MAX, FP16_MAX)
        lo, hi = y.min(-1, keepdim=True)[0], y.max(-1, keepdim=True)[0]
        # the two numbers that a row keeps are 16-bit by definition
        step = ((hi - lo).float().double() / 15).float().half().double()
        base = lo.float().half().double()
        code = torch.where(step > 0, ((y - base) / step).round(), torch.zeros_like(y))
        z = base + step * code.clamp(0, 15)
        outs.append(torch.where((s["slots"] >= 0)[:, None, None], z, prior.double()))
    return tuple(outs)


def _exact_attn(s):
    c = s["case"]
    h, d, grp, bs = c["kv_heads"], c["head"], c["group"], c["block"]
    rows = s["cache"].view(2, -1, s["cache"].shape[-1])
    out = s["out"].double()
    for i, length in enumerate(s["host_lens"]):
        a, e = s["host_starts"][i], s["host_starts"][i + 1]
        j = torch.arange(length, device=DEV)
        slot = s["table"][i, j // bs].long() * bs + j % bs
        k = _unpack(rows[0, slot], h, d, torch.float64)
        v = _unpack(rows[1, slot], h, d, torch.float64)
        for t0 in range(a, e, 256):  # a few queries at a time
            t1 = min(e, t0 + 256)
            p = length - e + torch.arange(t0, t1, device=DEV)
            see = j[None] <= p[:, None]
            if c["window"]:
                see &= (j[None] > p[:, None] - c["window"]) | (j[None] < c["sinks"])
            for head in range(h * grp):
                logit = (s["q"][t0:t1, head].double() @ k[:, head // grp].T) * s["scale"]
                prob = torch.softmax(logit.masked_fill(~see, -torch.inf), -1)
                out[t0:t1, head] = prob @ v[:, head // grp]
    return out


_exact = {"slots": _exact_slots, "qk": _exact_qk, "kv4": _exact_kv4, "attn": _exact_attn}
