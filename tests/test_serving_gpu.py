"""GPU tests of the serving operators around the paged cache against their
restatement in 64 bits (oracle/serving.py)."""

import random

import numpy as np
import pytest
import torch

from lmcache_b200 import abi, c_ops
from oracle import serving as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
FLAGS = abi


@pytest.fixture(autouse=True)
def clean_status():
    c_ops.device_status(0)
    yield
    c_ops.device_status(0)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


# ---------------------------------------------------------------------------
# build_slot_mapping
# ---------------------------------------------------------------------------

def run_slots(ctx, new, bs, cols, pad=0, nfree=None, lt=torch.int32, st=torch.int64, seed=0,
              col_pad=0, num_tokens=None):
    rs = np.random.RandomState(seed)
    ctx, new = np.asarray(ctx), np.asarray(new)
    b = len(ctx)
    pages = rs.permutation(b * cols + 100).astype(np.int64)
    table = np.full((b, cols), -7, np.int64)
    at = 0
    for i in range(b):
        has = min(cols, -(-max(0, int(ctx[i])) // bs))
        table[i, :has] = pages[at : at + has]
        at += has
    free = pages[at:] if nfree is None else pages[at : at + nfree]
    n = int(np.maximum(new, 0).sum()) + pad if num_tokens is None else num_tokens
    want = ref.build_slot_mapping(ctx, new, table, free, bs, n)
    wide = torch.full((b, cols + col_pad), -9, dtype=torch.int32, device=DEV)
    wide[:, :cols] = torch.from_numpy(table).int().to(DEV)
    t = wide[:, :cols]
    out = [torch.full((n,), 99, dtype=st, device=DEV), torch.full((n,), 99, dtype=st, device=DEV),
           torch.full((b + 1,), 99, dtype=torch.int32, device=DEV),
           torch.full((b,), 99, dtype=torch.int32, device=DEV),
           torch.full((1,), 99, dtype=torch.int32, device=DEV)]
    args = (torch.from_numpy(ctx).to(DEV, lt), torch.from_numpy(new).to(DEV, lt), t,
            torch.from_numpy(free).int().to(DEV), bs, *out)
    c_ops.build_slot_mapping(*args)
    got = [t] + out
    for g, w, name in zip(got, want, ("table", "slots", "positions", "starts", "lens", "used")):
        assert np.array_equal(g.cpu().numpy().astype(np.int64).reshape(-1),
                              np.asarray(w).reshape(-1)), name
    assert bool((wide[:, cols:] == -9).all())
    return args


@pytest.mark.parametrize("b", [1, 2, 31, 511, 512, 513, 1500])
@pytest.mark.parametrize("bs", [1, 16, 24, 128])
def test_slots_match(b, bs):
    rs = np.random.RandomState(b * 131 + bs)
    new_max, ctx_max = (60, 200) if bs > 1 else (9, 30)
    ctx, new = rs.randint(0, ctx_max, b), rs.randint(0, new_max, b)  # zero lengths among them
    cols = -(-(ctx_max + new_max) // bs) + 1
    run_slots(ctx, new, bs, cols, pad=int(rs.randint(0, 40)),
              lt=[torch.int32, torch.int64][b % 2], st=[torch.int64, torch.int32][bs % 3 % 2],
              col_pad=3)
    assert c_ops.device_status(0) == 0


def test_slots_page_ends_and_decode():
    # contexts that end on, before and behind a page's end; one new token each
    run_slots([0, 1, 15, 16, 17, 31, 32, 33], [1] * 8, 16, 4, pad=5)
    run_slots([0, 0, 0], [0, 0, 0], 16, 4, pad=3)  # nothing new
    run_slots([5], [0], 16, 4)                      # no token at all
    run_slots([0], [4097], 16, 300)                 # one long prompt
    assert c_ops.device_status(0) == 0


def test_slots_largest_batch():
    rs = np.random.RandomState(3)
    run_slots(rs.randint(0, 64, 16384), rs.randint(0, 5, 16384), 16, 6)
    assert c_ops.device_status(0) == 0


def test_slots_many_tokens():
    rs = np.random.RandomState(4)
    run_slots(rs.randint(0, 5000, 200), rs.randint(1, 1500, 200), 16, 420, pad=11)


@pytest.mark.parametrize("nfree", [0, 1, 7])
def test_slots_free_list_runs_out(nfree):
    run_slots([0, 20, 40, 3], [40, 30, 9, 100], 16, 9, nfree=nfree)
    assert c_ops.device_status(0) == FLAGS.LMCB_DEVICE_FLAG_PAGES_EXHAUSTED


def test_slots_table_row_ends():
    run_slots([0, 30, 70], [100, 100, 3], 16, 4)
    assert c_ops.device_status(0) == FLAGS.LMCB_DEVICE_FLAG_PAGES_EXHAUSTED


def test_slots_more_tokens_than_entries():
    args = None
    ctx, new = [3, 4, 5], [10, 20, 30]
    rs = np.random.RandomState(0)
    table = torch.from_numpy(rs.permutation(12).reshape(3, 4)).int().to(DEV)
    out = [torch.full((25,), 9, dtype=torch.int64, device=DEV) for _ in range(2)]
    starts = torch.empty(4, dtype=torch.int32, device=DEV)
    lens, used = torch.empty(3, dtype=torch.int32, device=DEV), torch.empty(
        1, dtype=torch.int32, device=DEV)
    dev = lambda a: torch.tensor(a, dtype=torch.int32, device=DEV)  # noqa: E731
    c_ops.build_slot_mapping(dev(ctx), dev(new), table, dev(list(range(50, 60))), 16, *out, starts,
                             lens, used)
    assert starts.tolist() == [0, 10, 25, 25]
    assert out[1].tolist() == list(range(3, 13)) + list(range(4, 19))
    assert c_ops.device_status(0) == FLAGS.LMCB_DEVICE_FLAG_LENGTH_OUT_OF_RANGE
    del args


def test_slots_negative_lengths_count_as_zero():
    run_slots([-5, 10, 3], [4, -2, 6], 16, 4)
    assert c_ops.device_status(0) == FLAGS.LMCB_DEVICE_FLAG_LENGTH_OUT_OF_RANGE


def test_slots_refuse_overlap_and_shapes():
    i32 = lambda n: torch.zeros(n, dtype=torch.int32, device=DEV)  # noqa: E731
    i64 = lambda n: torch.zeros(n, dtype=torch.int64, device=DEV)  # noqa: E731
    lens, new, table = i32(3), i32(3), i32(12).view(3, 4)
    ok = [lens, new, table, i32(5), 16, i64(8), i64(8), i32(4), i32(3), i32(1)]

    def bad(at, value, match):
        a = list(ok)
        a[at] = value
        with pytest.raises(RuntimeError, match=match):
            c_ops.build_slot_mapping(*a)

    c_ops.build_slot_mapping(*ok)
    bad(8, lens, "overlaps an input")      # lengths updated in place
    bad(6, ok[5], "outputs overlap")
    bad(3, table.view(-1), "overlaps an input")
    bad(1, i64(3), "same dtype")
    bad(0, i32(2), "contiguous vector of 3")
    bad(5, i32(8), "same dtype")
    bad(7, i32(3), "contiguous vector of 4")
    bad(5, torch.zeros(8, device=DEV), "int32 or int64")
    bad(2, table.t(), "dense rows")
    bad(4, 0, "block_size")
    bad(5, torch.zeros(8, dtype=torch.int64), "must be a CUDA tensor")


# ---------------------------------------------------------------------------
# qk_norm_rope
# ---------------------------------------------------------------------------

def cos_sin(limit, rot, dtype=torch.float32):
    inv = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / max(rot, 1))
    ang = torch.arange(limit, dtype=torch.float64)[:, None] * inv
    return torch.cat([ang.cos(), ang.sin()], -1).to(dtype)


def check_qk(got, x, w, pos, cache, eps, neox):
    """Half a step of the result's type; the fp32 arithmetic before it: a sum of
    D squares (D + 2 roundings at most, halved by the root), the root and
    three products (2^-22 together with rsqrt's 2 ulp), and the two products of
    a rotation, each 2^-24 of its own size."""
    want = ref.qk_norm_rope(x.cpu(), None if w is None else w.cpu(), pos.cpu(), cache.cpu(), eps,
                            neox)
    size = ref.qk_norm_rope(x.cpu(), None if w is None else w.cpu(), pos.cpu(),
                            torch.zeros_like(cache.cpu()), eps, neox)  # keeps the rest only
    plain = x.cpu().double()
    plain = plain / (plain.pow(2).mean(-1, keepdim=True) + eps).sqrt()
    if w is not None:
        plain = plain * w.cpu().double()
    d = x.shape[-1]
    rel = (d / 2 + 16) * 2.0**-24
    bound = half_step(got.dtype) * want.abs() + rel * 2 * plain.abs().amax(-1, keepdim=True)
    # fp16 subnormals: half a step of the smallest
    bound = bound + torch.finfo(got.dtype).smallest_normal * half_step(got.dtype) * 2
    err = (got.cpu().double() - want).abs()
    assert bool((err <= bound).all()), float((err - bound).max())
    del size


def qk_case(t, hq, hk, d, rot, neox, dtype, packed=False, offset=0, wdtype=None, cdtype=torch.float32,
            pdtype=torch.int64, weights=True, seed=0, in_place=False, limit=2048):
    g = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    if packed:
        qkv = rand(t, (hq + 2 * hk) * d + offset).to(dtype).to(DEV)
        q = qkv[:, offset : offset + hq * d].view(t, hq, d)
        k = qkv[:, offset + hq * d : offset + (hq + hk) * d].view(t, hk, d)
    else:
        q, k = rand(t, hq, d).to(dtype).to(DEV), rand(t, hk, d).to(dtype).to(DEV)
    wd = wdtype or dtype
    qw = (1 + 0.2 * rand(d)).to(wd).to(DEV) if weights else None
    kw = (1 + 0.2 * rand(d)).to(wd).to(DEV) if weights else None
    pos = torch.randint(0, limit, (t,), generator=g).to(pdtype).to(DEV)
    cache = cos_sin(limit, rot, cdtype).to(DEV)
    q0, k0 = q.clone(), k.clone()
    qo = q if in_place else torch.full((t, hq, d), 7.0, dtype=dtype, device=DEV)
    ko = k if in_place else torch.full((t, hk, d), 7.0, dtype=dtype, device=DEV)
    c_ops.qk_norm_rope(q, k, qw, kw, pos, cache, 1e-6, neox, qo, ko)
    check_qk(qo, q0, qw, pos, cache, 1e-6, neox)
    check_qk(ko, k0, kw, pos, cache, 1e-6, neox)
    if not in_place:
        assert torch.equal(q, q0) and torch.equal(k, k0)
    assert c_ops.device_status(0) == 0


@pytest.mark.parametrize("neox", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("d,rot", [(64, 64), (80, 80), (128, 128), (128, 64), (256, 256), (96, 32),
                                   (512, 128), (72, 72), (20, 12), (128, 0), (2, 2)])
def test_qk_matches(neox, dtype, d, rot):
    qk_case(37, 6, 2, d, rot, neox, dtype, seed=d + rot)


@pytest.mark.parametrize("t,hq,hk", [(1, 1, 1), (1, 32, 8), (3, 64, 8), (700, 28, 4), (5000, 8, 1),
                                     (2, 5, 0), (2, 0, 3), (0, 4, 4)])
def test_qk_shapes(t, hq, hk):
    qk_case(t, hq, hk, 128, 128, True, torch.bfloat16, seed=t)
    qk_case(t, hq, hk, 64, 64, False, torch.float16, seed=t)


@pytest.mark.parametrize("offset", [0, 1, 8])
@pytest.mark.parametrize("in_place", [False, True])
def test_qk_packed_and_in_place(offset, in_place):
    for dtype in (torch.bfloat16, torch.float32):
        for neox in (True, False):
            qk_case(65, 8, 2, 128, 128, neox, dtype, packed=True, offset=offset, in_place=in_place,
                    seed=offset)


@pytest.mark.parametrize("neox", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_qk_few_and_many_tokens(neox, dtype):
    """Few and many tokens, whole and partial rotation, packed and in place."""
    for t, hq, hk, d, rot in ((1, 3, 1, 128, 128), (700, 5, 2, 64, 32), (901, 4, 1, 80, 80),
                              (300, 2, 2, 256, 0), (1300, 12, 3, 128, 96), (40, 0, 2, 128, 128),
                              (650, 2, 0, 64, 64), (7, 40, 8, 512, 512)):
        qk_case(t, hq, hk, d, rot, neox, dtype, seed=t)
        qk_case(t, hq, hk, d, rot, neox, dtype, packed=True, in_place=True, offset=8, seed=t,
                wdtype=torch.float32, cdtype=torch.bfloat16, pdtype=torch.int32)


def test_qk_many_bad_positions():
    t = 1000
    cache = cos_sin(64, 128).to(DEV)
    q = torch.randn(t, 3, 128, device=DEV).bfloat16()
    k = torch.randn(t, 2, 128, device=DEV).bfloat16()
    pos = torch.randint(0, 64, (t,), device=DEV)
    bad = torch.randperm(t, device=DEV)[:300]
    pos[bad] = torch.where(bad % 2 == 0, -1, 1 << 40)
    qo, ko = torch.full_like(q, 3), torch.full_like(k, 3)
    c_ops.qk_norm_rope(q, k, None, None, pos, cache, 1e-6, True, qo, ko)
    assert c_ops.device_status(0) == FLAGS.LMCB_DEVICE_FLAG_POSITION_OUT_OF_RANGE
    good = torch.ones(t, dtype=torch.bool, device=DEV)
    good[bad] = False
    assert bool((qo[~good] == 3).all()) and bool((ko[~good] == 3).all())
    check_qk(qo[good], q[good], None, pos[good], cache, 1e-6, True)
    check_qk(ko[good], k[good], None, pos[good], cache, 1e-6, True)


@pytest.mark.parametrize("wdtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cdtype", [torch.float32, torch.bfloat16, torch.float16])
def test_qk_weight_cache_and_position_types(wdtype, cdtype):
    for dtype in (torch.bfloat16, torch.float32):
        for d in (128, 72):
            qk_case(19, 4, 2, d, d, True, dtype, wdtype=wdtype, cdtype=cdtype, pdtype=torch.int32)
            qk_case(19, 4, 2, d, d, False, dtype, wdtype=wdtype, cdtype=cdtype)
    qk_case(19, 4, 2, 128, 128, True, torch.bfloat16, weights=False)


def test_qk_zero_row_and_bad_positions():
    cache = cos_sin(64, 64).to(DEV)
    for d in (64, 72):  # the vector and the element kernel
        q = torch.randn(5, 3, d, device=DEV, dtype=torch.bfloat16)
        k = torch.randn(5, 2, d, device=DEV, dtype=torch.bfloat16)
        q[1] = 0
        pos = torch.tensor([0, 5, -1, 64, 63], device=DEV)
        qo, ko = torch.full_like(q, 3), torch.full_like(k, 3)
        c_ops.qk_norm_rope(q, k, None, None, pos, cache, 1e-6, True, qo, ko)
        assert c_ops.device_status(0) == FLAGS.LMCB_DEVICE_FLAG_POSITION_OUT_OF_RANGE
        assert bool((qo[1] == 0).all())
        assert bool((qo[2:4] == 3).all()) and bool((ko[2:4] == 3).all())
        good = [0, 1, 4]
        check_qk(qo[good], q[good], None, pos[good], cache, 1e-6, True)
        check_qk(ko[good], k[good], None, pos[good], cache, 1e-6, True)


def test_qk_refusals():
    q, k = torch.zeros(4, 2, 64, device=DEV), torch.zeros(4, 1, 64, device=DEV)
    pos, cache = torch.zeros(4, dtype=torch.int64, device=DEV), cos_sin(8, 64).to(DEV)
    qo, ko, w = torch.empty_like(q), torch.empty_like(k), torch.ones(64, device=DEV)
    ok = [q, k, w, w, pos, cache, 1e-6, True, qo, ko]
    c_ops.qk_norm_rope(*ok)

    def bad(at, value, match):
        a = list(ok)
        a[at] = value
        with pytest.raises(RuntimeError, match=match):
            c_ops.qk_norm_rope(*a)

    bad(0, q.view(4, 128), "must be .num_tokens, heads, head_size")
    bad(1, k.half(), "same dtype")
    bad(1, k[:3], "same tokens")
    bad(2, torch.ones(63, device=DEV), "head_size entries")
    bad(3, torch.ones(64), "must be a CUDA tensor")
    bad(4, pos[:3], "contiguous vector of 4")
    bad(5, cache[:, :63].contiguous(), "invalid shape")
    bad(5, cos_sin(8, 66).to(DEV), "invalid shape")
    bad(8, torch.empty(4, 3, 64, device=DEV), "shapes")
    bad(8, q.view(-1).roll(0)[: q.numel()].view_as(q) if False else k.expand(4, 2, 64), "dense")
    both = torch.zeros(5, 2, 64, device=DEV)
    a = list(ok)
    a[0], a[8] = both[:4], both[1:]
    with pytest.raises(RuntimeError, match="query_out must be query or overlap no input"):
        c_ops.qk_norm_rope(*a)
    a = list(ok)
    a[9] = qo[:, :1]
    with pytest.raises(RuntimeError, match="overlap"):
        c_ops.qk_norm_rope(*a)
    for queries, keys in ((q, q), (both[:4], both[1:])):  # in place over each other
        a = list(ok)
        a[0] = a[8] = queries
        a[1] = a[9] = keys
        with pytest.raises(RuntimeError, match="overlap"):
            c_ops.qk_norm_rope(*a)
    # parts of one packed output are no overlap
    packed = torch.zeros(4, 3 * 64, device=DEV)
    a = list(ok)
    a[8], a[9] = packed[:, :128].view(4, 2, 64), packed[:, 128:].view(4, 1, 64)
    c_ops.qk_norm_rope(*a)
    assert torch.equal(a[8], qo) and torch.equal(a[9], ko)


# ---------------------------------------------------------------------------
# kv4_store, kv4_load
# ---------------------------------------------------------------------------

def new_cache(blocks, bs, heads, d, fill=-1):
    return torch.full((2, blocks, bs, 1, ref.kv4_row_words(heads, d)), fill, dtype=torch.int32,
                      device=DEV)


def check_rows(cache, slots, x, half):
    """The stored words are exactly the oracle's."""
    h, d = x.shape[1:]
    want = ref.kv4_words(*ref.kv4_quantise(x.cpu()))
    flat = cache[half].reshape(-1, cache.shape[-1]).cpu()
    keep = slots.cpu() >= 0
    got = flat[slots.cpu()[keep].long(), : h * d // 8 + h]
    assert torch.equal(got, want[keep])


def store_case(t, heads, d, bs, dtype, x=None, stride_pad=0, st=torch.int64, seed=0, base=0):
    g = torch.Generator().manual_seed(seed)
    blocks = -(-t // bs) + 2
    page = torch.randperm(blocks * bs, generator=g)[:t].to(st)
    if t > 3:
        page[torch.randperm(t, generator=g)[: t // 5]] = -1
    slots = page.to(DEV)
    pair = []
    for i in range(2):
        rows = torch.randn(t, heads * d + stride_pad + base, generator=g).to(dtype)
        v = rows.to(DEV)[:, base : base + heads * d].view(t, heads, d)
        if x is not None:
            v.copy_(x[i] if isinstance(x, (list, tuple)) else x)
        pair.append(v)
    cache = new_cache(blocks, bs, heads, d)
    c_ops.kv4_store(pair[0], pair[1], cache, slots)
    for half in range(2):
        check_rows(cache, slots, pair[half], half)
    # rows without a slot, and the padding of every row, are left as they were
    flat = cache.view(2, blocks * bs, -1)
    used = heads * d // 8 + heads
    assert bool((flat[..., used:] == -1).all())
    free = torch.ones(blocks * bs, dtype=torch.bool, device=DEV)
    free[slots[slots >= 0].long()] = False
    assert bool((flat[:, free] == -1).all())
    # and read back
    outs = [torch.full((t, heads * d + stride_pad + base), 5.0, dtype=dtype, device=DEV)
            for _ in range(2)]
    views = [o[:, base : base + heads * d].view(t, heads, d) for o in outs]
    c_ops.kv4_load(cache, slots, *views)
    keep = (slots >= 0).cpu()
    for v, o, src in zip(views, outs, pair):
        codes, scale, zero = ref.kv4_quantise(src.cpu())
        # 15-bit products and one fp32 sum: the fp32 value is the exact one
        # rounded once, as for the output's own type after it
        want = (codes.float() * scale.float()[..., None] + zero.float()[..., None]).to(dtype)
        assert torch.equal(v.cpu()[keep], want[keep])
        assert bool((v.cpu()[~keep] == 5).all())
        assert bool((o[:, :base] == 5).all()) and bool((o[:, base + heads * d :] == 5).all())
    assert c_ops.device_status(0) == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("d", [8, 64, 72, 128, 136, 256])
@pytest.mark.parametrize("heads", [1, 3, 8])
def test_kv4_rows(dtype, d, heads):
    store_case(53, heads, d, 16, dtype, seed=d + heads)


@pytest.mark.parametrize("t", [1, 2, 255, 4099])
def test_kv4_row_counts(t):
    store_case(t, 8, 128, 16, torch.bfloat16, st=torch.int32, seed=t)
    store_case(t, 1, 64, 24, torch.float16, seed=t)


@pytest.mark.parametrize("pad,base", [(1, 0), (8, 0), (0, 1), (0, 8)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_kv4_strides(pad, base, dtype):
    store_case(40, 4, 128, 16, dtype, stride_pad=pad, base=base)


def special_rows(d, dtype):
    """Rows where a code or a parameter can go wrong."""
    g = torch.Generator().manual_seed(5)
    big = torch.finfo(dtype).max
    rows = [torch.zeros(d), torch.full((d,), 3.25), torch.full((d,), -1e-7),
            torch.randn(d, generator=g) * 1e-6, torch.randn(d, generator=g) * 1e-8,
            torch.randn(d, generator=g) * 1e4, 1000 + torch.randn(d, generator=g) * 0.01,
            torch.linspace(-65504, 65504, d), torch.linspace(0, 15, d)]
    steps = torch.arange(d) % 31  # quotients of exactly k and k + 1/2
    for s in (1.0, 0.25, 0.3, 1.7e-5):
        rows.append(steps * 0.5 * s)
        rows.append(steps * 0.5 * s - 7.5 * s)
    r = torch.randn(d, generator=g)
    r[0], r[1], r[2 % d] = float("nan"), float("inf"), -float("inf")
    rows.append(r)
    rows.append(torch.full((d,), float("nan")))
    r = torch.randn(d, generator=g)
    r[d // 2] = big
    rows.append(r)
    return torch.stack(rows).to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_kv4_special_rows(dtype, d):
    rows = special_rows(d, dtype)
    store_case(rows.shape[0], 1, d, 16, dtype, x=rows[:, None].to(DEV))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_kv4_codes_near_borders(dtype):
    """Values a few fp32 steps around every border between two codes."""
    d = 128
    g = torch.Generator().manual_seed(9)
    rows = []
    for _ in range(64):
        lo = torch.randn(1, generator=g).half().float()
        scale = (torch.rand(1, generator=g) * 0.5 + 0.01).half().float()
        border = lo + (torch.arange(d) % 15 + 0.5) * scale
        off = torch.randint(-3, 4, (d,), generator=g).float() * 2.0**-23
        r = border * (1 + off)
        r[0], r[1] = lo, lo + 15 * scale
        rows.append(r)
    x = torch.stack(rows).to(dtype)
    store_case(64, 1, d, 16, dtype, x=x[:, None].to(DEV))


@pytest.mark.parametrize("base", [1.0, 1.0003, -3.0007, 100.03, 30000.7])
def test_kv4_narrow_rows(base):
    """fp32 rows that are narrow against their offset: the zero's rounding and
    the quotient's are many steps, and quotients are far beyond 15."""
    d = 128
    g = torch.Generator().manual_seed(13)
    widths = 2.0 ** torch.arange(-24, 2).float()
    rows = torch.rand(len(widths), 3, d, generator=g, dtype=torch.float64)
    x = (base + widths.double()[:, None, None] * rows).float()
    store_case(len(widths), 3, d, 16, torch.float32, x=x.to(DEV))


def test_kv4_out_of_range_slots_and_refusals():
    cache = new_cache(2, 16, 2, 64)
    x = torch.randn(4, 2, 64, device=DEV)
    slots = torch.tensor([3, 32, 1 << 40, -5], device=DEV)
    c_ops.kv4_store(x, x, cache, slots)
    assert c_ops.device_status(0) == FLAGS.LMCB_DEVICE_FLAG_SLOT_OUT_OF_RANGE
    flat = cache.view(2, 32, -1)
    assert bool((flat[:, [i for i in range(32) if i != 3]] == -1).all())
    out = torch.full_like(x, 9)
    c_ops.kv4_load(cache, slots, out, out.clone())
    assert c_ops.device_status(0) == FLAGS.LMCB_DEVICE_FLAG_SLOT_OUT_OF_RANGE
    assert bool((out[1:] == 9).all()) and not bool((out[0] == 9).any())

    def bad(match, key=x, value=x, cache_=cache, slots_=slots):
        for fn in ("kv4_store", "kv4_load"):
            with pytest.raises(RuntimeError, match=match):
                if fn == "kv4_store":
                    c_ops.kv4_store(key, value, cache_, slots_)
                else:
                    c_ops.kv4_load(cache_, slots_, key, value)

    bad("same shape", value=x[:3])
    bad("same shape", value=x.half())
    bad("row", cache_=new_cache(2, 16, 1, 64))
    bad("int32", cache_=cache.long())
    bad("contiguous", cache_=cache[:, :, ::2])
    bad("head_size", key=torch.zeros(4, 2, 60, device=DEV), value=torch.zeros(4, 2, 60, device=DEV))
    bad("contiguous vector", slots_=slots[:3])
    bad("int32 or int64", slots_=slots.float())
    bad("must be a CUDA", slots_=slots.cpu())
    bad("dense", key=x.transpose(0, 1), value=x.transpose(0, 1))
    bad("overlaps kv_cache", value=cache.view(-1)[:512].view(torch.float32).view(4, 2, 64))
    with pytest.raises(RuntimeError, match="overlap"):
        c_ops.kv4_load(cache, slots, out, out)
    packed = torch.full((4, 4 * 64), 9.0, device=DEV)  # key and value side by side
    c_ops.kv4_load(cache, slots, packed[:, :128].view(4, 2, 64), packed[:, 128:].view(4, 2, 64))
    assert torch.equal(packed[0, :128].view(2, 64), packed[0, 128:].view(2, 64))
    assert bool((packed[1:] == 9).all())
    c_ops.kv4_store(x[:0], x[:0], cache, slots[:0])


# ---------------------------------------------------------------------------
# kv4_attention
# ---------------------------------------------------------------------------

class Batch:
    """A filled 4-bit cache and the queries of a batch."""

    def __init__(self, lens, qlens, hkv, group, d, bs, dtype, seed=0, pad=0, std=1.0, extra_cols=1,
                 shift=0.0):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.qlens = list(lens), list(qlens)
        self.hkv, self.group, self.d, self.bs, self.dtype = hkv, group, d, bs, dtype
        pages = [-(-max(0, n) // bs) for n in lens]
        blocks = sum(pages) + 2
        perm = torch.randperm(blocks, generator=g).int()
        cols = max(pages + [0]) + extra_cols
        self.table = torch.full((len(lens), cols), -1, dtype=torch.int32)
        self.cache = new_cache(blocks, bs, hkv, d)  # scales of unused rows are NaN
        self.codes, self.params = [], []
        at = 0
        for b, n in enumerate(lens):
            self.table[b, : pages[b]] = perm[at : at + pages[b]]
            at += pages[b]
            tok = torch.arange(max(0, n))
            slot = self.table[b].long()[tok // bs] * bs + tok % bs
            pair = [torch.randn(max(0, n), hkv, d, generator=g) * std + shift for _ in range(2)]
            quant = [ref.kv4_quantise(x) for x in pair]
            self.codes.append([q[0] for q in quant])
            self.params.append([q[1:] for q in quant])
            for half in range(2):
                words = ref.kv4_words(*quant[half])
                rows = self.cache[half].view(blocks * bs, -1)
                rows[slot.to(DEV), : words.shape[1]] = words.to(DEV)
        self.total = sum(qlens)
        self.q = (torch.randn(self.total + pad, hkv * group, d, generator=g) * 1.5).to(dtype).to(DEV)
        self.starts = torch.tensor([0] + list(np.cumsum(qlens)), dtype=torch.int32, device=DEV)
        self.lens_t = torch.tensor(lens, dtype=torch.int32, device=DEV)
        self.table = self.table.to(DEV)
        self.scale = d**-0.5

    def run(self, window=0, sinks=0, out=None, max_len=None, max_query=None, q=None, starts="auto"):
        q = self.q if q is None else q
        out = torch.full(q.shape, 3.0, dtype=q.dtype, device=DEV) if out is None else out
        if starts == "auto":
            starts = None if all(n == 1 for n in self.qlens) else self.starts
        c_ops.kv4_attention(q, self.cache, self.table, self.lens_t, starts,
                            max(self.qlens + [1]) if max_query is None else max_query,
                            max(self.lens + [1]) if max_len is None else max_len, self.hkv,
                            self.scale, window, sinks, out)
        return out

    def check(self, out, window=0, sinks=0, rows=None):
        at = 0
        for b, (n, length) in enumerate(zip(self.qlens, self.lens)):
            pick = range(n) if rows is None else sorted(set(r % n for r in rows)) if n else []
            pick = list(pick)
            if pick:
                q = self.q[at : at + n].cpu()[pick]
                pos = [length - n + i for i in pick]
                want, slack = ref.kv4_attention(q, self.codes[b], self.params[b], self.scale, pos,
                                                window, sinks, self.hkv)
                got = out[at : at + n].cpu().double()[pick]
                bound = half_step(self.dtype) * (want.abs() + slack) + slack + 2.0**-25
                err = (got - want).abs()
                assert bool((err <= bound).all()), (b, float((err / bound).max()))
            at += n
        assert bool((out[at:] == 3).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("hkv,group", [(1, 8), (2, 1), (8, 4), (3, 5), (4, 16), (5, 33), (16, 2)])
def test_attention_decode(dtype, d, hkv, group):
    b = Batch([1, 2, 15, 16, 17, 33, 0, 150], [1] * 8, hkv, group, d, 16, dtype, seed=d + group)
    b.check(b.run())
    assert c_ops.device_status(0) == 0


def test_attention_one_key_is_its_value():
    """A single visible key: the output is the stored value, rounded once."""
    for d in (64, 128, 256):
        b = Batch([1, 1, 1], [1] * 3, 2, 4, d, 16, torch.bfloat16, seed=d)
        out = b.run()
        slots = b.table[:, 0] * 16
        k = torch.empty(3, 2, d, dtype=torch.bfloat16, device=DEV)
        v = torch.empty_like(k)
        c_ops.kv4_load(b.cache, slots, k, v)
        assert torch.equal(out, v.repeat_interleave(4, 1))


@pytest.mark.parametrize("bs", [1, 3, 16, 24, 64, 256])
@pytest.mark.parametrize("lens", [[700], [3, 1000, 1, 0, 260], [513] * 7])
def test_attention_split_over_the_cache(bs, lens):
    b = Batch(lens, [1] * len(lens), 2, 4, 128, bs, torch.float16, seed=bs)
    b.check(b.run())
    b1 = Batch(lens, [1] * len(lens), 1, 8, 64, bs, torch.bfloat16, seed=bs)
    b1.check(b1.run())


def test_attention_long_and_skewed():
    b = Batch([20000, 5, 1, 300, 0, 77], [1] * 6, 1, 8, 128, 16, torch.bfloat16, seed=1)
    b.check(b.run())
    # the length hint sizes the launch only
    b.check(b.run(max_len=16))
    b.check(b.run(max_len=1 << 20))
    b.check(b.run(max_len=0))


@pytest.mark.parametrize("qlens,lens", [([3, 1, 2], [3, 40, 100]), ([8, 8], [300, 9]),
                                        ([5, 0, 7, 1], [70, 30, 7, 1]), ([17, 40], [17, 200]),
                                        ([130, 1, 64], [400, 50, 64])])
@pytest.mark.parametrize("hkv,group,d", [(2, 4, 128), (1, 7, 64), (8, 1, 128), (2, 3, 256)])
def test_attention_several_queries(qlens, lens, hkv, group, d):
    b = Batch(lens, qlens, hkv, group, d, 16, torch.bfloat16, seed=sum(lens), pad=3)
    b.check(b.run(), rows=[0, 1, 2, 7, 8, 9, 15, 16, 31, 63, 64, 100, -1, -2])
    assert c_ops.device_status(0) == 0


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 3), (7, 4), (16, 0), (33, 16), (64, 200),
                                          (1000, 4), (2**31 - 1, 4)])
@pytest.mark.parametrize("qlens", [[1, 1, 1, 1], [9, 1, 33, 4], [70, 2, 65, 128]])
def test_attention_window_and_sinks(window, sinks, qlens):
    lens = [max(q, n) for q, n in zip(qlens, [5, 64, 300, 131])]
    b = Batch(lens, qlens, 2, 4, 64, 24, torch.float16, seed=window % 1000 + sinks)
    b.check(b.run(window, sinks), window, sinks, rows=[0, 1, 5, 31, 32, 64, -1])
    b = Batch(lens, qlens, 1, 2, 128, 16, torch.bfloat16, seed=window % 1000 + sinks)
    b.check(b.run(window, sinks), window, sinks, rows=[0, 1, 5, 31, 32, 64, -1])


@pytest.mark.parametrize("dtype,window", [(torch.bfloat16, 0), (torch.float16, 0),
                                          (torch.float16, 1500)])
@pytest.mark.parametrize("d,hkv,group", [(128, 2, 8), (64, 1, 16), (256, 1, 4)])
def test_attention_long_suffix(dtype, window, d, hkv, group):
    """Hundreds of query rows over thousands of keys: every ring and buffer goes
    round many times, and every run gives the same bits."""
    b = Batch([5000, 700, 2500], [260, 70, 1], hkv, group, d, 16, dtype, seed=d)
    out = b.run(window, 4 if window else 0)
    b.check(out, window, 4 if window else 0, rows=[0, 17, 128, 255, -1])
    for _ in range(10):
        assert torch.equal(b.run(window, 4 if window else 0), out)
    assert c_ops.device_status(0) == 0


def test_attention_queries_before_the_cache():
    """More queries than tokens: the first ones stand before position 0 and see
    nothing, so their rows are zeros."""
    for qlens, lens in (([4, 70], [2, 3]), ([5], [0])):
        b = Batch(lens, qlens, 2, 2, 64, 16, torch.float16)
        out = b.run()
        b.check(out)
        assert bool((out[: qlens[0] - lens[0]] == 0).all())


def test_attention_padded_batch():
    """Requests without queries and rows behind the last one."""
    b = Batch([30, 0, 0], [1, 0, 0], 2, 4, 128, 16, torch.bfloat16, pad=7)
    b.check(b.run())
    assert c_ops.device_status(0) == 0


@pytest.mark.parametrize("std,shift", [(1e-4, 0.0), (300.0, 0.0), (0.01, 5.0), (1.0, -40.0)])
def test_attention_value_ranges(std, shift):
    """Small, large and shifted caches: scales over the fp16 range."""
    b = Batch([90, 300], [1, 1], 2, 4, 128, 16, torch.bfloat16, std=std, shift=shift)
    if std > 10:
        b.scale = 1e-5
    b.check(b.run())


def test_attention_scales_that_differ_by_powers():
    """Value scales that grow and shrink by many powers of two along the cache,
    and rows of one value only (scale 0)."""
    for d in (64, 128):
        b = Batch([257], [1], 1, 8, d, 16, torch.float16)
        g = torch.Generator().manual_seed(2)
        n = 257
        for half in range(2):
            codes = torch.randint(0, 16, (n, 1, d), generator=g)
            e = torch.randint(-14, 6, (n, 1), generator=g).double()
            scale = (2.0**e) if half else torch.full((n, 1), 0.05, dtype=torch.float64)
            scale[5::9] = 0
            zero = torch.randn(n, 1, generator=g).half().double()
            words = ref.kv4_words(codes, scale, zero)
            tok = torch.arange(n)
            slot = b.table[0].cpu().long()[tok // 16] * 16 + tok % 16
            b.cache[half].view(-1, b.cache.shape[-1])[slot.to(DEV), : words.shape[1]] = words.to(DEV)
            b.codes[0][half], b.params[0][half] = codes, (scale, zero)
        b.check(b.run())


def test_attention_query_ranges():
    """Tiny, huge and zero queries; a NaN query spoils its own row only."""
    b = Batch([100], [1], 1, 6, 128, 16, torch.bfloat16)
    q = b.q.clone()
    q[0, 0] = 0
    q[0, 1] *= 2.0**-60
    q[0, 2] *= 2.0**-30
    q[0, 3, 1:] *= 2.0**-20  # one value dominates the row
    b.q = q
    b.check(b.run())
    q2 = q.clone()
    q2[0, 4, 7] = float("nan")
    b.q = q2
    out = b.run()
    assert bool(out[0, 4].isnan().all())
    b.q = q
    keep = [0, 1, 2, 3, 5]
    clean = b.run()
    assert torch.equal(out[0, keep], clean[0, keep])


def test_attention_bad_pages_and_lengths():
    b = Batch([40, 40, 40], [1, 1, 1], 2, 2, 64, 16, torch.float16)
    good = b.run()
    b.table[1, 1] = b.cache.shape[1] + 5   # outside the cache: its keys are not seen
    b.table[2, 2] = -3
    out = b.run()
    assert c_ops.device_status(0) == FLAGS.LMCB_DEVICE_FLAG_SLOT_OUT_OF_RANGE
    assert torch.equal(out[0], good[0])
    keep = {1: list(range(16)) + list(range(32, 40)), 2: list(range(32))}
    for r, toks in keep.items():
        codes = [c[toks] for c in b.codes[r]]
        params = [(s[toks], z[toks]) for s, z in b.params[r]]
        want, slack = ref.kv4_attention(b.q[r : r + 1].cpu(), codes, params, b.scale, [99], 0, 0, 2)
        err = (out[r : r + 1].cpu().double() - want).abs()
        assert bool((err <= half_step(torch.float16) * (want.abs() + slack) + slack).all())
    # a length beyond the table's row counts as none
    b2 = Batch([40, 40], [1, 1], 2, 2, 64, 16, torch.float16)
    b2.lens_t[1] = 16 * b2.table.shape[1] + 1
    out = b2.run()
    assert c_ops.device_status(0) == FLAGS.LMCB_DEVICE_FLAG_LENGTH_OUT_OF_RANGE
    assert bool((out[1] == 0).all())
    # query_start that leaves the rows, descends or exceeds the promised length
    b3 = Batch([40, 40, 40], [2, 2, 2], 2, 2, 64, 16, torch.float16)
    good = b3.run()
    b3.starts[3] = 99
    out = b3.run()
    assert c_ops.device_status(0) == FLAGS.LMCB_DEVICE_FLAG_LENGTH_OUT_OF_RANGE
    assert torch.equal(out[:4], good[:4]) and bool((out[4:] == 3).all())
    b3.starts[3] = 6
    out = b3.run(max_query=1)
    assert c_ops.device_status(0) == FLAGS.LMCB_DEVICE_FLAG_LENGTH_OUT_OF_RANGE
    assert bool((out == 3).all())


@pytest.mark.parametrize("offset", [0, 1])
def test_attention_strided_queries(offset):
    for d, dtype in ((128, torch.bfloat16), (64, torch.float16)):
        b = Batch([50, 7, 90], [1, 2, 3], 2, 4, d, 16, dtype)
        wide = torch.zeros(6, 8 * d * 2 + 5 * offset, dtype=dtype, device=DEV)
        q = wide[:, offset : offset + 8 * d].view(6, 8, d)
        q.copy_(b.q)
        full = torch.full((6, 8 * d + 3 * offset), 3.0, dtype=dtype, device=DEV)
        out = full[:, : 8 * d].view(6, 8, d)
        b.run(q=q, out=out)
        assert torch.equal(out, b.run())


def test_attention_same_result_every_time():
    b = Batch([3000, 17, 900], [1] * 3, 2, 4, 128, 16, torch.bfloat16)
    first = b.run()
    for _ in range(5):
        assert torch.equal(b.run(), first)


def test_attention_far_offsets():
    """A cache whose rows lie beyond 2^32 words."""
    hkv, d, bs = 8, 128, 16
    words = ref.kv4_row_words(hkv, d)
    blocks = (1 << 32) // (2 * bs * words) + 70000
    free = torch.cuda.mem_get_info()[0]
    if free < 2 * blocks * bs * words * 4 + (4 << 30):
        pytest.skip("not enough device memory")
    b = Batch([100, 33], [1, 3], hkv, 2, d, bs, torch.bfloat16)
    want = b.run()
    big = torch.empty(2, blocks, bs, 1, words, dtype=torch.int32, device=DEV)
    n = b.cache.shape[1]
    big[:, blocks - n :] = b.cache
    b.table = torch.where(b.table >= 0, b.table + (blocks - n), b.table)
    b.cache = big
    assert torch.equal(b.run(), want)
    slots = torch.tensor([blocks * bs - 1, 0], device=DEV)
    x = torch.randn(2, hkv, d, device=DEV)
    c_ops.kv4_store(x, x, big, slots)
    for half in range(2):
        rows = big[half].view(-1, words)[slots]
        assert torch.equal(rows[:, : hkv * 17].cpu(), ref.kv4_words(*ref.kv4_quantise(x.cpu())))


def test_attention_refusals():
    b = Batch([20, 20], [1, 1], 2, 4, 64, 16, torch.float16)
    out = torch.empty_like(b.q)
    ok = [b.q, b.cache, b.table, b.lens_t, None, 1, 20, 2, 0.1, 0, 0, out]
    c_ops.kv4_attention(*ok)

    def bad(at, value, match):
        a = list(ok)
        a[at] = value
        with pytest.raises(RuntimeError, match=match):
            c_ops.kv4_attention(*a)

    bad(0, b.q.float(), "dtype")
    bad(0, b.q[:1], "shape")
    bad(1, b.cache[:1], "kv_cache")
    bad(2, b.table.long(), "int32")
    bad(2, b.table[:1], "contiguous vector of 1")
    bad(3, b.lens_t[:1], "contiguous vector of 2")
    bad(4, b.lens_t, "contiguous vector of 3")
    bad(5, 0, "invalid shape")
    bad(7, 3, "num_kv_heads must divide")
    bad(7, 4, "rows have")
    bad(9, -1, "invalid shape")
    bad(11, b.q, "overlaps")
    bad(11, out.cpu(), "must be a CUDA tensor")
    a = list(ok)
    a[0] = a[11] = None
    a[0], a[11] = b.q.float(), out.float()
    with pytest.raises(RuntimeError, match="bf16 or fp16"):
        c_ops.kv4_attention(*a)


@pytest.mark.parametrize("scale", [0.0, -0.11, 3.0])
@pytest.mark.parametrize("qlens", [[1, 1], [30, 2]])
def test_attention_other_scales(scale, qlens):
    """No scale (the mean of the values), a negative and a large one."""
    for d, dtype in ((128, torch.bfloat16), (64, torch.float16)):
        b = Batch([300, 77], qlens, 2, 4, d, 16, dtype, seed=d)
        b.scale = scale
        b.check(b.run())
        b.check(b.run(20, 3), 20, 3)


def test_attention_shared_pages():
    """Two requests on the same pages (a shared prefix) give the same rows."""
    b = Batch([333, 333, 90], [1, 1, 1], 2, 4, 128, 16, torch.bfloat16)
    b.table[1] = b.table[0]
    b.q[1] = b.q[0]
    out = b.run()
    assert torch.equal(out[0], out[1])


def test_attention_into_a_packed_buffer():
    """out beside the queries in one buffer of rows."""
    b = Batch([50, 70], [1, 1], 2, 4, 64, 16, torch.float16)
    want = b.run()
    buf = torch.zeros(2, 16 * 64, dtype=torch.float16, device=DEV)
    q, out = buf[:, : 8 * 64].view(2, 8, 64), buf[:, 8 * 64 :].view(2, 8, 64)
    q.copy_(b.q)
    b.run(q=q, out=out)
    assert torch.equal(out, want) and torch.equal(q, b.q)


# ---------------------------------------------------------------------------
# Streams, graphs, and all of them together
# ---------------------------------------------------------------------------

def test_on_another_stream_and_in_graphs():
    """Captured once, replayed over new inputs, two graphs in turn."""
    b = Batch([900, 40, 333], [1] * 3, 2, 4, 128, 16, torch.bfloat16, seed=1)
    c = Batch([64, 2000, 1], [1] * 3, 2, 4, 128, 16, torch.bfloat16, seed=2)
    want_b, want_c = b.run(), c.run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(b.run(), want_b)
    torch.cuda.synchronize()
    outs, graphs = [], []
    for batch in (b, c):
        out = torch.zeros_like(batch.q)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            batch.run(out=out)
        outs.append(out)
        graphs.append(graph)
    for _ in range(3):
        for out, graph in zip(outs, graphs):
            out.zero_()
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want_b) and torch.equal(outs[1], want_c)
    # new lengths and queries in the captured buffers
    b.lens_t.copy_(torch.tensor([500, 39, 2]))
    b.q.mul_(0.5)
    graphs[0].replay()
    torch.cuda.synchronize()
    b.lens = [500, 39, 2]
    b.codes = [[x[:n] for x in cs] for cs, n in zip(b.codes, b.lens)]
    b.params = [[(s[:n], z[:n]) for s, z in ps] for ps, n in zip(b.params, b.lens)]
    b.check(outs[0])
    assert c_ops.device_status(0) == 0


def test_two_streams_at_once():
    batches = [Batch([1500, 7, 600], [1] * 3, 2, 4, 128, 16, torch.bfloat16, seed=s)
               for s in range(2)]
    want = [x.run() for x in batches]
    streams = [torch.cuda.Stream() for _ in batches]
    torch.cuda.synchronize()
    got = []
    for _ in range(20):
        for x, s in zip(batches, streams):
            with torch.cuda.stream(s):
                got.append(x.run())
    torch.cuda.synchronize()
    for i, out in enumerate(got):
        assert torch.equal(out, want[i % 2])


def test_a_layer_of_a_serving_step():
    """Slot mapping, norm + rotation, 4-bit store, offload through the
    framework's connector, retrieval into other pages, attention: a prefill
    and two decode steps, each against the whole chain in 64 bits."""
    from lmcache_b200.v1.gpu_connector import VLLMPagedMemGPUConnectorV2

    hq, hk, d, bs, blocks, cols = 8, 2, 128, 16, 64, 12
    rng = random.Random(0)
    g = torch.Generator().manual_seed(11)
    words = c_ops.kv4_row_words(hk, d)
    caches = [new_cache(blocks, bs, hk, d) for _ in range(2)]  # two layers; layer 1 is used
    order = list(range(blocks))
    rng.shuffle(order)
    free = torch.tensor(order, dtype=torch.int32, device=DEV)
    table = torch.full((3, cols), -1, dtype=torch.int32, device=DEV)
    ctx = torch.zeros(3, dtype=torch.int32, device=DEV)
    weights = [(1 + 0.1 * torch.randn(d, generator=g)).bfloat16().to(DEV) for _ in range(2)]
    rope = cos_sin(512, d).to(DEV)
    history = [[], [], []]  # per request: (key, value) rows as stored, [n, hk, d]
    used = 0
    for step, new in enumerate(([70, 5, 33], [1, 1, 1], [1, 1, 1])):
        n = sum(new)
        new_t = torch.tensor(new, dtype=torch.int32, device=DEV)
        slots = torch.empty(n + 3, dtype=torch.int64, device=DEV)
        positions = torch.empty_like(slots)
        starts = torch.empty(4, dtype=torch.int32, device=DEV)
        lens = torch.empty(3, dtype=torch.int32, device=DEV)
        taken = torch.empty(1, dtype=torch.int32, device=DEV)
        c_ops.build_slot_mapping(ctx, new_t, table, free[used:], bs, slots, positions, starts, lens,
                                 taken)
        qkv = torch.randn(n + 3, (hq + 2 * hk) * d, generator=g).bfloat16().to(DEV)
        q = qkv[:, : hq * d].view(-1, hq, d)
        k = qkv[:, hq * d : (hq + hk) * d].view(-1, hk, d)
        v = qkv[:, (hq + hk) * d :].view(-1, hk, d)
        c_ops.qk_norm_rope(q, k, *weights, positions, rope, 1e-6, True, q, k)
        c_ops.kv4_store(k, v, caches[1], slots)
        out = torch.full((n + 3, hq, d), 3.0, dtype=torch.bfloat16, device=DEV)
        c_ops.kv4_attention(q, caches[1], table, lens, starts, max(new), int(lens.max()), hk,
                            d**-0.5, 0, 0, out)
        used += int(taken)
        at = 0
        for r in range(3):
            history[r].append((k[at : at + new[r]].cpu(), v[at : at + new[r]].cpu()))
            ks, vs = (torch.cat([h[i] for h in history[r]]) for i in range(2))
            assert ks.shape[0] == int(lens[r])
            quant = [ref.kv4_quantise(x) for x in (ks, vs)]
            pos = list(range(ks.shape[0] - new[r], ks.shape[0]))
            want, slack = ref.kv4_attention(q[at : at + new[r]].cpu(), [x[0] for x in quant],
                                            [x[1:] for x in quant], d**-0.5, pos, 0, 0, hk)
            err = (out[at : at + new[r]].cpu().double() - want).abs()
            assert bool((err <= half_step(torch.bfloat16) * (want.abs() + slack) + slack).all())
            at += new[r]
        assert bool((out[n:] == 3).all())
        ctx = lens
    # Request 0 goes out to an LMCache object and comes back into other pages.
    n0 = int(ctx[0])
    tok = torch.arange(n0, device=DEV)
    slots0 = table[0].long()[tok // bs] * bs + tok % bs
    connector = VLLMPagedMemGPUConnectorV2(words, 2)

    class Obj:
        tensor = torch.zeros(connector.get_shape(n0), dtype=torch.int32, device=DEV)

    connector.from_gpu(Obj, 0, n0, kvcaches=caches, slot_mapping=slots0)
    fresh = [new_cache(blocks, bs, hk, d) for _ in range(2)]
    pages = -(-n0 // bs)
    table2 = torch.randperm(blocks, generator=g)[:pages].int().to(DEV).view(1, -1)
    slots2 = table2[0].long()[tok // bs] * bs + tok % bs
    connector.to_gpu(Obj, 0, n0, kvcaches=fresh, slot_mapping=slots2)
    q = torch.randn(1, hq, d, generator=g).bfloat16().to(DEV)
    outs = []
    for cache, tab in ((caches[1], table[:1]), (fresh[1], table2)):
        out = torch.empty_like(q)
        c_ops.kv4_attention(q, cache, tab, ctx[:1].contiguous(), None, 1, n0, hk, d**-0.5, 0, 0, out)
        outs.append(out)
    assert torch.equal(*outs)
    assert c_ops.device_status(0) == 0
