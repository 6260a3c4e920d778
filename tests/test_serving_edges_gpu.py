"""GPU tests of the serving operators at the edges of what their calls allow:
tables with holes, batch sizes around a launch limit, values and lengths at the
ends of their types, keys that a query does not see."""

import ctypes
import os
import shutil
import subprocess
import sys

import numpy as np
import pytest
import torch

from lmcache_b200 import abi, c_ops
from oracle import serving as ref
from tests import test_serving_gpu as base

pytestmark = pytest.mark.gpu
DEV = "cuda"
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(autouse=True)
def clean_status():
    c_ops.device_status(0)
    yield
    c_ops.device_status(0)


# ---------------------------------------------------------------------------
# Tables with holes in front of the cache's first row
# ---------------------------------------------------------------------------

def with_hole(bs, pages, holes, zero_at, hkv, group, d, dtype, qlen=1, seed=0):
    """A request whose table has entries of -1 at `holes` and page 0 at `zero_at`."""
    n = bs * pages - bs // 2
    b = base.Batch([n], [qlen], hkv, group, d, bs, dtype, seed=seed)
    old = b.table[0, :pages].clone()
    # the page at zero_at moves to page 0, and what was on page 0 takes its place
    swap = b.cache.clone()
    first, there = 0, int(old[zero_at])
    b.cache[:, first], b.cache[:, there] = swap[:, there], swap[:, first]
    new = torch.where(old == there, first, torch.where(old == first, there, old))
    for h in holes:
        new[h] = -1
    b.table[0, :pages] = new
    gone = torch.zeros(n, dtype=torch.bool)
    for h in holes:
        gone[h * bs : (h + 1) * bs] = True
    return b, n, gone


def check_with_hole(b, n, gone, window, sinks):
    out = b.run(window, sinks)
    flags = c_ops.device_status(0)
    assert flags & abi.LMCB_DEVICE_FLAG_WAIT_TIMEOUT == 0
    pos = torch.arange(n - b.qlens[0], n)
    keys = torch.arange(n)
    for i, p in enumerate(pos):
        seen = ref.visible(int(p), keys, window, sinks) & ~gone
        codes = [c[seen] for c in b.codes[0]]
        params = [(s[seen], z[seen]) for s, z in b.params[0]]
        want, slack = ref.kv4_attention(b.q[i : i + 1].cpu(), codes, params, b.scale,
                                        [int(seen.sum())], 0, 0, b.hkv)
        err = (out[i : i + 1].cpu().double() - want).abs()
        half = base.half_step(b.dtype)
        assert bool((err <= half * (want.abs() + slack) + slack + 2.0**-25).all())
    return flags


@pytest.mark.parametrize("bs", [8, 16, 24, 64])
@pytest.mark.parametrize("hkv", [1, 2, 8])
def test_attention_hole_before_page_zero(bs, hkv):
    """Page 0 right behind an entry that is not there, at the start of a tile and
    inside one, one hole or several, with and without a window."""
    cases = [([0], 1), ([0, 1, 2], 3), ([2], 3), ([1, 2], 3), ([0, 3], 4), ([4], 5)]
    for i, (holes, zero_at) in enumerate(cases):
        b, n, gone = with_hole(bs, 7, holes, zero_at, hkv, 4, 128, torch.bfloat16, seed=i)
        assert check_with_hole(b, n, gone, 0, 0) == abi.LMCB_DEVICE_FLAG_SLOT_OUT_OF_RANGE
        for window, sinks in ((bs * 4 + 1, 0), (bs * 2, bs + 3), (5, 3 * bs)):
            check_with_hole(b, n, gone, window, sinks)


@pytest.mark.parametrize("qlen,hkv,group,d", [(3, 2, 4, 64), (40, 2, 2, 128), (1, 12, 2, 64),
                                              (2, 1, 4, 256)])
def test_attention_hole_before_page_zero_other_kernels(qlen, hkv, group, d):
    """The same with several queries, many query rows, and KV heads in groups."""
    for holes, zero_at in (([0], 1), ([2], 3)):
        b, n, gone = with_hole(16, 6, holes, zero_at, hkv, group, d, torch.float16, qlen=qlen)
        assert check_with_hole(b, n, gone, 0, 0) == abi.LMCB_DEVICE_FLAG_SLOT_OUT_OF_RANGE
        check_with_hole(b, n, gone, 20, 9)


def test_attention_after_the_free_list_ran_out():
    """build_slot_mapping leaves entries of -1 where its list ends; a later step
    puts page 0 behind them, and the attention reads the rest."""
    bs, d = 16, 128
    b = base.Batch([40], [1], 2, 4, d, bs, torch.bfloat16)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    table = torch.full((1, 4), -1, dtype=torch.int32, device=DEV)
    lens, starts, used = i32(0), i32(0, 0), i32(0)
    ctx = i32(0)
    for new, free in ((32, i32()), (8, i32(0))):
        slots = torch.empty(new, dtype=torch.int64, device=DEV)
        c_ops.build_slot_mapping(ctx, i32(new), table, free, bs, slots, torch.empty_like(slots),
                                 starts, lens, used)
        ctx = lens.clone()
    assert table.tolist() == [[-1, -1, 0, -1]] and lens.tolist() == [40]
    k, v = (torch.randn(8, 2, d, device=DEV).bfloat16() for _ in range(2))
    c_ops.kv4_store(k, v, b.cache, slots)
    c_ops.device_status(0)
    out = torch.empty_like(b.q)
    c_ops.kv4_attention(b.q, b.cache, table, lens, None, 1, 40, 2, b.scale, 0, 0, out)
    assert c_ops.device_status(0) == abi.LMCB_DEVICE_FLAG_SLOT_OUT_OF_RANGE
    quant = [ref.kv4_quantise(x.cpu()) for x in (k, v)]
    want, slack = ref.kv4_attention(b.q.cpu(), [x[0] for x in quant], [x[1:] for x in quant],
                                    b.scale, [8], 0, 0, 2)
    err = (out.cpu().double() - want).abs()
    assert bool((err <= base.half_step(torch.bfloat16) * (want.abs() + slack) + slack).all())


# ---------------------------------------------------------------------------
# Batches around the shared memory that a launch has without asking
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("slot", ["int64", "int32"])
@pytest.mark.parametrize("requests", [4074, 4075, 4096, 4097])
def test_slots_around_the_default_shared_memory(requests, slot):
    """The sums of 4075 to 4096 requests fill the default shared memory but for
    what the kernel has besides. In a process of its own: a larger batch before
    raises the limit for good."""
    code = ("import sys; sys.path[:0] = sys.argv[1:3]\n"
            "import numpy as np, torch\n"
            "from tests import test_serving_gpu as base\n"
            f"rs = np.random.RandomState({requests})\n"
            f"base.run_slots(rs.randint(0, 40, {requests}), rs.randint(0, 4, {requests}), 16, 4,"
            f" st=torch.{slot})\n"
            "assert base.c_ops.device_status(0) == 0\n")
    res = subprocess.run([sys.executable, "-c", code, ROOT, os.path.join(ROOT, "lmcache-ascend_b200")],
                         capture_output=True, text=True, cwd=ROOT, timeout=300)
    assert res.returncode == 0, res.stderr[-2000:]


# ---------------------------------------------------------------------------
# Many query rows: V of keys that a query does not see or gives no weight
# ---------------------------------------------------------------------------

def fill(b, r, half, codes, scale, zero):
    """Request r's rows of one half become these."""
    words = ref.kv4_words(codes, scale, zero)
    tok = torch.arange(codes.shape[0])
    slot = b.table[r].cpu().long()[tok // b.bs] * b.bs + tok % b.bs
    b.cache[half].view(-1, b.cache.shape[-1])[slot.to(DEV), : words.shape[1]] = words.to(DEV)
    b.codes[r][half], b.params[r][half] = codes, (scale, zero)


def weighted_bound(b, r, rows, want, window, sinks, spread):
    """What the result of each query row may be off by. Unlike the oracle's own
    bound it counts every key by its weight p, so that a key without weight has
    no share in it: V and P are rounded to fp16 (2^-11 each of sum p |v|); logits
    are off by d = 4 * 2^-19 of their terms, which moves the result by sum p d (v
    - result); (keys / 16 + 8) roundings of 2^-22 of sum p (|v| + 15 s). A P that
    is no normal number is off by 2^-25 where the row's largest is above 2^7; 16
    tokens with a value `spread` times theirs among them have it that much
    smaller."""
    n, length = b.qlens[r], b.lens[r]
    at = sum(b.qlens[:r])
    k, v = (ref.kv4_values(b.codes[r][i], *b.params[r][i]) for i in range(2))
    s = b.params[r][1][0]
    kabs = b.params[r][0][0][..., None] * 15 + b.params[r][0][1].abs()[..., None]
    out = torch.zeros_like(want)
    for i, row in enumerate(rows):
        seen = ref.visible(length - n + row, torch.arange(length), window, sinks)
        for h in range(b.hkv * b.group):
            kv = h // b.group
            x = b.q[at + row, h].cpu().double()
            p = torch.softmax((k[seen, kv] @ x) * b.scale, 0)
            mass = (kabs[seen, kv] * x.abs()).sum(-1) * abs(b.scale)
            big = v[seen, kv].abs()
            size = big + 15 * s[seen, kv, None] + want[i, h].abs()
            steps = (int(seen.sum()) / 16 + 8) * 2.0**-22
            out[i, h] = (2.0**-10 * (p @ big) + (p * (4 * mass * 2.0**-19 + steps)) @ size
                         + 2.0**-32 * spread * p.max() * (big * (p[:, None] > 2.0**-60)).sum(0))
    return out


def check_rows(b, out, r, rows, window=0, sinks=0, spread=1.0):
    at, n = sum(b.qlens[:r]), b.qlens[r]
    pos = [b.lens[r] - n + i for i in rows]
    want, _ = ref.kv4_attention(b.q[at : at + n].cpu()[rows], b.codes[r], b.params[r], b.scale, pos,
                                window, sinks, b.hkv)
    slack = weighted_bound(b, r, rows, want, window, sinks, spread)
    err = (out[at : at + n].cpu().double()[rows] - want).abs()
    bound = base.half_step(b.dtype) * (want.abs() + slack) + slack + 2.0**-25
    assert bool((err <= bound).all()), float((err / bound).max())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("power", [8, 10, 13, 17, 20])
def test_rows_large_value_out_of_sight(dtype, d, power):
    """The value of a key behind a query's position, or in front of its window,
    2^power times its neighbours': the query's row, which lives on those
    neighbours, is as good as without it."""
    n = 60
    for key, window, rows in ((8, 0, range(8)), (41, 0, range(32, 41)), (8, 5, range(13, 16)),
                              (8, 5, range(40, 60))):
        b = base.Batch([n], [n], 1, 2, d, 16, dtype, seed=d, std=2.0**-7)
        codes, (scale, zero) = b.codes[0][1], b.params[0][1]
        scale[key] = (scale[key] * 2.0**power).half().double()
        zero[key] = (zero[key] * 2.0**power).half().double()
        fill(b, 0, 1, codes, scale, zero)
        out = b.run(window, 0)
        check_rows(b, out, 0, list(rows), window, spread=2.0**power)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("power", [8, 10, 13, 17, 20])
@pytest.mark.parametrize("key", [0, 37, 410])
def test_rows_large_value_without_weight(dtype, d, power, key):
    """A key that every query sees and gives no weight, with a value 2^power
    times the others': the rows are as good as without it."""
    n, q = 430, 24
    b = base.Batch([n], [q], 1, 2, d, 16, dtype, seed=d + power, std=2.0**-7)
    codes, (scale, zero) = b.codes[0][1], b.params[0][1]
    scale[key] = (scale[key] * 2.0**power).half().double()
    zero[key] = (zero[key] * 2.0**power).half().double()
    assert float(scale.max()) < 65504 and float(zero.abs().max()) < 65504
    fill(b, 0, 1, codes, scale, zero)
    kc, (ks, kz) = b.codes[0][0], b.params[0][0]
    kz[key], ks[key], kc[key] = -60000.0, 2.0**-7, 0
    fill(b, 0, 0, kc, ks, kz)
    b.q[:, :, 1:] *= 0.01
    b.q[:, :, 0] = 8.0
    b.q[:] = b.q.abs()  # the logits of that key are far below the others'
    check_rows(b, b.run(), 0, [0, 1, 11, 23], spread=2.0**power)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_rows_not_finite_out_of_sight(dtype):
    """A value row that is no number (a page not made by kv4_store) spoils the
    queries that see it and no others."""
    n = 60
    b = base.Batch([n], [n], 1, 2, 128, 16, dtype)
    good = b.run()
    for key in (8, 41):
        slot = int(b.table[0, key // 16]) * 16 + key % 16
        word = b.cache[1].view(-1, b.cache.shape[-1])[slot]
        keep = int(word[16])
        for bad in (0x7E00, 0x7C00, 0x7E000000, 0x7C000000):  # s or z, NaN or infinite
            word[16] = bad
            out = b.run()
            assert bool(out[key:].isnan().all()) or bool((~out[key:].isfinite()).all())
            check_rows(b, out, 0, list(range(key)))
        word[16] = keep
    assert torch.equal(b.run(), good)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_rows_scales_that_differ_by_powers(dtype, d):
    """Value scales that grow and shrink by many powers of two along the cache,
    and rows of one value only (scale 0), with many query rows."""
    n, q = 300, 40
    b = base.Batch([n], [q], 1, 2, d, 16, dtype)
    g = torch.Generator().manual_seed(2)
    for half in range(2):
        codes = torch.randint(0, 16, (n, 1, d), generator=g)
        e = torch.randint(-14, 6, (n, 1), generator=g).double()
        scale = (2.0**e) if half else torch.full((n, 1), 0.05, dtype=torch.float64)
        scale[5::9] = 0
        codes[5::9] = 0
        zero = torch.randn(n, 1, generator=g).half().double()
        fill(b, 0, half, codes, scale, zero)
    check_rows(b, b.run(), 0, [0, 1, 15, 16, 39], spread=2.0**19)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("std,shift", [(1e-4, 0.0), (300.0, 0.0), (0.01, 5.0), (1.0, -40.0)])
def test_rows_value_ranges(dtype, std, shift):
    """Small, large and shifted caches with many query rows."""
    b = base.Batch([90, 300], [30, 50], 2, 4, 128, 16, dtype, std=std, shift=shift)
    if std > 10:
        b.scale = 1e-5
    out = b.run()
    for r in range(2):
        check_rows(b, out, r, [0, 7, 29])


@pytest.mark.parametrize("d", [64, 128, 256])
def test_rows_of_one_value(d):
    """Caches whose rows hold one value each (scale 0), down to the smallest."""
    n, q = 150, 30
    b = base.Batch([n], [q], 1, 2, d, 16, torch.float16)
    for value in (0.0, 2.0**-24, -3.0, 65504.0):
        zero = torch.full((n, 1), value, dtype=torch.float64)
        fill(b, 0, 1, torch.zeros(n, 1, d, dtype=torch.long), torch.zeros_like(zero), zero)
        out = b.run()
        assert bool((out == value).all())


# ---------------------------------------------------------------------------
# kv4_store: the scale
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("exponent", [-12, 0, 13])
def test_kv4_scale_of_every_span(exponent):
    """Every fp32 span of a binade: rows [0, span, ...], whose scale is the fp32
    product of the span with fp32(1 / 15), rounded to fp16. That is a fifteenth of the
    span but where the product and the quotient, a step of fp32 apart, lie on both
    sides of one of the (at most 2049) borders of fp16 in two binades."""
    n, d = 1 << 23, 8
    span = torch.arange(n, device=DEV, dtype=torch.int32).add_((127 + exponent) << 23).view(
        torch.float32)
    x = torch.zeros(n, 1, d, device=DEV)
    x[:, 0, 3] = span
    cache = torch.full((2, n // 16, 16, 1, ref.kv4_row_words(1, d)), -1, dtype=torch.int32,
                       device=DEV)
    c_ops.kv4_store(x, x, cache, torch.arange(n, device=DEV, dtype=torch.int32))
    got = cache[0].view(n, -1)[:, 1].contiguous().view(torch.float16)[::2]
    fifteenth = float(torch.tensor(1.0 / 15.0, dtype=torch.float32))
    assert torch.equal(got, (span.double() * fifteenth).float().half())
    quotient = (span.double() / 15.0).half()
    assert int((got != quotient).sum()) <= 2 * 2049
    assert torch.equal(cache[0], cache[1])


# ---------------------------------------------------------------------------
# The widest windows, and queries before the cache
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("window", [2**31 - 1, 2**31 - 2, 2**31 - 40, 2**30, 7])
@pytest.mark.parametrize("qlen,length", [(8, 5), (4, 1), (3, 0), (70, 30), (200, 130)])
@pytest.mark.parametrize("d,dtype", [(64, torch.float16), (128, torch.bfloat16)])
def test_window_with_queries_before_the_cache(window, qlen, length, d, dtype):
    """More queries than tokens under a window of any width: queries before
    position 0 give zeros, the others see their keys."""
    b = base.Batch([length, 50], [qlen, 2], 1, 2, d, 16, dtype, seed=qlen)
    out = b.run(window, 3)
    b.check(out, window, 3, rows=list(range(0, qlen, 7)) + [-1, -2, -3, qlen - length])
    assert bool((out[: qlen - length] == 0).all())
    assert c_ops.device_status(0) == 0


# ---------------------------------------------------------------------------
# Waits that give up
# ---------------------------------------------------------------------------

WAIT_SOURCE = r"""
#include "kv4_attention.cuh"

// A warp waits for the first phase of an mbarrier, `limit` polls at most, and
// each lane writes what it was told. `arrive`: the phase ends before the wait.
__global__ void wait_kernel(unsigned limit, int arrive, int* told) {
  __shared__ uint64_t bar;
  const int lane = threadIdx.x;
  if (lane == 0) {
    lmcb::kv4::mbar_init(&bar, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    if (arrive) lmcb::kv4::mbar_arrive(&bar);
  }
  __syncwarp();
  told[lane] = lmcb::kv4::warp_wait(&bar, 0, limit);
}

extern "C" int run_wait(unsigned limit, int arrive, int* told) {
  wait_kernel<<<1, 32>>>(limit, arrive, told);
  return cudaDeviceSynchronize();
}
"""


@pytest.fixture(scope="module")
def wait_library(tmp_path_factory):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        pytest.skip("no nvcc")
    where = tmp_path_factory.mktemp("wait")
    source, library = where / "wait.cu", where / "wait.so"
    source.write_text(WAIT_SOURCE)
    subprocess.run([nvcc, "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a", "-shared",
                    "-Xcompiler", "-fPIC", "-I" + os.path.join(ROOT, "include"),
                    "-I" + os.path.join(ROOT, "lmcache-ascend_b200", "csrc"), str(source), "-o",
                    str(library)], check=True, timeout=300)
    return ctypes.CDLL(str(library))


@pytest.mark.parametrize("limit", [0, 1, 64])
@pytest.mark.parametrize("arrive", [0, 1])
def test_a_wait_tells_the_warp_one_thing(wait_library, arrive, limit):
    """A wait that nobody answers gives up after its polls, for every lane, and
    one whose phase has ended does not."""
    told = torch.full((32,), -1, dtype=torch.int32, device=DEV)
    assert wait_library.run_wait(limit, arrive, ctypes.c_void_p(told.data_ptr())) == 0
    assert told.tolist() == [arrive if limit else 0] * 32


# ---------------------------------------------------------------------------
# qk_norm_rope: infinities and NaN
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("neox", [True, False])
@pytest.mark.parametrize("d,rot", [(128, 64), (128, 128), (64, 0), (256, 32), (80, 40), (72, 24)])
@pytest.mark.parametrize("value", [float("inf"), -float("inf"), float("nan")])
def test_qk_not_finite(dtype, neox, d, rot, value):
    """One element, or one weight, that is not finite, at every place: the
    results are not finite exactly where the definition has it. Rows of
    vectors and rows of elements (by the sizes) alike."""
    cache = base.cos_sin(32, rot).to(DEV)
    cache[:4] = base.cos_sin(36, rot)[32:].to(DEV)  # no angle 0: sin 0 times inf is no matter here
    g = torch.Generator().manual_seed(1)
    x = torch.randn(d, 1, d, generator=g).to(dtype)
    pos = torch.randint(1, 32, (d,), generator=g).to(DEV)
    q = x.clone()
    q[torch.arange(d), 0, torch.arange(d)] = value  # row i: element i
    q, k = q.to(DEV), x.to(DEV)
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    c_ops.qk_norm_rope(q, k, None, None, pos, cache, 1e-6, neox, qo, ko)
    base.check_qk(ko, k, None, pos, cache, 1e-6, neox)

    def same_kind(got, want):
        got, want = got.cpu().double(), want.to(dtype).double()
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got.isinf(), want.isinf())
        assert torch.equal(got[want.isinf()], want[want.isinf()])
        return ~want.isnan() & ~want.isinf(), got, want

    fine, got, want = same_kind(qo, ref.qk_norm_rope(q.cpu(), None, pos.cpu(), cache.cpu(), 1e-6,
                                                     neox))
    assert bool((got[fine] == 0).all()) and bool((want[fine] == 0).all())
    for at in sorted({0, 1, rot // 2, max(rot - 1, 0), min(rot, d - 1), d - 2, d - 1}):
        w = torch.ones(d)
        w[at] = value
        w = w.to(DEV)
        c_ops.qk_norm_rope(k, k, w, None, pos, cache, 1e-6, neox, qo, ko)
        want = ref.qk_norm_rope(k.cpu(), w.cpu(), pos.cpu(), cache.cpu(), 1e-6, neox)
        fine, got, want = same_kind(qo, want)
        rel = base.half_step(dtype) + (d / 2 + 16) * 2.0**-23
        size = ref.qk_norm_rope(k.cpu(), None, pos.cpu(), cache.cpu(), 1e-6, neox).abs().amax(-1)
        bound = rel * (want[fine].abs() + size.max()) + 2.0**-24
        assert bool(((got[fine] - want[fine]).abs() <= bound).all())


# ---------------------------------------------------------------------------
# Few query rows: value rows that are no numbers
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d,group", [(64, 1), (64, 2), (128, 1), (256, 1)])
def test_decode_not_finite_out_of_sight(dtype, d, group):
    """Several queries in the decode kernel: a value row that is no number (a page
    not made by kv4_store) spoils the queries that see it and no others."""
    n, q = 40, 8
    b = base.Batch([n], [q], 2, group, d, 16, dtype)
    good = b.run()
    for key in (33, 38):
        slot = int(b.table[0, key // 16]) * 16 + key % 16
        row = b.cache[1].view(-1, b.cache.shape[-1])[slot]
        keep = row.clone()
        for bad in (0x7E00, 0x7C00, 0x7E000000, 0x7C000000):  # s or z, NaN or infinite
            row[2 * d // 8 : 2 * d // 8 + 2] = bad
            out = b.run()
            first = key - (n - q)  # the first query that sees it
            assert bool((~out[first:].isfinite()).any(-1).all())
            assert torch.equal(out[:first], good[:first])
        row.copy_(keep)
    assert torch.equal(b.run(), good)


# ---------------------------------------------------------------------------
# Many query rows on streams and in graphs, and the ends of the shapes
# ---------------------------------------------------------------------------

def test_rows_on_streams_and_in_graphs():
    """The kernel for many query rows with its cache split over CTAs: two graphs
    replayed in turn, over new lengths too, and two streams at once."""
    batches = [base.Batch([3000, 40], [30, 20], 1, 2, 128, 16, torch.bfloat16, seed=s)
               for s in range(2)]
    want = [b.run() for b in batches]
    outs, graphs = [], []
    for b in batches:
        out, graph = torch.full_like(b.q, 3.0), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            b.run(out=out)
        outs.append(out)
        graphs.append(graph)
    for _ in range(3):
        for out, graph in zip(outs, graphs):
            out.fill_(3.0)
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))
    b = batches[0]
    b.lens_t.copy_(torch.tensor([1777, 25]))
    graphs[0].replay()
    torch.cuda.synchronize()
    b.lens = [1777, 25]
    b.codes = [[x[:n] for x in cs] for cs, n in zip(b.codes, b.lens)]
    b.params = [[(s[:n], z[:n]) for s, z in ps] for ps, n in zip(b.params, b.lens)]
    b.check(outs[0], rows=[0, 1, 15, 29])
    b = base.Batch([3000, 40], [30, 20], 1, 2, 128, 16, torch.bfloat16, seed=0)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(10):
        for x, s in zip((b, batches[1]), streams):
            with torch.cuda.stream(s):
                got.append(x.run())
    torch.cuda.synchronize()
    for i, out in enumerate(got):
        assert torch.equal(out, want[i % 2])
    assert c_ops.device_status(0) == 0


@pytest.mark.parametrize("qlen", [1, 17])
def test_attention_most_requests(qlen):
    """4096 requests, one of them long, most with one query, some without."""
    rs = np.random.RandomState(qlen)
    lens = rs.randint(1, 40, 4096)
    lens[1234] = 900
    qlens = np.minimum(rs.randint(0, qlen + 1, 4096), lens)
    qlens[[0, 4095]] = 1
    b = base.Batch([int(n) for n in lens], [int(n) for n in qlens], 1, 1, 64, 16, torch.float16,
                   pad=2)
    b.check(b.run(max_query=qlen), rows=[0, 5, -1])
    assert c_ops.device_status(0) == 0


@pytest.mark.parametrize("hkv,group,d", [(1, 4096, 64), (8, 512, 64), (128, 1, 64), (64, 1, 256),
                                         (256, 16, 64)])
def test_attention_most_heads(hkv, group, d):
    """Up to 4096 query heads, over one KV head or many."""
    b = base.Batch([70, 3], [1, 2], hkv, group, d, 16, torch.bfloat16)
    out = b.run()
    heads = sorted({0, 1, group - 1, group % (hkv * group), hkv * group // 2, hkv * group - 1})
    at = 0
    for r, n in enumerate(b.qlens):
        for h in heads:
            kv = h // group
            pick = [[c[:, kv : kv + 1] for c in b.codes[r]],
                    [(s[:, kv : kv + 1], z[:, kv : kv + 1]) for s, z in b.params[r]]]
            pos = [b.lens[r] - n + i for i in range(n)]
            want, slack = ref.kv4_attention(b.q[at : at + n, h : h + 1].cpu(), *pick, b.scale, pos,
                                            0, 0, 1)
            err = (out[at : at + n, h : h + 1].cpu().double() - want).abs()
            assert bool((err <= 2.0**-8 * (want.abs() + slack) + slack).all())
        at += n
    assert c_ops.device_status(0) == 0


@pytest.mark.parametrize("qlens,max_query", [([1, 1, 1], 40), ([2, 0, 3], 64), ([1, 1, 1], 3)])
def test_attention_longer_promises(qlens, max_query):
    """A promised length that no request reaches, pages of 1024 tokens, a block
    table that is part of a wider one, and rows behind the last request."""
    b = base.Batch([700, 5, 1030], qlens, 2, 4, 128, 1024, torch.bfloat16, pad=5)
    wide = torch.full((3, b.table.shape[1] + 7), -5, dtype=torch.int32, device=DEV)
    wide[:, 3 : 3 + b.table.shape[1]] = b.table
    b.table = wide[:, 3 : 3 + b.table.shape[1]]
    out = b.run(max_query=max_query, starts=b.starts, max_len=5000)
    b.check(out)
    assert c_ops.device_status(0) == 0
