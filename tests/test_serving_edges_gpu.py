"""GPU tests of the serving operators at the edges of what their calls allow:
tables with holes, batch sizes around a launch limit, values and lengths at the
ends of their types, keys that a query does not see."""

import os
import subprocess
import sys

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
