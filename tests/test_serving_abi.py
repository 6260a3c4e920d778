"""CPU tests of the serving operators' refusals, at the C entry and in c_ops:
every bad call is an error before anything reaches a GPU."""

import ctypes

import pytest
import torch

from lmcache_b200 import abi, c_ops

INT32, INT64 = abi.LMCB_DTYPE_INT32, abi.LMCB_DTYPE_INT64
BF16, FP16, FP32 = abi.LMCB_DTYPE_BF16, abi.LMCB_DTYPE_FP16, abi.LMCB_DTYPE_FP32
P = 1 << 20  # an address that no refused call touches


def refused(name, status, *args):
    with pytest.raises(abi.LmcbError) as err:
        abi.call(name, *args)
    assert err.value.status == status, err.value


def slot_args(**kw):
    a = dict(ctx=P, new=P, len_type=INT32, batch=4, table=P, stride=8, cols=8, free=P, nfree=16,
             block=16, tokens=32, slots=P, positions=P, slot_type=INT64, starts=P, lens=P, used=P)
    a.update(kw)
    return list(a.values()) + [0]


@pytest.mark.parametrize("kw,status", [
    (dict(len_type=BF16), abi.LMCB_ERR_UNSUPPORTED_DTYPE),
    (dict(slot_type=FP32), abi.LMCB_ERR_UNSUPPORTED_DTYPE),
    (dict(batch=-1), abi.LMCB_ERR_INVALID_ARGUMENT),
    (dict(stride=7), abi.LMCB_ERR_INVALID_ARGUMENT),
    (dict(block=0), abi.LMCB_ERR_INVALID_ARGUMENT),
    (dict(cols=1 << 20, stride=1 << 20, block=1 << 12), abi.LMCB_ERR_INVALID_ARGUMENT),
    (dict(tokens=-1), abi.LMCB_ERR_INVALID_ARGUMENT),
    (dict(nfree=-1), abi.LMCB_ERR_INVALID_ARGUMENT),
    (dict(batch=16385), abi.LMCB_ERR_CAPACITY),
    (dict(ctx=None), abi.LMCB_ERR_INVALID_ARGUMENT),
    (dict(table=None), abi.LMCB_ERR_INVALID_ARGUMENT),
    (dict(free=None), abi.LMCB_ERR_INVALID_ARGUMENT),
    (dict(slots=None), abi.LMCB_ERR_INVALID_ARGUMENT),
    (dict(starts=None), abi.LMCB_ERR_INVALID_ARGUMENT),
])
def test_build_slot_mapping_refuses(kw, status):
    refused("lmcb_build_slot_mapping", status, *slot_args(**kw))


def qk_args(**kw):
    a = dict(q=P, k=P, type=BF16, qs=512, ks=256, qw=P, qwt=BF16, kw=P, kwt=BF16, pos=P,
             post=INT64, cache=P, cachet=FP32, rot=128, maxpos=1024, neox=1, eps=1e-6, tokens=8,
             hq=4, hk=2, d=128, qo=P, qos=512, ko=P, kos=256)
    a.update(kw)
    return list(a.values()) + [0]


@pytest.mark.parametrize("kw,status", [
    (dict(type=INT32), abi.LMCB_ERR_UNSUPPORTED_DTYPE),
    (dict(cachet=INT64), abi.LMCB_ERR_UNSUPPORTED_DTYPE),
    (dict(qwt=INT64), abi.LMCB_ERR_UNSUPPORTED_DTYPE),
    (dict(post=BF16), abi.LMCB_ERR_UNSUPPORTED_DTYPE),
    (dict(rot=127), abi.LMCB_ERR_INVALID_ARGUMENT),
    (dict(rot=130), abi.LMCB_ERR_INVALID_ARGUMENT),
    (dict(qs=511), abi.LMCB_ERR_INVALID_ARGUMENT),
    (dict(kos=255), abi.LMCB_ERR_INVALID_ARGUMENT),
    (dict(maxpos=0), abi.LMCB_ERR_INVALID_ARGUMENT),
    (dict(d=0), abi.LMCB_ERR_INVALID_ARGUMENT),
    (dict(tokens=1 << 31), abi.LMCB_ERR_INVALID_ARGUMENT),
    (dict(q=None), abi.LMCB_ERR_INVALID_ARGUMENT),
    (dict(ko=None), abi.LMCB_ERR_INVALID_ARGUMENT),
    (dict(pos=None), abi.LMCB_ERR_INVALID_ARGUMENT),
    (dict(cache=None), abi.LMCB_ERR_INVALID_ARGUMENT),
])
def test_qk_norm_rope_refuses(kw, status):
    refused("lmcb_qk_norm_rope", status, *qk_args(**kw))


def test_row_words():
    lib = abi.load()
    assert lib.lmcb_kv4_row_words(8, 128) == 136
    assert lib.lmcb_kv4_row_words(1, 128) == 20  # 17 rounded up to 16 bytes
    assert lib.lmcb_kv4_row_words(3, 64) == 28
    for heads, size in ((0, 128), (8, 0), (8, 12), (8, 264)):
        assert lib.lmcb_kv4_row_words(heads, size) == 0
        with pytest.raises(RuntimeError):
            c_ops.kv4_row_words(heads, size)
    assert c_ops.kv4_row_words(8, 256) == 264


@pytest.mark.parametrize("kw,status", [
    (dict(type=INT32), abi.LMCB_ERR_UNSUPPORTED_DTYPE),
    (dict(slot_type=FP16), abi.LMCB_ERR_UNSUPPORTED_DTYPE),
    (dict(d=100), abi.LMCB_ERR_INVALID_ARGUMENT),
    (dict(d=264), abi.LMCB_ERR_INVALID_ARGUMENT),
    (dict(ks=1023), abi.LMCB_ERR_INVALID_ARGUMENT),
    (dict(blocks=1 << 28), abi.LMCB_ERR_INVALID_ARGUMENT),
    (dict(tokens=-1), abi.LMCB_ERR_INVALID_ARGUMENT),
    (dict(cache=None), abi.LMCB_ERR_INVALID_ARGUMENT),
    (dict(k=None), abi.LMCB_ERR_INVALID_ARGUMENT),
    (dict(slots=None), abi.LMCB_ERR_INVALID_ARGUMENT),
])
def test_kv4_rows_refuse(kw, status):
    a = dict(k=P, v=P, type=BF16, ks=1024, vs=1024, cache=P, blocks=8, bs=16, slots=P,
             slot_type=INT64, tokens=8, heads=8, d=128)
    a.update(kw)
    refused("lmcb_kv4_store", status, *a.values(), 0)
    refused("lmcb_kv4_load", status, a["cache"], a["blocks"], a["bs"], a["slots"], a["slot_type"],
            a["k"], a["v"], a["type"], a["ks"], a["vs"], a["tokens"], a["heads"], a["d"], 0)


def attn_args(**kw):
    a = dict(q=P, type=BF16, qs=1024, rows=4, cache=P, blocks=64, bs=16, table=P, ts=16, cols=16,
             lens=P, starts=None, batch=4, maxq=1, maxlen=256, hkv=2, hq=8, d=128, scale=0.1,
             window=0, sinks=0, out=P, os=1024, work=P, workbytes=1 << 30)
    a.update(kw)
    return list(a.values()) + [0]


@pytest.mark.parametrize("kw,status", [
    (dict(type=FP32), abi.LMCB_ERR_UNSUPPORTED_DTYPE),
    (dict(d=96), abi.LMCB_ERR_INVALID_ARGUMENT),
    (dict(hq=9), abi.LMCB_ERR_INVALID_ARGUMENT),
    (dict(hkv=0), abi.LMCB_ERR_INVALID_ARGUMENT),
    (dict(window=-1), abi.LMCB_ERR_INVALID_ARGUMENT),
    (dict(sinks=-1), abi.LMCB_ERR_INVALID_ARGUMENT),
    (dict(rows=3), abi.LMCB_ERR_INVALID_ARGUMENT),     # fewer rows than requests
    (dict(maxq=0), abi.LMCB_ERR_INVALID_ARGUMENT),
    (dict(qs=1023), abi.LMCB_ERR_INVALID_ARGUMENT),
    (dict(os=1023), abi.LMCB_ERR_INVALID_ARGUMENT),
    (dict(ts=15), abi.LMCB_ERR_INVALID_ARGUMENT),
    (dict(blocks=1 << 28), abi.LMCB_ERR_INVALID_ARGUMENT),
    (dict(cols=1 << 28, ts=1 << 28), abi.LMCB_ERR_INVALID_ARGUMENT),
    (dict(batch=4097, rows=4097), abi.LMCB_ERR_CAPACITY),
    (dict(batch=4096, rows=4096, cols=1 << 20, ts=1 << 20), abi.LMCB_ERR_CAPACITY),
    (dict(q=None), abi.LMCB_ERR_INVALID_ARGUMENT),
    (dict(lens=None), abi.LMCB_ERR_INVALID_ARGUMENT),
    (dict(cache=P + 4), abi.LMCB_ERR_INVALID_ARGUMENT),
    (dict(maxlen=1 << 14, work=None), abi.LMCB_ERR_CAPACITY),
    (dict(maxlen=1 << 14, work=P + 8), abi.LMCB_ERR_CAPACITY),
    (dict(maxlen=1 << 14, workbytes=64), abi.LMCB_ERR_CAPACITY),
])
def test_kv4_attention_refuses(kw, status):
    refused("lmcb_kv4_attention", status, *attn_args(**kw))


def test_workspace_size():
    n = ctypes.c_size_t(7)
    for batch, query, length in ((4, 1, 16), (4, 1, 1 << 20), (1, 8, 1 << 20), (1, 1, 0)):
        abi.call("lmcb_kv4_attention_workspace", batch, query, length, 8, 32, 128, 0, 0,
                 ctypes.byref(n))
        assert 0 < n.value < 64 << 20
    # no request, and units enough for every CTA: nothing is split
    for batch, query in ((0, 1), (64, 4096)):
        abi.call("lmcb_kv4_attention_workspace", batch, query, 1 << 20, 8, 32, 128, 0, 0,
                 ctypes.byref(n))
        assert n.value == 0
    refused("lmcb_kv4_attention_workspace", abi.LMCB_ERR_INVALID_ARGUMENT, 4, 1, 16, 8, 32, 100, 0,
            0, ctypes.byref(n))
    refused("lmcb_kv4_attention_workspace", abi.LMCB_ERR_INVALID_ARGUMENT, 4, 1, 16, 8, 32, 128, 0,
            0, None)


def test_c_ops_refuse_cpu_tensors():
    i32 = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        c_ops.build_slot_mapping(i32, i32, torch.zeros(2, 4, dtype=torch.int32), i32, 16,
                                 torch.zeros(4, dtype=torch.int64),
                                 torch.zeros(4, dtype=torch.int64), i32, i32, i32)
    x = torch.zeros(2, 2, 64)
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        c_ops.qk_norm_rope(x, x, None, None, i32, torch.zeros(8, 64), 1e-6, True, x, x)
    cache = torch.zeros(2, 1, 16, 1, 20, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        c_ops.kv4_store(x, x, cache, i32)
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        c_ops.kv4_load(cache, i32, x, x)
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        c_ops.kv4_attention(x, cache, i32.view(2, 1), i32, None, 1, 16, 2, 1.0, 0, 0, x)


def test_empty_calls_are_accepted():
    abi.call("lmcb_qk_norm_rope", *qk_args(tokens=0))
    abi.call("lmcb_kv4_store", None, None, BF16, 1024, 1024, None, 0, 16, None, INT64, 0, 8, 128, 0)
    abi.call("lmcb_kv4_attention", *attn_args(batch=0, rows=0))
