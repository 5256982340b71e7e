"""Ragged serving operators on the host: refusals of the C ABI before anything
touches a device, the Python wrappers' refusals, and the plan's 64-bit form
against the page allocator's own tables."""
import ctypes

import pytest
import torch

from q3vl import _lib, ops
from q3vl.kv_pages import KVPagePool
from tests import ragged_oracle as ora

ONE = ctypes.c_void_p(16)
ODD = ctypes.c_void_p(18)


def refused(name, args, text, status=_lib.Q3_ERR_INVALID):
    rc = _lib.raw(name)(*args)
    msg = _lib.load().q3_last_error()
    assert rc == status, (name, rc, msg)
    assert text in msg, msg


def plan_args(**kw):
    a = dict(q=ONE, past=ONE, B=4, table=ONE, stride=8, width=8, page=64, free=ONE, n_free=3,
             delta=None, n=16, cu=ONE, kv=ONE, req=ONE, pos=ONE, slots=ONE, counts=ONE, s=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,text", [
    (dict(q=None), b"null"), (dict(counts=None), b"null"), (dict(slots=None), b"null"),
    (dict(B=-1), b"B=-1"), (dict(B=8193), b"8192"), (dict(n=-1), b"n_tokens"),
    (dict(n=1 << 31), b"n_tokens"), (dict(page=0), b"page_tokens"), (dict(page=96), b"page_tokens"),
    (dict(width=0), b"width"), (dict(stride=7), b"stride"), (dict(width=1 << 25, stride=1 << 25), b"32-bit"),
    (dict(free=None), b"free list"), (dict(n_free=-1), b"free list"), (dict(pos=ctypes.c_void_p(20)), b"misaligned")])
def test_plan_refusals(kw, text):
    refused("q3_ragged_plan", plan_args(**kw), text)


def rope_args(**kw):
    a = dict(qkv=ONE, qs=1536, qw=ONE, kw=ONE, pos=ONE, ax=0, inv=ONE, slots=ONE, out=ONE, os=1024,
             k=ONE, v=ONE, n=4, Hq=8, Hkv=2, d=128, page=64, pages=10, sh=20, sw=20, eps=1e-6, s=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,text", [
    (dict(d=64), b"head_dim"), (dict(n=-1), b"bad shape"), (dict(Hkv=0), b"bad shape"),
    (dict(qkv=None), b"null"), (dict(v=None), b"null"), (dict(qs=1528), b"strides"),
    (dict(qs=1540), b"multiples of 8"), (dict(os=1016), b"strides"), (dict(qkv=ODD), b"misaligned"),
    (dict(pages=1 << 26), b"32-bit"), (dict(sh=30), b"sections"), (dict(page=0), b"bad shape")])
def test_norm_rope_refusals(kw, text):
    refused("q3_qkv_norm_rope_ragged", rope_args(**kw), text)


def decode_args(**kw):
    a = dict(q=ONE, qs=1024, k=ONE, v=ONE, out=ONE, os=1024, B=4, Hq=8, Hkv=2, d=128, table=ONE,
             stride=8, width=8, page=64, pages=10, lens=ONE, scale=0.1, ws=ONE, nb=1 << 30, s=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,text", [
    (dict(d=64), b"head_dim"), (dict(B=-1), b"bad shape"), (dict(Hq=7), b"bad shape"),
    (dict(q=None), b"null"), (dict(ws=None), b"null"), (dict(page=32), b"page_tokens"),
    (dict(width=0), b"table width"), (dict(stride=4), b"stride"), (dict(pages=0), b"pages"),
    (dict(pages=1 << 25), b"too large"), (dict(qs=1000), b"strides"), (dict(os=1028), b"strides"),
    (dict(k=ODD), b"misaligned"), (dict(nb=100), b"workspace of 100")])
def test_decode_refusals(kw, text):
    refused("q3_attn_decode_ragged", decode_args(**kw), text)


def test_decode_refuses_more_than_16_heads_a_group():
    refused("q3_attn_decode_ragged", decode_args(Hq=34, qs=1 << 20, os=1 << 20), b"above 16",
            _lib.Q3_ERR_UNSUPPORTED)
    f = _lib.raw("q3_attn_decode_ragged_workspace_bytes")
    assert f(34, 2) == 0 and f(7, 2) == 0 and f(32, 8) > 0


def test_empty_calls_are_accepted_on_the_host():
    assert _lib.raw("q3_qkv_norm_rope_ragged")(*rope_args(n=0, qkv=None)) == 0
    assert _lib.raw("q3_attn_decode_ragged")(*decode_args(B=0, q=None)) == 0


def test_wrappers_refuse_cpu_tensors():
    t = torch.zeros(2, dtype=torch.int32)
    tab = torch.zeros(2, 4, dtype=torch.int32)
    pool = torch.zeros(4, 1, 64, 128, dtype=torch.bfloat16)
    x = torch.zeros(2, 4, 128, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.ragged_plan(t, t, tab, page_tokens=64, n_tokens=2)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.attn_decode_ragged(x, pool, pool, tab, t)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.qkv_norm_rope_ragged(x.view(2, -1), pool[0, 0, 0], pool[0, 0, 0], t.long(),
                                 torch.zeros(64), t.long(), pool, pool, Hq=2, Hkv=1)


def test_plan_form_hands_out_pages_as_the_allocator_does():
    """Growing slots 0..2 through the 64-bit form from the allocator's free order
    gives the allocator's own tables."""
    page, past, q = 64, [100, 0, 64], [30, 200, 1]
    pool = KVPagePool(32, page, max_seqs=3, buckets=())
    for b in range(3):
        pool.reserve(b, past[b])
    table = pool.table(range(3), 8).tolist()
    used = {p for r in table for p in r}
    free = [p for p in range(32) if p not in used]
    for b in range(3):
        pool.reserve(b, past[b] + q[b])
    want = pool.table(range(3), 8).tolist()
    ora.plan(q, past, table, page, sum(q), free)
    assert table == want
    pool.close()
