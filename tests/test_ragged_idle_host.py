"""Decode over packed rows: refusals on the host, before anything touches a device."""
import ctypes

import pytest
import torch

from q3vl import _lib, ops

ONE, ODD = ctypes.c_void_p(16), ctypes.c_void_p(18)


def args(**kw):
    a = dict(q=ONE, qs=1024, k=ONE, v=ONE, out=ONE, os=1024, n=9, B=4, Hq=8, Hkv=2, d=128, table=ONE,
             stride=8, width=8, page=64, pages=10, cu=ONE, lens=ONE, scale=0.1, ws=ONE, nb=1 << 30,
             s=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,text", [
    (dict(cu=None), b"cu_q"), (dict(cu=ODD), b"cu_q"), (dict(n=-1), b"n_tokens"),
    (dict(n=1 << 30), b"n_tokens"), (dict(n=1 << 31, Hkv=1), b"n_tokens"), (dict(d=64), b"head_dim"),
    (dict(B=-1), b"bad shape"), (dict(Hkv=0), b"bad shape"), (dict(q=None), b"null"),
    (dict(lens=None), b"null"), (dict(page=96), b"page_tokens"), (dict(qs=1000), b"strides"),
    (dict(nb=100), b"workspace of 100")])
def test_refusals(kw, text):
    rc = _lib.raw("q3_attn_decode_ragged_packed")(*args(**kw))
    msg = _lib.load().q3_last_error()
    assert rc == _lib.Q3_ERR_INVALID and text in msg, (rc, msg)


def test_empty_calls_are_accepted():
    assert _lib.raw("q3_attn_decode_ragged_packed")(*args(B=0, cu=None, q=None)) == 0
    assert _lib.raw("q3_attn_decode_ragged_packed")(*args(n=0, cu=None, q=None)) == 0


def test_the_wrapper_refuses_cpu_tensors():
    pool = torch.zeros(4, 1, 64, 128, dtype=torch.bfloat16)
    t = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.attn_decode_ragged(torch.zeros(2, 4, 128, dtype=torch.bfloat16), pool, pool,
                               torch.zeros(2, 4, dtype=torch.int32), t,
                               cu_q=torch.zeros(3, dtype=torch.int32))
