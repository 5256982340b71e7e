"""Lengths past the table: recorded by the plan, and the other requests of the batch
get what they would have got."""
import pytest
import torch

from q3vl import ops
from tests import ragged_oracle as ora

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16 = torch.bfloat16


@pytest.fixture(autouse=True)
def clean_error_word():
    ops.device_error(clear=True)
    yield
    assert ops.device_error(clear=True) == 0


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("with_free", [True, False])
def test_a_cached_length_past_the_table_is_recorded(with_free):
    """Also of a request that brings no token, whose kv_lens is clamped all the same."""
    free = i32([20, 21]) if with_free else None
    p = ops.ragged_plan(i32([0, 1]), i32([200, 10]), i32([[3], [8]]), page_tokens=64, n_tokens=2,
                        free_pages=free)
    assert ops.device_error() == 0x902
    assert p.kv_lens.tolist() == [64, 11] and p.slots.tolist() == [8 * 64 + 10, -1]
    p = ops.ragged_plan(i32([0, 1]), i32([64, 10]), i32([[3], [8]]), page_tokens=64, n_tokens=2,
                        free_pages=free)
    assert ops.device_error() == 0 and p.kv_lens.tolist() == [64, 11]


def test_the_other_requests_are_not_touched():
    Hq, Hkv, page, q_lens, past = 4, 2, 64, [70, 30, 1], [10, 20, 63]
    table = [[3], [8], [5]]
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(10, Hkv, page, 128, generator=g).to(BF16) for _ in range(2))
    q = torch.randn(101, Hq, 128, generator=g).to(BF16)
    p = ops.ragged_plan(i32(q_lens), i32(past), i32(table), page_tokens=page, n_tokens=101)
    assert ops.device_error() == 0x902
    assert p.cu_q.tolist() == [0, 70, 100, 101] and p.kv_lens.tolist() == [64, 50, 64]
    assert p.slots.tolist() == [3 * 64 + t if t < 64 else -1 for t in range(10, 80)] + \
        [8 * 64 + t for t in range(20, 50)] + [5 * 64 + 63]
    got = ops.attn_prefill_ragged(q.to(DEV), k.to(DEV), v.to(DEV), i32(table), p.cu_q, p.kv_lens)
    want, tol = ora.attention(q, k, v, table, [64, 50, 64], q_lens)
    ora.check("others", got[70:], want[70:], tol[70:])
    ora.check("the clamped one", got[:70], want[:70], tol[:70])
    dec = ops.attn_decode_ragged(q.to(DEV), k.to(DEV), v.to(DEV), i32(table[2:]), p.kv_lens[2:],
                                 cu_q=p.cu_q[2:])
    ora.check("decode", dec[100:], want[100:], tol[100:])
