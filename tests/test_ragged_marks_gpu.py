"""Ragged attentions on the GPU: every key counted at long lengths, and prefill
batches of more requests than a CTA has threads."""
import math

import pytest
import torch

from q3vl import ops
from tests import ragged_marks as mk
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


def cumsum(q_lens):
    cu = [0]
    for x in q_lens:
        cu.append(cu[-1] + x)
    return cu


# ------------------------------------------------------- every key is counted
@pytest.mark.parametrize("lens,Hq,Hkv,page", [
    ([30000], 4, 1, 256), ([3] * 17 + [20000], 1, 1, 128), ([7000, 1, 9000], 16, 2, 64),
    ([9000, 100, 0, 2500], 12, 1, 64), ([32768, 257, 12345, 700], 32, 8, 256),
    ([0] * 40 + [3000] + [0] * 40 + [1], 8, 4, 64), ([1152] * 40, 4, 1, 64), ([2049] * 150, 9, 1, 192),
    ([5, 0, 64, 65, 6000] * 70, 8, 2, 64)])
def test_decode_counts_every_key(lens, Hq, Hkv, page):
    k, v, table = mk.pool(lens, Hkv, page, seed=len(lens))
    q = torch.zeros(len(lens), Hq, 128, dtype=BF16, device=DEV)
    got = ops.attn_decode_ragged(q, k.to(DEV), v.to(DEV), i32(table), i32(lens))
    want = mk.expected(lens, Hq, Hkv)
    ora.check("decode", got, want, mk.bound(want))


@pytest.mark.parametrize("q_lens,pasts,Hq,Hkv,page", [
    ([9], [17000], 8, 1, 128), ([1, 2], [9000, 4000], 4, 1, 64), ([31, 260], [5000, 1778], 6, 1, 256),
    ([16], [12345], 16, 1, 192), ([512], [32256], 32, 8, 256), ([1], [30000], 4, 1, 256),
    ([4096, 1100, 2, 1733], [0, 64, 8000, 5], 8, 2, 256), ([300, 0, 1, 77], [20000, 4, 11111, 0], 1, 1, 64)])
@pytest.mark.parametrize("causal", [True, False])
def test_prefill_counts_every_key(q_lens, pasts, Hq, Hkv, page, causal):
    lens = [a + b for a, b in zip(q_lens, pasts)]
    k, v, table = mk.pool(lens, Hkv, page, seed=len(lens))
    q = torch.zeros(sum(q_lens), Hq, 128, dtype=BF16, device=DEV)
    got = ops.attn_prefill_ragged(q, k.to(DEV), v.to(DEV), i32(table), i32(cumsum(q_lens)), i32(lens),
                                  causal=causal)
    seen = [p + i + 1 if causal else n for m, p, n in zip(q_lens, pasts, lens) for i in range(m)]
    want = mk.expected(seen, Hq, Hkv)
    ora.check("prefill", got, want, mk.bound(want))


# ------------------------------- more requests than a prefill CTA has threads
@pytest.mark.parametrize("B,Hq,Hkv", [(384, 4, 1), (385, 4, 2), (400, 8, 2), (1000, 4, 1)])
@pytest.mark.parametrize("causal", [True, False])
def test_prefill_of_many_requests(B, Hq, Hkv, causal):
    g = torch.Generator().manual_seed(B)
    some = [0, 1, 1, 2, 5, 33, 130]
    q_lens = [some[int(i)] for i in torch.randint(0, len(some), (B,), generator=g)]
    for a, b in ((0, 37), (B // 2, B // 2 + 95), (B - 41, B - 1)):     # runs of empty requests
        q_lens[a:b] = [0] * (b - a)
    q_lens[B // 3], q_lens[B // 2 + 95], q_lens[-1] = 300, 7, 3
    pasts = torch.randint(0, 150, (B,), generator=g).tolist()
    pasts[B // 3], pasts[B // 4] = 900, 2500
    lens = [a + b for a, b in zip(q_lens, pasts)]
    k, v, table = ora.make_pool(lens, Hkv, 64, seed=B, stale=math.nan)
    q = torch.randn(sum(q_lens), Hq, 128, generator=g).to(BF16)
    want, tol = ora.attention(q, k, v, table, lens, q_lens, causal=causal)
    args = (q.to(DEV), k.to(DEV), v.to(DEV), i32(table), i32(cumsum(q_lens)), i32(lens))
    got = ops.attn_prefill_ragged(*args, causal=causal)
    ora.check("prefill", got, want, tol)
    assert torch.equal(got, ops.attn_prefill_ragged(*args, causal=causal))
