"""Rows of NaN through the ragged attentions on the GPU: a row is NaN whether its
keys are taken by one CTA or joined from pieces."""
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


# one request in one CTA; pieces on most SMs; the rows of many pieces by thread
@pytest.mark.parametrize("q_lens,pasts,Hq,Hkv", [
    ([3], [40], 4, 1), ([3], [17000], 4, 1), ([130, 300], [9000, 5000], 8, 2), ([200], [6000], 16, 1)])
def test_prefill_keeps_a_rows_nan(q_lens, pasts, Hq, Hkv):
    lens = [a + b for a, b in zip(q_lens, pasts)]
    k, v, table = mk.pool(lens, Hkv, 64, seed=2)
    q = torch.zeros(sum(q_lens), Hq, 128, dtype=BF16)
    q[1, 1, 5] = math.nan                                 # one value of one head's query
    q[2, 0, 0] = math.inf                                 # scores of both signs infinite
    got = ops.attn_prefill_ragged(q.to(DEV), k.to(DEV), v.to(DEV), i32(table),
                                  i32(cumsum(q_lens)), i32(lens)).cpu()
    seen = [p + i + 1 for m, p in zip(q_lens, pasts) for i in range(m)]
    want = mk.expected(seen, Hq, Hkv)
    for row, head in ((1, 1), (2, 0)):
        assert bool(got[row, head].isnan().all()), (row, head)
        got[row, head] = 0
        want[row, head] = 0
    ora.check("other rows", got, want, mk.bound(want))


@pytest.mark.parametrize("past", [40, 17000])
def test_prefill_keeps_the_nan_of_one_score(past):
    """A NaN key in the first tile, and last keys whose scores are so high that the
    first tile's weight is 0 in fp32."""
    L = past + 2
    k, v, table = mk.pool([L], 1, 64, seed=3)
    q = torch.full((2, 4, 128), 8.0, dtype=BF16)
    for j, pg in enumerate(table[0]):
        n = min(64, L - j * 64)
        k[pg, 0, :n] = 40.0 if j * 64 + n > L - 2 else -40.0
    k[table[0][0], 0, 7] = math.nan
    got = ops.attn_prefill_ragged(q.to(DEV), k.to(DEV), v.to(DEV), i32(table), i32([0, 2]), i32([L]))
    assert bool(got.isnan().all())
    dec = ops.attn_decode_ragged(q[:1].to(DEV), k.to(DEV), v.to(DEV), i32(table), i32([L]))
    assert bool(dec.isnan().all())
