"""Rows all of whose scores pass fp32's lowest value, through the ragged attentions
on the GPU: such keys count for nothing, so the rows are zeros, as a row that sees
no key, whether one CTA takes them or pieces are joined."""
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


def rows(n, Hq, G):
    """Query rows of head 0 (of each G) with scores of -1e40 against keys of -1e20,
    of head 1 with zeros, and NaN in one value of head 2."""
    q = torch.zeros(n, Hq, 128, dtype=BF16)
    q[:, 0::G] = 1e20
    q[:, 2::G, 9] = float("nan")
    return q


def check(got, seen, Hq, Hkv, G):
    got, want = got.cpu(), mk.expected(seen, Hq, Hkv)
    some = torch.tensor(seen) > 0
    assert bool(got[some][:, 2::G].isnan().all()) and not bool(got[:, 0::G].any())
    got[:, 2::G] = 0
    want[:, 0::G] = 0
    want[:, 2::G] = 0
    ora.check("other rows", got, want, mk.bound(want))


@pytest.mark.parametrize("lens,Hq,Hkv", [
    ([64], 4, 1), ([1, 64, 3], 8, 2),                    # whole pairs
    ([700], 4, 1), ([30000], 4, 1),                      # few pieces; many, joined by dims
    ([3000] * 30, 3, 1), ([5000, 0, 77], 24, 2), ([20000], 16, 1)])
def test_decode(lens, Hq, Hkv):
    G = Hq // Hkv
    k, v, table = mk.pool(lens, Hkv, 64, seed=6)
    live = ~k.isnan()
    k[live] = -1e20
    got = ops.attn_decode_ragged(rows(len(lens), Hq, G).to(DEV), k.to(DEV), v.to(DEV), i32(table),
                                 i32(lens))
    check(got, lens, Hq, Hkv, G)


@pytest.mark.parametrize("q_lens,pasts,Hq,Hkv", [
    ([3], [40], 4, 1), ([3], [17000], 4, 1), ([130, 300], [9000, 5000], 8, 2), ([200], [6000], 16, 1)])
def test_prefill(q_lens, pasts, Hq, Hkv):
    G = Hq // Hkv
    lens = [a + b for a, b in zip(q_lens, pasts)]
    k, v, table = mk.pool(lens, Hkv, 64, seed=6)
    live = ~k.isnan()
    k[live] = -1e20
    got = ops.attn_prefill_ragged(rows(sum(q_lens), Hq, G).to(DEV), k.to(DEV), v.to(DEV),
                                  i32(table), i32(cumsum(q_lens)), i32(lens))
    check(got, [p + i + 1 for m, p in zip(q_lens, pasts) for i in range(m)], Hq, Hkv, G)
