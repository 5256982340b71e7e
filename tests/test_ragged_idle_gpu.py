"""Steps in which a request of the decoding part brings no token: its neighbours
keep their own queries, through one call and through a captured step."""
import math

import pytest
import torch

from q3vl import ops
from tests import ragged_oracle as ora

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16 = torch.bfloat16
INV = 1.0 / (5e6 ** (torch.arange(0, 128, 2, dtype=torch.float32) / 128))


@pytest.fixture(autouse=True)
def clean_error_word():
    ops.device_error(clear=True)
    yield
    assert ops.device_error(clear=True) == 0


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def rnd(*shape, seed=0, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * std).to(BF16)


def cumsum(q_lens):
    cu = [0]
    for x in q_lens:
        cu.append(cu[-1] + x)
    return cu


@pytest.mark.parametrize("q_lens,lens,Hq,Hkv,page", [
    ([0, 1, 1, 0, 1], [700, 64, 0, 300, 5000], 4, 1, 64), ([0], [90], 4, 1, 64), ([0, 0, 1], [9, 9, 1], 8, 2, 64),
    ([1, 0] * 150, [5, 77] * 150, 8, 2, 64), ([0] * 40 + [1] + [0] * 40 + [1], [300] * 40 + [9000] + [0] * 40 + [65], 24, 2, 128),
    ([1, 0, 1], [30000, 20000, 1], 4, 1, 256), ([0, 1] * 20, [3000] * 40, 3, 1, 192)])
def test_decode_takes_the_rows_of_cu_q(q_lens, lens, Hq, Hkv, page):
    n, first = sum(q_lens), 3                       # three rows before the first request's
    k, v, table = ora.make_pool(lens, Hkv, page, seed=len(lens), stale=math.nan)
    q = rnd(n, Hq, 128, seed=4, std=1.5)
    want, tol = ora.attention(q, k, v, table, [x if m else 0 for x, m in zip(lens, q_lens)], q_lens)
    rows = torch.full((first + n + 2, Hq + 2, 128), math.nan, dtype=BF16, device=DEV)
    rows[first:first + n, :Hq] = q.to(DEV)
    out = torch.full((first + n + 2, Hq + 1, 128), 9.0, dtype=BF16, device=DEV)
    cu = i32([first + x for x in cumsum(q_lens)])
    pools = (k.to(DEV), v.to(DEV), i32(table))
    got = ops.attn_decode_ragged(rows[:, :Hq], *pools, i32(lens), cu_q=cu, out=out[:, :Hq])
    ora.check("decode", got[first:first + n], want, tol)
    assert bool((out[:first] == 9).all()) and bool((out[first + n:] == 9).all())
    assert bool((out[:, Hq] == 9).all())
    if all(q_lens):
        assert torch.equal(got[first:first + n], ops.attn_decode_ragged(q.to(DEV), *pools, i32(lens)))


def test_with_every_token_there_the_two_forms_are_one():
    lens = [329, 585, 0, 2048, 580, 1, 0, 153]
    k, v, table = ora.make_pool(lens, 8, 256, seed=1, stale=math.nan)
    q = rnd(8, 32, 128, seed=4)
    args = (q.to(DEV), k.to(DEV), v.to(DEV), i32(table), i32(lens))
    assert torch.equal(ops.attn_decode_ragged(*args),
                       ops.attn_decode_ragged(*args, cu_q=i32(list(range(9)))))
    # and in place of q
    buf = q.to(DEV)
    ops.attn_decode_ragged(buf, *args[1:], cu_q=i32(list(range(9))), out=buf)
    assert torch.equal(buf, ops.attn_decode_ragged(*args))


def test_requests_that_are_not_one_token_are_left_out_and_recorded():
    lens, Hq, Hkv = [100, 80, 60], 4, 2
    k, v, table = ora.make_pool(lens, Hkv, 64, seed=2, stale=math.nan)
    q = rnd(4, Hq, 128, seed=4)
    args = (q.to(DEV), k.to(DEV), v.to(DEV), i32(table), i32(lens))
    want, tol = ora.attention(q[3:], k, v, table[2:], [60], [1])

    def run(cu, live):
        out = torch.full((4, Hq, 128), 9.0, dtype=BF16, device=DEV)
        ops.attn_decode_ragged(*args, cu_q=i32(cu), out=out)
        assert ops.device_error() == 0x925
        if live:
            ora.check("the third", out[3:], want, tol)
        assert bool((out[:3 if live else 4] == 9).all())
    run([0, 3, 3, 4], True)          # request 0 has three tokens
    run([-1, 3, 3, 4], True)                         # starts before the rows
    run([4, 5, 5, 6], False)                         # rows behind the last one
    run([3, 2, 2, 0], False)         # descending
    bad = ops.attn_decode_ragged
    with pytest.raises(ValueError):
        bad(*args, cu_q=i32([0, 1, 2]))
    with pytest.raises(TypeError):
        bad(*args, cu_q=i32([0, 1, 2, 3]).long())
    with pytest.raises(RuntimeError):
        bad(*args, cu_q=torch.tensor([0, 1, 2, 3], dtype=torch.int32))


def test_a_captured_step_with_slots_that_go_idle_and_come_back():
    """plan -> norm + rotary + slots -> decode of slots 0..2 -> prefill of slot 3,
    captured once and replayed with other token counts."""
    B, d, n, Hq, Hkv, page, W = 4, 3, 40, 8, 2, 64, 6
    width = (Hq + 2 * Hkv) * 128
    qw, kw = 1 + rnd(128, seed=1, std=0.2), 1 + rnd(128, seed=2, std=0.2)
    dqw, dkw, inv = qw.to(DEV), kw.to(DEV), INV.to(DEV)
    kp, vp = rnd(24, Hkv, page, 128, seed=3).to(DEV), rnd(24, Hkv, page, 128, seed=4).to(DEV)
    ref = [[3] + [-1] * 5, [5, 6] + [-1] * 4, [7] + [-1] * 5, [-1] * 6]
    free, lens = [20, 21, 22, 23, 0, 1, 2, 9], [62, 128, 1, 0]
    table, dfree, start, past = i32(ref), i32(free), i32([0]), i32(lens)
    q_lens = i32([1, 1, 1, 0])
    x = torch.zeros(n, width, dtype=BF16, device=DEV)
    out = torch.zeros(n, Hq, 128, dtype=BF16, device=DEV)

    def step():
        p = ops.ragged_plan(q_lens, past, table, page_tokens=page, n_tokens=n, free_pages=dfree,
                            free_start=start)
        q = ops.qkv_norm_rope_ragged(x, dqw, dkw, p.positions, inv, p.slots, kp, vp, Hq=Hq, Hkv=Hkv)
        ops.attn_decode_ragged(q, kp, vp, table[:d], p.kv_lens[:d], cu_q=p.cu_q[:d + 1], out=out)
        ops.attn_prefill_ragged(q, kp, vp, table[d:], p.cu_q[d:], p.kv_lens[d:], out=out)
        past.copy_(p.kv_lens)
        start.add_(p.counts[1:])
        return q
    keep = [t.clone() for t in (past, start, table, kp, vp)]
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        step()
    torch.cuda.synchronize()
    for t, old in zip((past, start, table, kp, vp), keep):
        t.copy_(old)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        q = step()
    left = list(free)
    for i, counts in enumerate([[1, 1, 1, 0], [1, 0, 1, 17], [0, 0, 1, 1], [0, 0, 0, 0], [0, 1, 0, 37],
                                [1, 1, 0, 1], [1, 1, 1, 5]]):
        q_lens.copy_(i32(counts))
        x.copy_(rnd(n, width, seed=500 + i))
        out.fill_(3.0)
        g.replay()
        *_, took = ora.plan(counts, lens, ref, page, n, left)
        del left[:took[1]]
        lens = [a + b for a, b in zip(lens, counts)]
        assert past.tolist() == lens and table.tolist() == ref
        m = sum(counts)
        want, tol = ora.attention(q[:m].cpu(), kp.cpu(), vp.cpu(), ref,
                                  [a if b else 0 for a, b in zip(lens, counts)], counts)
        ora.check(f"step {i}", out[:m], want, tol)
        assert bool((out[m:] == 3).all())
