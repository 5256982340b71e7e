"""Ragged serving operators on the GPU against their 64-bit forms: plan, norm +
rotary + slots, decode attention; sizes and lengths at tile and page borders,
padding, stale NaN rows, strides, bad entries, graphs and streams."""
import math

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


def rnd(*shape, seed=0, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * std).to(BF16)


# ------------------------------------------------------------------ the plan
PLANS = [
    ([1] * 8, [384, 1998, 116, 1596, 1772, 8, 1824, 0], 256, 0),
    ([0], [0], 64, 3),
    ([1], [63], 64, 0),
    ([1], [64], 64, 0),
    ([65, 0, 1, 128, 0, 64], [0, 5, 63, 64, 0, 1], 64, 37),
    ([3] * 600, list(range(600)), 64, 1),               # more requests than threads
    ([700, 1, 0, 2500], [190, 191, 192, 193], 192, 130),
]


@pytest.mark.parametrize("q,past,page,pad", PLANS)
@pytest.mark.parametrize("with_free", [True, False])
def test_plan(q, past, page, pad, with_free):
    B = len(q)
    W = max(1, max(-(-(a + b) // page) for a, b in zip(q, past))) + 1
    g = torch.Generator().manual_seed(B)
    ids = torch.randperm(B * W + 3, generator=g).tolist()
    table = []
    for b in range(B):
        n = -(-past[b] // page) if with_free else -(-(past[b] + q[b]) // page)
        table.append([ids.pop() for _ in range(n)] + [-1] * (W - n))
    delta = torch.randint(-900, 900, (B, 1), generator=g).tolist()
    n_tok = sum(q) + pad
    want_table = [list(r) for r in table]
    want = ora.plan(q, past, want_table, page, n_tok, ids if with_free else None,
                    [d[0] for d in delta])
    # the table as a view into a wider one, with its other columns untouched
    wide = torch.full((B, W + 5), -7, dtype=torch.int32, device=DEV)
    wide[:, :W] = i32(table)
    got = ops.ragged_plan(i32(q), i32(past), wide[:, :W], page_tokens=page, n_tokens=n_tok,
                          free_pages=i32(ids) if with_free else None,
                          rope_delta=torch.tensor(delta, device=DEV))
    for name, x in zip(("cu_q", "kv_lens", "requests", "positions", "slots", "counts"), want):
        assert getattr(got, name).tolist() == x, name
    assert wide[:, :W].tolist() == want_table
    assert bool((wide[:, W:] == -7).all())


def test_plan_at_the_largest_batch_and_with_no_request():
    B = 8192
    q = [b % 3 for b in range(B)]
    past = [(7 * b) % 130 for b in range(B)]
    table = [[-1] * 4 for _ in range(B)]
    ids = list(range(B * 4, 0, -1))
    for b in range(B):
        for j in range(-(-past[b] // 64)):
            table[b][j] = ids.pop()
    want_table = [list(r) for r in table]
    want = ora.plan(q, past, want_table, 64, sum(q), ids)
    t = i32(table)
    got = ops.ragged_plan(i32(q), i32(past), t, page_tokens=64, n_tokens=sum(q), free_pages=i32(ids))
    for name, x in zip(got._fields, want):
        assert getattr(got, name).tolist() == x, name
    assert t.tolist() == want_table
    none = torch.empty(0, dtype=torch.int32, device=DEV)
    got = ops.ragged_plan(none, none, torch.empty(0, 4, dtype=torch.int32, device=DEV),
                          page_tokens=64, n_tokens=5)
    assert got.cu_q.tolist() == [0] and got.slots.tolist() == [-1] * 5
    assert got.counts.tolist() == [0, 0]


def test_plan_records_what_does_not_fit():
    t = i32([[4, -1], [5, -1]])
    # the free list is one page short: request 1's new page is missing
    p = ops.ragged_plan(i32([64, 64]), i32([64, 60]), t, page_tokens=64, n_tokens=128,
                        free_pages=i32([9]))
    assert ops.device_error() == 0x903
    assert p.counts.tolist() == [128, 2] and t.tolist() == [[4, 9], [5, -1]]
    assert p.slots.tolist() == [9 * 64 + i for i in range(64)] + \
        [5 * 64 + i for i in range(60, 64)] + [-1] * 60
    # a table that does not map a position; a position past the table
    p = ops.ragged_plan(i32([2]), i32([63]), i32([[3, -1]]), page_tokens=64, n_tokens=2)
    assert ops.device_error() == 0x903 and p.slots.tolist() == [3 * 64 + 63, -1]
    p = ops.ragged_plan(i32([3]), i32([126]), i32([[3, 8]]), page_tokens=64, n_tokens=3)
    assert ops.device_error() == 0x902
    assert p.slots.tolist() == [8 * 64 + 62, 8 * 64 + 63, -1] and p.kv_lens.tolist() == [128]
    # more tokens than the packed buffer; a negative length
    p = ops.ragged_plan(i32([3, 3]), i32([0, 0]), i32([[3], [8]]), page_tokens=64, n_tokens=4)
    assert ops.device_error() == 0x904
    assert p.cu_q.tolist() == [0, 3, 4] and p.kv_lens.tolist() == [3, 1]
    p = ops.ragged_plan(i32([-5, 2]), i32([0, 1]), i32([[3], [8]]), page_tokens=64, n_tokens=2)
    assert ops.device_error() == 0x901
    assert p.cu_q.tolist() == [0, 0, 2] and p.slots.tolist() == [8 * 64 + 1, 8 * 64 + 2]


# -------------------------------------------------- norm, rotary, K/V to slots
INV = 1.0 / (5e6 ** (torch.arange(0, 128, 2, dtype=torch.float32) / 128))


@pytest.mark.parametrize("n,Hq,Hkv,axes,page,pad", [
    (1, 32, 8, 1, 256, 0), (8, 4, 1, 3, 64, 0), (3, 1, 1, 1, 64, 1), (129, 5, 1, 3, 192, 19),
    (700, 32, 8, 3, 256, 3), (1037, 6, 2, 3, 64, 0), (2, 40, 8, 3, 64, 2),
    (5, 128, 64, 1, 64, 0), (3000, 2, 1, 3, 64, 7)])
def test_norm_rope_slots(n, Hq, Hkv, axes, page, pad):
    width = (Hq + 2 * Hkv) * 128
    pages = -(-n // page) + 1
    qkv = rnd(n, width, seed=n)
    qw, kw = 1 + rnd(128, seed=1, std=0.2), 1 + rnd(128, seed=2, std=0.2)
    g = torch.Generator().manual_seed(3)
    pos = torch.randint(0, 1 << 20, (axes, n), generator=g)
    pos[:, 0] = torch.tensor([0, 1, 2 ** 31 + 5])[:axes]       # near zero, and past 32 bits
    pos = pos[0] if axes == 1 else pos
    slots = torch.randperm(pages * page, generator=g)[:n]
    if pad:
        slots[torch.randperm(n, generator=g)[:pad]] = -1
        qkv[slots < 0] = math.nan
    k0 = rnd(pages, Hkv, page, 128, seed=4)
    v0 = rnd(pages, Hkv, page, 128, seed=5)
    # qkv as columns of a wider buffer, q into one with a guard behind each row
    wide = torch.full((n, width + 64), math.nan, dtype=BF16, device=DEV)
    wide[:, :width] = qkv.to(DEV)
    guard = torch.full((n, Hq + 1, 128), 77.0, dtype=BF16, device=DEV)
    k, v = k0.to(DEV), v0.to(DEV)
    q = ops.qkv_norm_rope_ragged(wide[:, :width], qw.to(DEV), kw.to(DEV), pos.to(DEV),
                                 INV.to(DEV), slots.to(DEV), k, v, Hq=Hq, Hkv=Hkv,
                                 out=guard[:, :Hq])
    wq, wk, wv, tq, tk = ora.norm_rope(torch.nan_to_num(qkv), qw, kw, pos, INV, Hq, Hkv)
    live = slots >= 0
    ora.check("q", q.cpu()[live], wq[live], tq[live])
    assert bool((guard[:, Hq] == 77).all())
    assert bool((q.cpu()[~live] == 77).all())                   # padding rows left as they were
    want_k, tol_k = k0.double(), torch.zeros(k0.shape, dtype=torch.float64)
    want_v = v0.clone()
    s = slots[live]
    want_k[s // page, :, s % page] = wk[live]
    tol_k[s // page, :, s % page] = tk[live]
    want_v[s // page, :, s % page] = wv[live].to(BF16)
    ora.check("k", k, want_k, tol_k)
    assert torch.equal(v.cpu(), want_v)


def test_norm_rope_equals_the_table_kernel_within_its_roundings():
    """Against q3_qkv_norm_rope at text positions: that kernel rounds cos, sin, n
    and both products to bf16, four half steps on values up to |a| + |b|."""
    n, Hq, Hkv = 40, 8, 2
    qkv = rnd(n, (Hq + 2 * Hkv) * 128, seed=8)
    qw, kw = 1 + rnd(128, seed=1, std=0.2), 1 + rnd(128, seed=2, std=0.2)
    t = torch.arange(n, dtype=torch.float64)[:, None] * INV.double()
    k = torch.zeros(1, Hkv, 64, 128, dtype=BF16, device=DEV)
    v = torch.zeros_like(k)
    old, _, _ = ops.qkv_norm_rope(qkv.to(DEV), qw.to(DEV), kw.to(DEV), t.cos().to(BF16).to(DEV),
                                  t.sin().to(BF16).to(DEV), B=1, S=n, Hq=Hq, Hkv=Hkv)
    q = ops.qkv_norm_rope_ragged(qkv.to(DEV), qw.to(DEV), kw.to(DEV),
                                 torch.arange(n, device=DEV), INV.to(DEV),
                                 torch.arange(n, device=DEV), k, v, Hq=Hq, Hkv=Hkv)
    _, _, _, tq, _ = ora.norm_rope(qkv, qw, kw, torch.arange(n), INV, Hq, Hkv)
    y = old[0].transpose(0, 1).double().cpu()
    x = qkv.double().view(n, -1, 128)[:, :Hq]
    m = (x / (x.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * qw.double()).abs()
    mag = (m[..., :64] + m[..., 64:]).repeat(1, 1, 2)
    ora.check("q", q, y, tq + 6 * ora.BF16_HALF * mag)


def test_norm_rope_records_a_slot_outside_the_pool():
    n, Hq, Hkv = 3, 2, 1
    qkv = rnd(n, 4 * 128).to(DEV)
    w = torch.ones(128, dtype=BF16, device=DEV)
    k = torch.zeros(2, 1, 64, 128, dtype=BF16, device=DEV)
    v = torch.zeros_like(k)
    out = torch.full((n, Hq, 128), 5.0, dtype=BF16, device=DEV)
    ops.qkv_norm_rope_ragged(qkv, w, w, torch.arange(n, device=DEV), INV.to(DEV),
                             torch.tensor([128, -2, 127], device=DEV), k, v, Hq=Hq, Hkv=Hkv, out=out)
    assert ops.device_error() == 0x911
    assert bool((out[:2] == 5).all()) and torch.equal(v[1, 0, 63], qkv[2, 3 * 128:])
    assert int((v != 0).any(-1).sum()) == 1
    q = ops.qkv_norm_rope_ragged(qkv[:0], w, w, torch.arange(0, device=DEV), INV.to(DEV),
                                 torch.arange(0, device=DEV), k, v, Hq=Hq, Hkv=Hkv)
    assert q.shape == (0, Hq, 128)


# ------------------------------------------------------------ decode attention
def decode_case(lens, Hq, Hkv, page, seed=0, stale=math.nan, std=1.5, **kw):
    k, v, table = ora.make_pool(lens, Hkv, page, seed=seed, stale=stale, **kw)
    q = rnd(len(lens), Hq, 128, seed=seed + 9, std=std)
    return q, k, v, table


@pytest.mark.parametrize("lens,Hq,Hkv,page", [
    ([1], 4, 1, 64), ([0], 4, 1, 64), ([700], 4, 1, 64), ([64], 1, 1, 64), ([65, 63], 2, 2, 64),
    ([329, 585, 0, 2048, 580, 1, 0, 153], 32, 8, 256),
    ([1000, 17], 3, 1, 192), ([130, 4097, 64], 10, 2, 128), ([257, 1], 16, 2, 64),
    ([1500, 66, 0], 16, 1, 64), ([900, 31], 24, 2, 256), ([40, 2000], 9, 1, 64),
    ([5] * 300, 8, 2, 64), ([0] * 40 + [3000] + [0] * 40 + [1], 8, 4, 64),
    ([30000], 4, 1, 256), ([0, 0, 0], 8, 2, 64), ([9000, 100, 0, 2500], 12, 1, 64),
    ([1100], 2, 1, 64), ([3] * 17 + [20000], 1, 1, 128), ([7000, 1, 9000], 16, 2, 64)])
def test_decode(lens, Hq, Hkv, page):
    q, k, v, table = decode_case(lens, Hq, Hkv, page, seed=len(lens))
    want, tol = ora.attention(q, k, v, table, lens, [1] * len(lens))
    got = ops.attn_decode_ragged(q.to(DEV), k.to(DEV), v.to(DEV), i32(table), i32(lens))
    ora.check("decode", got, want, tol)
    again = ops.attn_decode_ragged(q.to(DEV), k.to(DEV), v.to(DEV), i32(table), i32(lens))
    assert torch.equal(got, again)                       # the same order every time


def test_decode_matches_the_one_length_kernel():
    L, Hq, Hkv, page = 1152, 32, 8, 256
    q, k, v, table = decode_case([L] * 8, Hq, Hkv, page, stale=0.0)
    args = (q.to(DEV), k.to(DEV), v.to(DEV), i32(table))
    _, tol = ora.attention(q, k, v, table, [L] * 8, [1] * 8)
    old = ops.attn_decode_paged(*args, kv_len=L).double().cpu()
    ora.check("decode", ops.attn_decode_ragged(*args, i32([L] * 8)), old, 2 * tol)


def test_decode_strides_scale_guard_and_large_scores():
    lens, Hq, Hkv, page = [200, 0, 999], 8, 2, 64
    q, k, v, table = decode_case(lens, Hq, Hkv, page, seed=3, std=40.0)
    rows = torch.full((3, Hq + 2 * Hkv, 128), math.nan, dtype=BF16, device=DEV)
    rows[:, :Hq] = q.to(DEV)
    out = torch.full((3, Hq + 1, 128), 9.0, dtype=BF16, device=DEV)
    wide = torch.full((3, 40), -1, dtype=torch.int32, device=DEV)
    wide[:, :len(table[0])] = i32(table)
    for scale in (0.25, -0.1, 0.0):
        want, tol = ora.attention(q, k, v, table, lens, [1] * 3, scale=scale)
        _, pos = ora.attention(q, k, v, table, lens, [1] * 3, scale=abs(scale))
        got = ops.attn_decode_ragged(rows[:, :Hq], k.to(DEV), v.to(DEV), wide, i32(lens),
                                     scale=scale, out=out[:, :Hq])
        ora.check(f"scale {scale}", got, want, torch.maximum(tol, pos))
        assert bool((out[:, Hq] == 9).all())


def test_decode_clamps_bad_lengths_and_entries():
    lens, Hq, Hkv, page = [128, 100], 4, 2, 64
    q, k, v, table = decode_case(lens, Hq, Hkv, page, stale=0.0)
    dev = (q.to(DEV), k.to(DEV), v.to(DEV))
    got = ops.attn_decode_ragged(*dev, i32(table), i32([129, -1]))   # two pages hold 128
    assert ops.device_error() == 0x921
    want, tol = ora.attention(q, k, v, table, [128, 0], [1, 1])
    ora.check("clamped", got, want, tol)
    bad = [list(r) for r in table]
    bad[0][1], bad[1][0] = -1, k.shape[0]
    got = ops.attn_decode_ragged(*dev, i32(bad), i32(lens))
    assert ops.device_error() == 0x922
    bad[0][1] = bad[1][0] = 0
    want, tol = ora.attention(q, k, v, bad, lens, [1, 1])
    ora.check("page 0", got, want, tol)


def test_decode_in_a_graph_with_new_lengths_and_on_two_streams():
    Hq, Hkv, page = 8, 2, 64
    sets = [[700, 64, 0], [1, 900, 333]]
    q, k, v, table = decode_case([960] * 3, Hq, Hkv, page, stale=0.0)
    dq, dk, dv, dt, dl = q.to(DEV), k.to(DEV), v.to(DEV), i32(table), i32(sets[0])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ops.attn_decode_ragged(dq, dk, dv, dt, dl)
    torch.cuda.current_stream().wait_stream(s)
    graphs = []
    for _ in range(2):                                    # two graphs over the same inputs
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = ops.attn_decode_ragged(dq, dk, dv, dt, dl)
        graphs.append((g, o))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for lens in sets:
        dl.copy_(i32(lens))
        torch.cuda.synchronize()
        for _ in range(5):                                # both in flight at once
            for (g, _), st in zip(graphs, streams):
                with torch.cuda.stream(st):
                    g.replay()
        torch.cuda.synchronize()
        want, tol = ora.attention(q, k, v, table, lens, [1] * 3)
        for _, o in graphs:
            ora.check("replayed", o, want, tol)


# ----------------------------------------------------------- prefill attention
def prefill_case(q_lens, pasts, Hq, Hkv, page, seed=0, stale=math.nan, std=1.5):
    lens = [max(0, a + b) for a, b in zip(q_lens, pasts)]
    k, v, table = ora.make_pool(lens, Hkv, page, seed=seed, stale=stale)
    q = rnd(sum(q_lens), Hq, 128, seed=seed + 9, std=std)
    cu = [0]
    for x in q_lens:
        cu.append(cu[-1] + x)
    return q, k, v, table, cu, lens


@pytest.mark.parametrize("q_lens,pasts,Hq,Hkv,page", [
    ([1], [0], 4, 1, 64), ([128], [0], 1, 1, 64), ([5, 0, 70], [0, 64, 63], 4, 1, 64),
    ([26, 46, 28, 100], [0] * 4, 4, 1, 64), ([257], [0], 2, 2, 192), ([300, 1], [5, 900], 3, 1, 64),
    ([130], [1000], 32, 8, 256), ([64, 65], [64, 4032], 10, 2, 128), ([33], [3000], 16, 1, 64),
    ([70, 2], [1, 0], 12, 1, 64), ([515], [0], 14, 2, 64), ([1] * 70, list(range(70)), 8, 4, 64),
    ([700], [0], 8, 1, 64), ([9, 40], [-4, -40], 4, 2, 64)])
@pytest.mark.parametrize("causal", [True, False])
def test_prefill(q_lens, pasts, Hq, Hkv, page, causal):
    q, k, v, table, cu, lens = prefill_case(q_lens, pasts, Hq, Hkv, page, seed=len(q_lens))
    want, tol = ora.attention(q, k, v, table, lens, q_lens, causal=causal)
    args = (q.to(DEV), k.to(DEV), v.to(DEV), i32(table), i32(cu), i32(lens))
    got = ops.attn_prefill_ragged(*args, causal=causal)
    ora.check("prefill", got, want, tol)
    assert torch.equal(got, ops.attn_prefill_ragged(*args, causal=causal))


@pytest.mark.parametrize("q_lens,pasts,Hq,Hkv,page", [
    ([9], [17000], 8, 1, 128), ([1, 2], [9000, 4000], 4, 1, 64), ([31, 260], [5000, 1778], 6, 1, 256),
    ([16], [12345], 16, 1, 192)])
def test_prefill_of_few_rows_with_many_pieces(q_lens, pasts, Hq, Hkv, page):
    """One item cut over most SMs: the rows' bases rise from piece to piece."""
    q, k, v, table, cu, lens = prefill_case(q_lens, pasts, Hq, Hkv, page, seed=21)
    for b, n in enumerate(lens):                    # keys grow along the request
        for j in range(-(-n // page)):
            k[table[b][j]] *= 0.25 + 2.0 * j * page / n
    want, tol = ora.attention(q, k, v, table, lens, q_lens)
    args = (q.to(DEV), k.to(DEV), v.to(DEV), i32(table), i32(cu), i32(lens))
    got = ops.attn_prefill_ragged(*args)
    ora.check("prefill", got, want, tol)
    assert torch.equal(got, ops.attn_prefill_ragged(*args))


def test_prefill_matches_the_one_start_kernel():
    B, S, Hq, Hkv, page, start = 2, 300, 8, 2, 128, 128
    q, k, v, table, cu, lens = prefill_case([S] * B, [start] * B, Hq, Hkv, page, stale=0.0)
    _, tol = ora.attention(q, k, v, table, lens, [S] * B)
    dk, dv, dt = k.to(DEV), v.to(DEV), i32(table)
    qd = q.to(DEV)
    old = torch.empty(B, Hq, S, 128, dtype=BF16, device=DEV)
    ops.attn_prefill_tc_paged(qd.view(B, S, Hq, 128).transpose(1, 2).contiguous(), dk, dv, dt,
                              start_pos=start, causal=True, scale=1 / math.sqrt(128), out=old)
    got = ops.attn_prefill_ragged(qd, dk, dv, dt, i32(cu), i32(lens))
    ora.check("prefill", got, old.transpose(1, 2).reshape(B * S, Hq, 128).double().cpu(), 2 * tol)


def test_prefill_of_a_part_of_a_batch_leaves_other_rows():
    q_lens, pasts, Hq, Hkv, page = [1, 70, 133, 2], [600, 0, 50, 7], 8, 2, 64
    q, k, v, table, cu, lens = prefill_case(q_lens, pasts, Hq, Hkv, page, seed=4)
    rows = torch.full((q.shape[0] + 5, Hq + 2 * Hkv, 128), math.nan, dtype=BF16, device=DEV)
    rows[:q.shape[0], :Hq] = q.to(DEV)
    out = torch.full((q.shape[0] + 5, Hq + 1, 128), 9.0, dtype=BF16, device=DEV)
    want, tol = ora.attention(q, k, v, table, lens, q_lens)
    dc, dl, dt = i32(cu), i32(lens), i32(table)
    got = ops.attn_prefill_ragged(rows[:, :Hq], k.to(DEV), v.to(DEV), dt[1:3], dc[1:4], dl[1:3],
                                  out=out[:, :Hq])
    a, b = cu[1], cu[3]
    ora.check("part", got[a:b], want[a:b], tol[a:b])
    assert bool((out[:a] == 9).all()) and bool((out[b:] == 9).all())
    assert bool((out[:, Hq] == 9).all())


def test_prefill_of_rising_scores_rescales():
    """Keys whose scores grow along the cache move a row's base at every tile."""
    q, k, v, table, cu, lens = prefill_case([40], [1500], 4, 1, 64, stale=0.0)
    ramp = torch.linspace(0.0, 6.0, lens[0])
    for i, pg in enumerate(table[0]):
        n = min(64, lens[0] - i * 64)
        if n > 0:
            k[pg, 0, :n] = (ramp[i * 64:i * 64 + n, None] * torch.ones(128)).to(BF16)
    q = q.abs()
    want, tol = ora.attention(q, k, v, table, lens, [40], scale=1.0)
    got = ops.attn_prefill_ragged(q.to(DEV), k.to(DEV), v.to(DEV), i32(table), i32(cu), i32(lens),
                                  scale=1.0)
    ora.check("rising", got, want, tol)


def test_prefill_clamps_bad_lengths_and_entries():
    q, k, v, table, cu, lens = prefill_case([70, 30], [0, 60], 4, 2, 64, stale=0.0)
    dev = (q.to(DEV), k.to(DEV), v.to(DEV))
    # request 1's rows end past the packed buffer, and its length past its table
    got = ops.attn_prefill_ragged(*dev, i32(table), i32([0, 70, 130]), i32([70, 129]))
    assert ops.device_error() == 0x931
    want, tol = ora.attention(q, k, v, [table[0], table[1]], [70, 128], [70, 30])
    ora.check("clamped", got, want, tol)
    got = ops.attn_prefill_ragged(*dev, i32(table), i32([0, 70, 60]), i32([70, -1]))
    assert ops.device_error() == 0x931
    ora.check("none", got[:70], want[:70], tol[:70])
    bad = [list(r) for r in table]
    bad[0][1], bad[1][0] = -1, k.shape[0]
    got = ops.attn_prefill_ragged(*dev, i32(bad), i32(cu), i32(lens))
    assert ops.device_error() == 0x932
    bad[0][1] = bad[1][0] = 0
    want, tol = ora.attention(q, k, v, bad, lens, [70, 30])
    ora.check("page 0", got, want, tol)


def test_prefill_in_a_graph_with_new_lengths():
    Hq, Hkv, page, n = 8, 2, 64, 200
    sets = [([120, 80], [0, 500]), ([1, 150], [700, 3]), ([0, 0], [4, 0])]
    q, k, v, table, _, _ = prefill_case([100, 100], [800, 800], Hq, Hkv, page, stale=0.0)
    dq, dk, dv, dt = q.to(DEV), k.to(DEV), v.to(DEV), i32(table)
    dc, dl = i32([0, 0, 0]), i32([0, 0])
    out = torch.zeros_like(dq)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        ops.attn_prefill_ragged(dq, dk, dv, dt, dc, dl, out=out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.attn_prefill_ragged(dq, dk, dv, dt, dc, dl, out=out)
    for qs, ps in sets:
        lens = [a + b for a, b in zip(qs, ps)]
        dc.copy_(i32([0, qs[0], qs[0] + qs[1]]))
        dl.copy_(i32(lens))
        out.fill_(3.0)
        g.replay()
        torch.cuda.synchronize()
        m = sum(qs)
        want, tol = ora.attention(q[:m], k, v, table, lens, qs)
        ora.check("replayed", out[:m], want, tol)
        assert bool((out[m:] == 3).all())


# ------------------------------------------------------- the operators together
def test_scores_below_the_lowest_fp32_value():
    """Keys whose scores pass fp32 count for nothing, whole pieces of them too."""
    L, hidden, Hq, Hkv, page = 30000, 20032, 4, 1, 64
    q, k, v, table = decode_case([L], Hq, Hkv, page, seed=5)
    q.fill_(1e20)                                   # products of -1e40
    k[table[0][:hidden // page]] = -1e20
    for j, pg in enumerate(table[0][hidden // page:]):
        k[pg, :, :min(page, L - hidden - j * page)] = 0.0
    want, tol = ora.attention(q, k, v, [table[0][hidden // page:]], [L - hidden], [1])
    args = (q.to(DEV), k.to(DEV), v.to(DEV), i32(table))
    ora.check("decode", ops.attn_decode_ragged(*args, i32([L])), want, tol)
    ora.check("prefill", ops.attn_prefill_ragged(*args, i32([0, 1]), i32([L])), want, tol)
    # nothing but such keys and one plain one at the end
    want = v[table[0][hidden // page], :, :1].double().expand(1, Hq, 128)
    tol = 2 * ora.BF16_HALF * want.abs() + 1e-30
    ora.check("decode", ops.attn_decode_ragged(*args, i32([hidden + 1])), want, tol)


def test_results_in_place_of_q():
    q_lens, pasts, Hq, Hkv, page = [70, 1, 300], [5, 900, 64], 8, 2, 64
    q, k, v, table, cu, lens = prefill_case(q_lens, pasts, Hq, Hkv, page, seed=6)
    rest = (k.to(DEV), v.to(DEV), i32(table))
    buf = q.to(DEV)
    want = ops.attn_prefill_ragged(buf, *rest, i32(cu), i32(lens))
    got = ops.attn_prefill_ragged(buf, *rest, i32(cu), i32(lens), out=buf)
    assert got is buf and torch.equal(got, want)
    buf = q[:3].to(DEV)
    want = ops.attn_decode_ragged(buf, *rest, i32(lens))
    assert torch.equal(ops.attn_decode_ragged(buf, *rest, i32(lens), out=buf), want)
    # the q part of packed qkv rows, heads of a token shared by several warps
    Hq, Hkv = 32, 8
    qkv = rnd(9, (Hq + 2 * Hkv) * 128, seed=7).to(DEV)
    w = torch.ones(128, dtype=BF16, device=DEV)
    pools = torch.zeros(4, 1, Hkv, 64, 128, dtype=BF16, device=DEV)
    pos = torch.arange(9, device=DEV)
    args = (w, w, pos, INV.to(DEV), pos)
    want = ops.qkv_norm_rope_ragged(qkv, *args, pools[0], pools[1], Hq=Hq, Hkv=Hkv)
    part = qkv.view(9, Hq + 2 * Hkv, 128)[:, :Hq]
    ops.qkv_norm_rope_ragged(qkv, *args, pools[2], pools[3], Hq=Hq, Hkv=Hkv, out=part)
    assert torch.equal(part, want) and torch.equal(pools[:2], pools[2:])


def test_plan_continues_the_free_list():
    t = i32([[4, -1, -1], [5, -1, -1]])
    free, start = i32([9, 8, 7, 6]), i32([0])
    past = i32([64, 60])
    for step, taken in ((0, 2), (1, 0)):
        p = ops.ragged_plan(i32([1, 5]), past, t, page_tokens=64, n_tokens=6, free_pages=free,
                            free_start=start)
        assert p.counts.tolist() == [6, taken]
        past, start = p.kv_lens.clone(), start + p.counts[1:]
    assert t.tolist() == [[4, 9, -1], [5, 8, -1]] and start.tolist() == [2]
    p = ops.ragged_plan(i32([100, 100]), past, t, page_tokens=64, n_tokens=200, free_pages=free,
                        free_start=start)
    assert t.tolist() == [[4, 9, 7], [5, 8, 6]] and p.counts.tolist() == [200, 2]
    ops.ragged_plan(i32([1]), i32([192]), i32([[1, 2, 3, -1]]), page_tokens=64, n_tokens=1,
                    free_pages=free, free_start=i32([4]))
    assert ops.device_error() == 0x903                    # the list is used up


def test_serve_a_mixed_batch():
    """Prompts (one with an image), then steps that mix decoding requests with a
    new request's prompt: every step's q, cache rows and attention against the
    64-bit forms, pages handed out on the device."""
    Hq, Hkv, page, W = 8, 2, 64, 6
    width = (Hq + 2 * Hkv) * 128
    qw, kw = 1 + rnd(128, seed=1, std=0.2), 1 + rnd(128, seed=2, std=0.2)
    ids = torch.randperm(40, generator=torch.Generator().manual_seed(5)).tolist()
    kp = torch.full((40, Hkv, page, 128), math.nan, dtype=BF16, device=DEV)
    vp = torch.full_like(kp, math.nan)
    table = torch.full((4, W), -1, dtype=torch.int32, device=DEV)
    free, start = i32(ids), i32([0])
    ref_table, ref_free = [[-1] * W for _ in range(4)], list(ids)
    past = [0, 0, 0, 0]
    # request 1's prompt: 3 text tokens, a 4 x 6 image after merging 8 x 12, 5 text tokens
    types = torch.tensor([[0] * 3 + [1] * 24 + [0] * 5], device=DEV)
    mm_pos, mm_delta = ops.rope_index(types, torch.tensor([[1, 8, 12]], device=DEV))
    delta = torch.zeros(4, dtype=torch.int64, device=DEV)
    # (new tokens per request); decoding requests first, then prompts
    steps = [[60, 32, 0, 0], [1, 1, 130, 0], [1, 1, 1, 0], [1, 1, 1, 7], [1, 1, 1, 1], [1, 0, 1, 1]]
    for n_step, q_lens in enumerate(steps):
        n = sum(q_lens) + 3                                # three padding rows
        plan = ops.ragged_plan(i32(q_lens), i32(past), table, page_tokens=page, n_tokens=n,
                               free_pages=free, free_start=start, rope_delta=delta)
        want = ora.plan(q_lens, past, ref_table, page, n, ref_free, delta.tolist())
        del ref_free[:want[5][1]]
        for name, x in zip(plan._fields, want):
            assert getattr(plan, name).tolist() == x, (n_step, name)
        assert table.tolist() == ref_table
        start += plan.counts[1:]
        qkv = rnd(n, width, seed=100 + n_step)
        pos = plan.positions.expand(3, n).contiguous()
        if n_step == 0:                                    # the image's own positions
            pos[:, 60:92] = mm_pos[:, 0]
            delta[1] = mm_delta[0, 0]
        q = ops.qkv_norm_rope_ragged(qkv.to(DEV), qw.to(DEV), kw.to(DEV), pos, INV.to(DEV),
                                     plan.slots, kp, vp, Hq=Hq, Hkv=Hkv)
        live = sum(q_lens)
        wq, wk, wv, tq, tk = ora.norm_rope(qkv, qw, kw, pos.cpu(), INV, Hq, Hkv)
        ora.check("q", q[:live], wq[:live], tq[:live])
        s = plan.slots[:live].cpu()
        ora.check("k", kp.cpu()[s // page, :, s % page], wk[:live], tk[:live])
        assert torch.equal(vp.cpu()[s // page, :, s % page], wv[:live].to(BF16))
        # the requests with one token through decode, the others through prefill
        first = next((b for b, m in enumerate(q_lens) if m != 1), 4)
        out = torch.full((n, Hq, 128), 3.0, dtype=BF16, device=DEV)
        if first:
            ops.attn_decode_ragged(q[:first], kp, vp, table[:first], plan.kv_lens[:first],
                                   out=out[:first])
        ops.attn_prefill_ragged(q, kp, vp, table[first:], plan.cu_q[first:], plan.kv_lens[first:],
                                out=out)
        total = [a + b for a, b in zip(q_lens, past)]
        wo, to = ora.attention(q[:live].cpu(), kp.cpu(), vp.cpu(), ref_table,
                               [x if m else 0 for x, m in zip(total, q_lens)], q_lens)
        ora.check(f"step {n_step}", out[:live], wo, to)
        assert bool((out[live:] == 3).all())
        past = total
    assert past == [65, 36, 134, 9]


def test_decode_steps_in_one_graph_grow_their_tables():
    """plan -> norm + rotary + slots -> attention -> lengths + 1, captured once
    and replayed across page borders."""
    B, Hq, Hkv, page, W = 3, 4, 1, 64, 5
    width = (Hq + 2 * Hkv) * 128
    qw, kw = (1 + rnd(128, seed=1, std=0.2)).to(DEV), (1 + rnd(128, seed=2, std=0.2)).to(DEV)
    kp = rnd(24, Hkv, page, 128, seed=3).to(DEV)
    vp = rnd(24, Hkv, page, 128, seed=4).to(DEV)
    past0 = [62, 128, 1]
    table = i32([[3, -1, -1, -1, -1], [5, 6, -1, -1, -1], [7, -1, -1, -1, -1]])
    free = [20, 21, 22, 23, 0, 1, 2, 9]
    ones, past, start, dfree = i32([1] * B), i32(past0), i32([0]), i32(free)
    x, inv = torch.zeros(B, width, dtype=BF16, device=DEV), INV.to(DEV)

    def step():
        p = ops.ragged_plan(ones, past, table, page_tokens=page, n_tokens=B, free_pages=dfree,
                            free_start=start)
        q = ops.qkv_norm_rope_ragged(x, qw, kw, p.positions, inv, p.slots, kp, vp, Hq=Hq, Hkv=Hkv)
        o = ops.attn_decode_ragged(q, kp, vp, table, p.kv_lens)
        past.copy_(p.kv_lens)
        start.add_(p.counts[1:])
        return q, o
    keep = [t.clone() for t in (past, start, table, kp, vp)]
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        step()
    torch.cuda.synchronize()
    for t, k in zip((past, start, table, kp, vp), keep):
        t.copy_(k)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        q, o = step()
    ref = table.tolist()
    left, lens = list(free), list(past0)
    for i in range(140):
        x.copy_(rnd(B, width, seed=1000 + i))
        g.replay()
        *_, counts = ora.plan([1] * B, lens, ref, page, B, left)
        del left[:counts[1]]
        lens = [n + 1 for n in lens]
        if i % 35 == 0 or i == 139:
            assert past.tolist() == lens and table.tolist() == ref
            wo, to = ora.attention(q.cpu(), kp.cpu(), vp.cpu(), ref, lens, [1] * B)
            ora.check(f"replay {i}", o, wo, to)
    assert left == free[int(start):]


def test_pages_past_4_gib():
    """Rows whose byte and element offsets pass 32 bits: written by the norm +
    rotary call, read by both attentions."""
    Hq, Hkv, page, pages = 4, 1, 256, 1 << 17              # 8.6 GB each for K and V
    kp = torch.empty(pages, Hkv, page, 128, dtype=BF16, device=DEV)
    vp = torch.empty_like(kp)
    ids = [pages - 1, 66000, 3, pages - 2]
    n = 700
    table = i32([ids])
    qkv = rnd(n, (Hq + 2) * 128, seed=21)
    qw, kw = 1 + rnd(128, seed=1, std=0.2), 1 + rnd(128, seed=2, std=0.2)
    plan = ops.ragged_plan(i32([n]), i32([0]), table, page_tokens=page, n_tokens=n)
    q = ops.qkv_norm_rope_ragged(qkv.to(DEV), qw.to(DEV), kw.to(DEV), plan.positions, INV.to(DEV),
                                 plan.slots, kp, vp, Hq=Hq, Hkv=Hkv)
    k4, v4 = kp[torch.tensor(ids, device=DEV)].cpu(), vp[torch.tensor(ids, device=DEV)].cpu()
    _, wk, wv, _, tk = ora.norm_rope(qkv, qw, kw, torch.arange(n), INV, Hq, Hkv)
    ora.check("k", k4[:3, 0].reshape(-1, 128)[:n], wk[:, 0], tk[:, 0])
    assert torch.equal(v4[:3, 0].reshape(-1, 128)[:n], wv[:, 0].to(BF16))
    want, tol = ora.attention(q.cpu(), k4, v4, [[0, 1, 2, 3]], [n], [n])
    ora.check("prefill", ops.attn_prefill_ragged(q, kp, vp, table, plan.cu_q, plan.kv_lens), want, tol)
    ora.check("decode", ops.attn_decode_ragged(q[-1:], kp, vp, table, plan.kv_lens), want[-1:], tol[-1:])


def test_calls_captured_without_a_call_before():
    """A process may capture first: nothing is set up on the stream or allocated
    outside torch's graph pool."""
    import os
    import subprocess
    import sys
    code = """
import sys, torch
sys.path[:0] = ['qwen3-vl_b200', '.']
from q3vl import ops
from tests import ragged_oracle as ora
k, v, table = ora.make_pool([300, 70], 2, 64, stale=0.0)
q = torch.randn(5, 8, 128).to(torch.bfloat16)
d = 'cuda:0'
a = [t.to(d) for t in (q, k, v, torch.tensor(table, dtype=torch.int32))]
cu = torch.tensor([0, 2, 5], dtype=torch.int32, device=d)
kv = torch.tensor([300, 70], dtype=torch.int32, device=d)
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    x = ops.attn_prefill_ragged(*a, cu, kv)
    y = ops.attn_decode_ragged(a[0][:2], *a[1:], kv)
    p = ops.ragged_plan(kv, kv, a[3], page_tokens=64, n_tokens=370)
g.replay()
torch.cuda.synchronize()
w, t = ora.attention(q, k, v, table, [300, 70], [2, 3])
ora.check('prefill', x, w, t)
w, t = ora.attention(q[:2], k, v, table, [300, 70], [1, 1])
ora.check('decode', y, w, t)
print('fine', p.cu_q.tolist())
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "fine [0, 300, 370]" in r.stdout, r.stderr[-2000:]


def test_wrapper_refusals():
    q, k, v, table = decode_case([100, 30], 8, 2, 64, stale=0.0)
    a = [q.to(DEV), k.to(DEV), v.to(DEV), i32(table)]
    kv, cu = i32([100, 30]), i32([0, 1, 2])

    def bad(err, f, *args, **kw):
        with pytest.raises(err):
            f(*args, **kw)
    d, pf = ops.attn_decode_ragged, ops.attn_prefill_ragged
    bad(TypeError, d, a[0].float(), *a[1:], kv)
    bad(TypeError, d, *a, kv.long())
    bad(ValueError, d, *a, kv[:1])
    bad(TypeError, d, *a[:3], a[3].long(), kv)
    bad(ValueError, d, *a[:3], a[3][:1], kv)
    bad(ValueError, d, a[0], a[1], a[2][:1], a[3], kv)
    bad(ValueError, d, a[0], a[1].transpose(0, 1), a[2].transpose(0, 1), a[3], kv)
    bad(ValueError, d, a[0][..., :64], *a[1:], kv)
    bad(ValueError, d, a[0].flatten(), *a[1:], kv)
    bad(ValueError, pf, a[0].flatten(), *a[1:], cu, kv)
    bad(ValueError, d, a[0].transpose(1, 2).contiguous().transpose(1, 2), *a[1:], kv)
    bad(ValueError, d, *a, kv, out=torch.empty(2, 4, 128, dtype=BF16, device=DEV))
    bad(TypeError, d, *a, kv, out=torch.empty(2, 8, 128, device=DEV))
    bad(RuntimeError, d, *a, kv.cpu())
    bad(RuntimeError, d, a[0][:, :7], *a[1:], kv)           # 7 query heads over 2
    bad(RuntimeError, d, a[0][:1].expand(2, 8, 128), *a[1:], kv)  # rows that overlap
    bad(ValueError, pf, *a, cu[:2], kv)
    bad(RuntimeError, pf, *a, cu, kv, scale=0.0)
    bad(ValueError, ops.ragged_plan, kv, kv[:1], a[3], page_tokens=64, n_tokens=2)
    bad(ValueError, ops.ragged_plan, kv, kv, a[3], page_tokens=64, n_tokens=-1)
    bad(RuntimeError, ops.ragged_plan, kv, kv, a[3], page_tokens=100, n_tokens=2)
    bad(ValueError, ops.ragged_plan, kv, kv, a[3], page_tokens=64, n_tokens=2,
        rope_delta=torch.zeros(3, dtype=torch.int64, device=DEV))
    n = 3
    qkv, w = rnd(n, 12 * 128).to(DEV), torch.ones(128, dtype=BF16, device=DEV)
    pos, sl = torch.arange(n, device=DEV), torch.arange(n, device=DEV)
    f = lambda **kw: ops.qkv_norm_rope_ragged(                                  # noqa: E731
        kw.get("qkv", qkv), w, w, kw.get("pos", pos), kw.get("inv", INV.to(DEV)), kw.get("sl", sl),
        a[1], a[2], Hq=kw.get("Hq", 8), Hkv=kw.get("Hkv", 2), out=kw.get("out"))
    f()
    bad(ValueError, f, Hkv=1)
    bad(ValueError, f, Hq=7)
    bad(ValueError, f, pos=pos[:2])
    bad(ValueError, f, pos=pos.expand(2, n))
    bad(ValueError, f, pos=pos.int())
    bad(ValueError, f, inv=INV[:32].to(DEV))
    bad(TypeError, f, sl=sl.int())
    bad(ValueError, f, sl=sl[:2])
    bad(ValueError, f, out=torch.empty(n, 7, 128, dtype=BF16, device=DEV))
    torch.cuda.synchronize()
