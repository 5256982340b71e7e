"""Ragged serving operators on the host: refusals of the C ABI before anything
touches a device, the Python wrappers' refusals, and the plan's 64-bit form
against the page allocator's own tables."""
import ctypes

import numpy as np
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
             start=None, delta=None, n=16, cu=ONE, kv=ONE, req=ONE, pos=ONE, slots=ONE, counts=ONE, s=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,text", [
    (dict(q=None), b"null"), (dict(counts=None), b"null"), (dict(slots=None), b"null"),
    (dict(B=-1), b"B=-1"), (dict(B=8193), b"8192"), (dict(n=-1), b"n_tokens"),
    (dict(n=1 << 31), b"n_tokens"), (dict(page=0), b"page_tokens"), (dict(page=96), b"page_tokens"),
    (dict(width=0), b"width"), (dict(stride=7), b"stride"), (dict(width=1 << 25, stride=1 << 25), b"32-bit"),
    (dict(free=None), b"free list"), (dict(free=None, n_free=0, start=ONE), b"free list"), (dict(n_free=-1), b"free list"), (dict(pos=ctypes.c_void_p(20)), b"misaligned")])
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
    (dict(k=ODD), b"misaligned"), (dict(nb=100), b"workspace of 100"),
    (dict(Hq=1024, Hkv=1024, width=1 << 22, stride=1 << 22), b"32-bit tiles")])
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


# ------------------------------------------------ the kernels' work division
def decode_ranges(lens, Hkv, grid):
    """attn_decode_ragged's division: [(cta, pair, first tile, end tile, tiles)]."""
    tiles = [-(-x // 64) for x in lens]
    units = [(b * Hkv + h, t, n) for b, n in enumerate(tiles) for h in range(Hkv) for t in range(n)]
    U = len(units)
    nc = min(grid, U)
    out, desc, owner = [], {}, {}
    for c in range(nc):
        u = u0 = U * c // nc
        u1 = U * (c + 1) // nc
        while u < u1:
            pair, t0, n = units[u]
            t1 = min(n, t0 + u1 - u)
            out.append((c, pair, t0, t1, n))
            if t0 == 0 and t1 < n:
                desc[c] = (pair, ((u + n) * nc - 1) // U)
                owner[pair] = c
            elif t1 < n:
                # what the split join reads in the CTAs between: the pair's first
                # CTA (the largest k with cut(k) <= its first tile) and its last
                first = u - t0
                assert owner[pair] == ((first + 1) * nc - 1) // U
                assert desc[owner[pair]] == (pair, ((first + n) * nc - 1) // U)
            u += t1 - t0
        assert u == u1 and u0 <= u1
    return out, desc


def join_check(pieces, desc):
    """Each pair or item is either one whole piece or the pieces that its
    descriptor's slots name, in order, without a gap."""
    split = {}
    for c, key, t0, t1, n in pieces:
        assert 0 <= t0 < t1 <= n
        if (t0, t1) != (0, n):
            slot = 2 * c + (1 if t0 == 0 else 0)
            split.setdefault(key, []).append((slot, t0, t1, n))
    slots = [s for v in split.values() for s, *_ in v]
    assert len(slots) == len(set(slots))
    named = {}
    for c, (key, last) in desc.items():
        named[key] = [2 * c + 1] + [2 * k for k in range(c + 1, last + 1)]
    assert set(named) == set(split)
    for key, parts in split.items():
        assert [s for s, *_ in parts] == named[key]
        assert parts[0][1] == 0 and parts[-1][2] == parts[-1][3]
        assert all(a[2] == b[1] for a, b in zip(parts, parts[1:]))


LENGTHS = [[1], [0], [700], [0, 0, 64, 65, 0], [329, 585, 758, 2048, 580, 1405, 0, 153],
           [5] * 300, [30000, 1, 1, 1], [0] * 40 + [3000]]


@pytest.mark.parametrize("lens", LENGTHS)
@pytest.mark.parametrize("Hkv", [1, 3, 8])
@pytest.mark.parametrize("grid", [1, 5, 148])
def test_decode_division_covers_every_tile_once(lens, Hkv, grid):
    pieces, desc = decode_ranges(lens, Hkv, grid)
    seen = sorted((k, t) for _, k, t0, t1, _ in pieces for t in range(t0, t1))
    assert seen == sorted((b * Hkv + h, t) for b, x in enumerate(lens) for h in range(Hkv)
                          for t in range(-(-x // 64)))
    join_check(pieces, desc)
    per = [sum(p[3] - p[2] for p in pieces if p[0] == c) for c in range(min(grid, len(seen)))]
    assert not per or max(per) - min(per) <= 1


ITEM_COST = 256        # places of the list an item takes besides its keys


def n_tiles(T, q, L, i, causal=True):
    x = L - q + min(q, (i + 1) * 2 * T) if causal else L
    return 1 if x <= 128 else -(-x // 128)


def weight(T, q, L, i, causal=True):
    return (max(L - q, 0) + min(q, (i + 1) * 2 * T) if causal else L) + ITEM_COST


def places(T, q, L, i, causal=True):
    """Places of items [0, i), as the kernel sums them in closed form."""
    if not causal:
        return i * (L + ITEM_COST)
    n, base = -(-q // (2 * T)), max(L - q, 0) + ITEM_COST
    full = i if i < n else max(n - 1, 0)
    s = full * base + T * full * (full + 1)
    return s + base + q if i > full else s


def item_at(T, q, L, rem, causal=True):
    """The kernel's fp32 root and its correction."""
    f = np.float32
    n = -(-q // (2 * T))
    h = f(max(L - q, 0)) + f(ITEM_COST + T)
    x = (np.sqrt(h * h + f(4) * f(T) * f(rem)) - h) / (f(2) * f(T)) if causal else \
        f(rem) / f(L + ITEM_COST)
    i = min(max(int(x), 0), n - 1)
    steps = 0
    while i > 0 and places(T, q, L, i, causal) > rem:
        i, steps = i - 1, steps + 1
    while i + 1 < n and places(T, q, L, i + 1, causal) <= rem:
        i, steps = i + 1, steps + 1
    return i, steps


def test_places_in_closed_form_and_the_item_of_a_place():
    import random
    r = random.Random(2)
    for _ in range(300):
        T = r.choice([128, 64, 42, 32, 25, 21, 18, 16, 10, 8])
        q, past = r.randint(1, 900), r.choice([0, 1, 63, 64, 127, 128, 129, 5000, -3, -400])
        L = max(0, q + past)
        n = -(-q // (2 * T))
        for causal in (True, False):
            sums = [sum(weight(T, q, L, k, causal) for k in range(i)) for i in range(n + 1)]
            assert [places(T, q, L, i, causal) for i in range(n + 1)] == sums
            for _ in range(20):
                rem = r.randrange(sums[-1])
                i, steps = item_at(T, q, L, rem, causal)
                assert sums[i] <= rem < sums[i + 1] and steps <= 2
    # prompts of millions of tokens: the fp32 root stays within a few items
    for T, q, past in ((8, 3_000_000, 0), (32, 10_000_000, 5), (128, 1_000_000, 900_000_000)):
        L, n = q + past, -(-q // (2 * T))
        for _ in range(50):
            i = r.randrange(n)
            rem = places(T, q, L, i) + r.choice([0, 1, 200])
            got, steps = item_at(T, q, L, rem)
            assert got == i and steps <= 64, (T, q, past, i, steps)


def cut_tile(pos, w, nt, snap):
    if pos >= w:
        return nt
    t = min(max(pos - ITEM_COST + 64, 0) // 128, nt)
    if t < snap and 2 * t < nt:
        return 0
    return nt if nt - t < snap else t


def prefill_ranges(qs, Ls, T, Hkv, grid, causal=True):
    """attn_prefill_ragged's division, walked as the kernel's roles walk it."""
    items, u = [], 0
    for b, (q, L) in enumerate(zip(qs, Ls)):
        for h in range(Hkv):
            for i in range(-(-q // (2 * T))):
                w = weight(T, q, L, i, causal)
                items.append(((b, h, i), n_tiles(T, q, L, i, causal), u, w))
                u += w
    U, nc = u, min(grid, u // 128)
    share = U // nc if nc else 0
    rest = U - share * nc

    def cut(k):
        return share * k + rest * k // nc
    snap = min(share // 1024, 2)
    pieces, desc, at = [], {}, 0
    for c in range(nc):
        u0, u1 = cut(c), cut(c + 1)
        assert u1 - u0 >= 128
        while items[at][2] + items[at][3] <= u0:
            at += 1
        k = at
        while k < len(items) and items[k][2] < u1:
            key, nt, base, w = items[k]
            t0 = cut_tile(max(u0 - base, 0), w, nt, snap)
            t1 = cut_tile(min(u1 - base, w), w, nt, snap)
            if t0 < t1:
                pieces.append((c, key, t0, t1, nt))
                if t0 == 0 and t1 < nt:
                    last, x = c, c + 1
                    while x < nc:                # 32 candidates at a time, as the warp does
                        n = 0
                        for lane in range(32):
                            y = x + lane
                            n += y < nc and cut_tile(cut(min(y, nc)) - base, w, nt, snap) < nt
                        last += n
                        if n < 32:
                            break
                        x += 32
                    desc[c] = (key, last)
            k += 1
    assert not nc or cut(nc) == U
    return pieces, desc, items


def test_prefill_division_covers_every_tile_once():
    import random
    r = random.Random(5)
    cases = [([512], [32768], 32, 8), ([1], [1], 32, 1), ([0, 3, 0], [9, 3, 0], 128, 2),
             ([4096, 1, 77], [4096, 1, 5000], 32, 8), ([16], [300000], 8, 1), ([5], [2], 25, 1),
             ([1] * 200, list(range(1, 201)), 32, 2)]
    for _ in range(60):
        B = r.randint(1, 9)
        qs = [r.choice([0, 1, 5, 64, 65, 300, 1111]) for _ in range(B)]
        cases.append((qs, [q + r.choice([0, 0, 1, 500, 9000]) for q in qs],
                      r.choice([128, 64, 42, 32, 18, 8]), r.choice([1, 2, 8])))
    for qs, Ls, T, Hkv in cases:
        for grid in (1, 7, 148):
            for causal in (True, False):
                pieces, desc, items = prefill_ranges(qs, Ls, T, Hkv, grid, causal)
                seen = [(k, t) for _, k, t0, t1, _ in pieces for t in range(t0, t1)]
                assert len(seen) == len(set(seen))
                assert sorted(seen) == sorted((k, t) for k, nt, *_ in items for t in range(nt))
                join_check(pieces, desc)


def prefill_args(**kw):
    a = dict(q=ONE, qs=1024, k=ONE, v=ONE, out=ONE, os=1024, n=100, B=4, Hq=8, Hkv=2, d=128,
             table=ONE, stride=8, width=8, page=64, pages=10, cu=ONE, lens=ONE, causal=1, scale=0.1,
             ws=ONE, nb=1 << 30, s=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,text", [
    (dict(d=64), b"head_dim"), (dict(B=-1), b"bad shape"), (dict(Hq=7), b"bad shape"),
    (dict(n=-1), b"bad shape"), (dict(q=None), b"null"), (dict(cu=None), b"null"),
    (dict(page=32), b"page_tokens"), (dict(width=0), b"table width"), (dict(stride=4), b"stride"),
    (dict(pages=0), b"pages"), (dict(pages=1 << 25), b"too large"), (dict(qs=1000), b"strides"),
    (dict(os=1028), b"strides"), (dict(q=ODD), b"misaligned"), (dict(scale=0.0), b"positive"),
    (dict(scale=-1.0), b"positive"), (dict(scale=float("nan")), b"positive"),
    (dict(scale=float("inf")), b"positive"), (dict(nb=100), b"workspace of 100")])
def test_prefill_refusals(kw, text):
    refused("q3_attn_prefill_ragged", prefill_args(**kw), text)


def test_prefill_refuses_more_than_16_heads_a_group_and_accepts_empty_calls():
    refused("q3_attn_prefill_ragged", prefill_args(Hq=34, qs=1 << 20, os=1 << 20), b"above 16",
            _lib.Q3_ERR_UNSUPPORTED)
    assert _lib.raw("q3_attn_prefill_ragged")(*prefill_args(B=0, q=None)) == 0
    assert _lib.raw("q3_attn_prefill_ragged")(*prefill_args(n=0, q=None)) == 0


def test_calls_run_on_the_tensors_own_device(monkeypatch):
    """A call whose tensors are on device 1 while device 0 is current switches to
    device 1 and passes its current stream."""
    seen, at = [], [0]

    class Guard:
        def __init__(self, dev):
            self.dev = dev

        def __enter__(self):
            self.old, at[0] = at[0], self.dev

        def __exit__(self, *a):
            at[0] = self.old

    def entry(*args):
        seen.append((at[0],) + args)
        return 0
    monkeypatch.setattr(torch.cuda, "current_device", lambda: at[0])
    monkeypatch.setattr(torch.cuda, "device", Guard)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda d: 100 + d, raising=False)
    monkeypatch.setattr(_lib, "raw", lambda name: entry)
    ops._ragged_call("q3_x", 0, 7)
    ops._ragged_call("q3_x", 1, 8)
    assert seen == [(0, 7, 100), (1, 8, 101)] and at == [0]
    monkeypatch.setattr(_lib, "raw", lambda name: lambda *a: _lib.Q3_ERR_INVALID)
    with pytest.raises(_lib.Q3Error):
        ops._ragged_call("q3_x", 0, 7)


def test_workspace_sizes_are_asked_on_the_tensors_device(monkeypatch):
    at, asked = [0], []

    class Guard:
        def __init__(self, dev):
            self.dev = dev

        def __enter__(self):
            self.old, at[0] = at[0], self.dev

        def __exit__(self, *a):
            at[0] = self.old

    def size(*args):
        asked.append((at[0],) + args)
        return 64 + at[0]
    monkeypatch.setattr(torch.cuda, "device", Guard)
    monkeypatch.setattr(_lib, "raw", lambda name: size)
    monkeypatch.setattr(ops, "_ragged_ws_bytes", {})
    q = torch.zeros(1)
    for dev, args in ((0, (8, 2)), (1, (8, 2)), (0, (8, 2)), (0, (4, 2))):
        ws, n = ops._ragged_workspace(q, dev, "q3_x", *args)
        assert n == 64 + dev and ws.dtype == torch.uint8 and ws.numel() == n
    assert asked == [(0, 8, 2), (1, 8, 2), (0, 4, 2)] and at == [0]
