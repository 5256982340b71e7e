"""Plain 64-bit forms of the ragged serving operators, on the CPU, and the error
bounds that the GPU tests allow.

Every sum over keys is a loop over requests and heads with the request's own
rows gathered through its block table, as the formulas are written; nothing is
shared with the kernels' tiling.
"""
import math

import torch

HD = 128
# one bf16 rounding moves a value by at most half a step: eps / 2 of it
BF16_HALF = torch.finfo(torch.bfloat16).eps / 2


def plan(q_lens, past, table, page, n_tokens, free=None, delta=None):
    """ragged_plan on lists (table: list of lists, changed in place)."""
    cu, kv, req, pos, slots = [0], [], [], [], []
    taken = 0
    for b, (q, p) in enumerate(zip(q_lens, past)):
        if free is not None:
            have, want = -(-p // page), -(-(p + q) // page)
            for j in range(have, want):
                table[b][j] = free[taken]
                taken += 1
        for i in range(q):
            t = p + i
            req.append(b)
            pos.append(t + (delta[b] if delta is not None else 0))
            slots.append(table[b][t // page] * page + t % page)
        cu.append(cu[-1] + q)
        kv.append(p + q)
    counts = [len(req), taken]
    pad = n_tokens - len(req)
    return cu, kv, req + [-1] * pad, pos + [0] * pad, slots + [-1] * pad, counts


def axis_of(j, section):
    if j % 3 == 1 and j < 3 * section[1]:
        return 1
    if j % 3 == 2 and j < 3 * section[2]:
        return 2
    return 0


def norm_rope(qkv, qw, kw, positions, inv_freq, Hq, Hkv, section=(24, 20, 20), eps=1e-6):
    """q [n, Hq, 128], k, v [n, Hkv, 128] in fp64 and the bound for q and k."""
    n = qkv.shape[0]
    x = qkv.double().view(n, Hq + 2 * Hkv, HD)
    pos = positions.double().expand(3, n) if positions.dim() == 1 else positions.double()
    ang = torch.stack([pos[axis_of(j, section)] * inv_freq[j].double() for j in range(HD // 2)], 1)
    c, s = ang.cos()[:, None], ang.sin()[:, None]
    w = torch.cat([qw.double().expand(Hq, HD), kw.double().expand(Hkv, HD)])
    y = x[:, :Hq + Hkv]
    y = y / (y.pow(2).mean(-1, keepdim=True) + eps).sqrt() * w
    a, b = y[..., :64], y[..., 64:]
    out = torch.cat([a * c - b * s, b * c + a * s], -1)
    # one rounding of the result, and fp32 error of n (about 140 roundings of a
    # sum of squares, halved by the root, and four products), of the sine and
    # cosine (2 ulp each, and 1 of the reduced angle) and of the two products:
    # under 100 * 2^-24 of |a| + |b|
    mag = (a.abs() + b.abs()).repeat(1, 1, 2)
    tol = BF16_HALF * out.abs() + 100 * 2.0 ** -24 * mag
    return out[:, :Hq], out[:, Hq:], x[:, Hq + Hkv:], tol[:, :Hq], tol[:, Hq:]


def rows_of(pool, ids, h, L, page):
    ids = torch.as_tensor(ids[:-(-L // page)], dtype=torch.long)
    return pool[ids, h].reshape(-1, HD)[:L].double()


def attention(q, k_pages, v_pages, table, kv_lens, q_lens, scale=None, causal=True):
    """Packed q [sum q_lens, Hq, 128] -> (out, bound).  Query i of request b sees
    positions [0, kv_len - q_len + i] (all of kv_len when not causal).

    The bound: one bf16 rounding of the output; each probability rounded to
    bf16 (half a step of it, so BF16_HALF * sum p|v|); and fp32: a score is a sum
    of 128 products, off by at most 128 * 2^-24 * sum |q k| * scale, which the
    exponential turns into a relative error of p, in the numerator and in the
    sum; 2^-21 for the exponentials and the sums of p and p v over up to 2^15
    keys in runs of at most 2^9 (2^-15)."""
    n, Hq, _ = q.shape
    Hkv, page = k_pages.shape[1], k_pages.shape[2]
    G = Hq // Hkv
    scale = 1.0 / math.sqrt(HD) if scale is None else scale
    out = torch.zeros(n, Hq, HD, dtype=torch.float64)
    tol = torch.zeros_like(out)
    first = 0
    for b, (m, L) in enumerate(zip(q_lens, kv_lens)):
        if m and L:
            pos = torch.arange(L - m, L) if causal else torch.full((m,), L - 1)
            hidden = torch.arange(L)[None] > pos[:, None]
            for h in range(Hkv):
                k = rows_of(k_pages, table[b], h, L, page)
                v = rows_of(v_pages, table[b], h, L, page)
                for g in range(G):
                    qq = q[first:first + m, h * G + g].double()
                    sc = (qq @ k.T * scale).masked_fill(hidden, -math.inf)
                    seen = ~hidden.all(1)
                    p = torch.zeros_like(sc)
                    p[seen] = torch.softmax(sc[seen], -1)
                    o = p @ v
                    a = p @ v.abs()
                    mag = (qq.abs() @ k.abs().T * scale).amax(-1, keepdim=True)
                    rel = 2 * 130 * 2.0 ** -24 * mag + 2.0 ** -15 + 2.0 ** -21
                    out[first:first + m, h * G + g] = o
                    tol[first:first + m, h * G + g] = \
                        (BF16_HALF * o.abs() + (BF16_HALF + rel) * a) * (1 + BF16_HALF)
        first += m
    return out, tol


def check(name, got, want, tol):
    g = got.detach().double().cpu()
    assert g.shape == want.shape, f"{name}: {tuple(g.shape)} vs {tuple(want.shape)}"
    assert torch.isfinite(g).all(), f"{name}: non-finite output"
    over = (g - want).abs() - tol
    worst = int(over.argmax()) if over.numel() else 0
    assert over.numel() == 0 or over.max() <= 0, \
        f"{name}: off by {(g - want).abs().flatten()[worst]:.3e} at {worst}, " \
        f"bound {tol.flatten()[worst]:.3e}"


def make_pool(lens, Hkv, page, seed=0, stale=None, extra=2, width=None):
    """Pools with each request's rows in shuffled pages; every other row, in the
    last page of a request and in unused pages, holds `stale` (or old values)."""
    g = torch.Generator().manual_seed(seed)
    counts = [-(-x // page) for x in lens]
    n = sum(counts) + extra
    ids = torch.randperm(n, generator=g).tolist()
    W = max(1, max(counts, default=1)) if width is None else width
    k = torch.randn(n, Hkv, page, HD, generator=g).to(torch.bfloat16)
    v = torch.randn(n, Hkv, page, HD, generator=g).to(torch.bfloat16)
    table, at = [], 0
    live = torch.zeros(n, page, dtype=torch.bool)
    for x, c in zip(lens, counts):
        row = ids[at:at + c]
        at += c
        for i, pg in enumerate(row):
            live[pg, :min(page, x - i * page)] = True
        table.append(row + [-1] * (W - c))
    if stale is not None:
        dead = ~live[:, None, :, None].expand_as(k)
        k[dead] = stale
        v[dead] = stale
    return k, v, table
