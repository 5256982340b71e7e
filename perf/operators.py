"""Serving a ragged batch over paged K/V: the workloads that the ragged operators are timed on.

A serving step takes requests of different lengths at once: some bring a prompt
(or a chunk of one), some one new token.  Four operators carry it, here in
plain torch (`own` false) and as the calls that a user makes of q3vl.ops
(`own` true):

  plan     ops.ragged_plan           block tables, slot maps and positions
                                     from the requests' lengths
  qkv      ops.qkv_norm_rope_ragged  per-head QK-RMSNorm, 3-axis interleaved
                                     rotary positions, K/V rows to their slots
  decode   ops.attn_decode_ragged    attention of one new token per request,
                                     each over its own length of the page pool
  prefill  ops.attn_prefill_ragged   causal attention of packed prompt chunks
                                     over the page pool

Head counts are the 8B text decoder's (32 query and 8 K/V heads), its
tensor-parallel shards' (16/4, 4/1) and generic ones; page sizes and the K/V
buckets (2048, 8192) are the page pool's.
"""
import math
import os
import random
import sys

import torch

own = False

HD = 128
BF16 = torch.bfloat16
THETA = 5e6
SECTION = (24, 20, 20)
EPS = 1e-6


def _ops():
    path = os.path.abspath("qwen3-vl_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    from q3vl import ops
    return ops


# --------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------
def listed():
    return [
        # a decode step of a small server: 8 requests, one new token each
        dict(name="plan_decode_8", op="plan", B=8, q_max=1, past_max=2047, page=256, pad=0, lens=1),
        # a mixed step: 64 slots, prompt chunks of up to 512 tokens beside
        # single tokens and idle slots, packed into a padded token buffer
        dict(name="plan_mixed_64", op="plan", B=64, q_max=512, past_max=8191, page=64, pad=37, lens=2),
        # admission of a large queue: 1024 requests, prompts of up to 512 tokens
        dict(name="plan_queue_1024", op="plan", B=1024, q_max=512, past_max=2048, page=256, pad=0, lens=3),
        # the new tokens of a decode step, 8B heads, one text axis
        dict(name="qkv_decode_8", op="qkv", n=8, Hq=32, Hkv=8, axes=1, page=256, pad=0, far=2048),
        # an odd number of image and text tokens on one of 8 tensor-parallel
        # ranks, padded at the end
        dict(name="qkv_image_1037_tp8", op="qkv", n=1037, Hq=4, Hkv=1, axes=3, page=64, pad=19, far=32768),
        # the packed prompts of one large prefill step
        dict(name="qkv_prompts_16384", op="qkv", n=16384, Hq=32, Hkv=8, axes=3, page=256, pad=0, far=131072),
        # one request on one of 8 tensor-parallel ranks
        dict(name="decode_1_tp8", op="decode", B=1, Hq=4, Hkv=1, max_len=700, page=64, idle=0, lens=4),
        # 8 slots of a 2048-token bucket at different lengths, one of them idle
        dict(name="decode_8_bucket", op="decode", B=8, Hq=32, Hkv=8, max_len=2048, page=256, idle=1, lens=5),
        # 32 long conversations, the lengths spread over two orders of magnitude
        dict(name="decode_32_long", op="decode", B=32, Hq=32, Hkv=8, max_len=32768, page=256, idle=0, lens=6),
        # four short prompts on one of 8 tensor-parallel ranks
        dict(name="prefill_4_short_tp8", op="prefill", B=4, Hq=4, Hkv=1, q_max=100, past_max=0, page=64, idle=0, lens=7),
        # one 512-token chunk of a long prompt, on a cache near 32k tokens
        dict(name="prefill_chunk_32k", op="prefill", B=1, Hq=32, Hkv=8, q_max=512, past_max=32256, page=256, idle=0, lens=8),
        # six prompts of up to 4096 tokens, some on a cached prefix
        dict(name="prefill_6_prompts", op="prefill", B=6, Hq=32, Hkv=8, q_max=4096, past_max=1024, page=256, idle=0, lens=9),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("plan", "qkv", "decode", "prefill"))
    page = rng.choice((64, 128, 256, 192))
    lens = rng.randrange(1 << 30)
    if op == "plan":
        B = _log(rng, 1, 1024)
        return dict(op=op, B=B, q_max=_log(rng, 1, 512), past_max=_log(rng, 1, 8192 if B <= 256 else 2048),
                    page=page, pad=rng.choice((0, 1, 130)), lens=lens)
    Hkv = rng.choice((1, 2, 4, 8))
    if op == "qkv":
        Hq = Hkv * rng.choice((1, 2, 3, 4, 5, 7, 8) if Hkv < 8 else (1, 2, 3, 4))
        n = _log(rng, 1, 16384 * 40 // max(40, Hq + 2 * Hkv))
        return dict(op=op, n=n, Hq=Hq, Hkv=Hkv, axes=rng.choice((1, 3)), page=page,
                    pad=rng.choice((0, 1, 33)) if n > 64 else 0, far=_log(rng, 64, 1 << 20))
    Hq = Hkv * rng.choice((1, 2, 3, 4, 5, 6, 7, 8, 12, 16) if Hkv < 8 else (1, 2, 4, 8))
    Hq = min(Hq, 32 // Hkv * Hkv)
    if op == "decode":
        B = _log(rng, 1, 24)
        return dict(op=op, B=B, Hq=Hq, Hkv=Hkv, max_len=_log(rng, 1, 32768), page=page,
                    idle=rng.choice((0, 1)) if B > 1 else 0, lens=lens)
    B = _log(rng, 1, 6)
    q_max = _log(rng, 1, 2048)
    past_max = _log(rng, 1, 4096) if q_max > 256 else _log(rng, 1, 16384)
    return dict(op=op, B=B, Hq=Hq, Hkv=Hkv, q_max=q_max, past_max=past_max, page=page,
                idle=rng.choice((0, 1)) if B > 1 else 0, lens=lens)


def _spread(r, lo, hi):
    """A length between lo and hi, spread over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(r.uniform(math.log(max(lo, 1)), math.log(max(hi, 1))))))))


def _lengths(case):
    """(new tokens, tokens cached before) of each request: the same for every seed."""
    r = random.Random(case["lens"])
    op, B = case["op"], case["B"]
    if op == "decode":
        past = [_spread(r, max(1, case["max_len"] // 128), case["max_len"]) for _ in range(B)]
        past[r.randrange(B)] = case["max_len"]
        q = [0] * B
        if case["idle"]:
            past[past.index(min(past))] = 0
        return q, past
    q = [_spread(r, 1, case["q_max"]) for _ in range(B)]
    past = [r.randint(0, case["past_max"]) for _ in range(B)]
    if op == "prefill":
        q = [_spread(r, max(1, case["q_max"] // 4), case["q_max"]) for _ in range(B)]
        q[r.randrange(B)] = case["q_max"]
        past = [x if r.random() < 0.5 else 0 for x in past]
        if B == 1:
            past[0] = case["past_max"]
        if case["idle"]:
            q[q.index(min(q))] = 0
    elif B > 8:
        q = [0 if r.random() < 0.05 else x for x in q]
    return q, past


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------
def _rand(gen, *shape, std=1.0):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32).mul_(std).to(BF16)


def _pool(gen, tokens, Hkv, page, std):
    """A page pool with room for `tokens`, filled all over: pages that were in use before hold old rows."""
    out = torch.empty(tokens // page, Hkv, page, HD, device="cuda", dtype=BF16)
    for i in range(0, out.shape[0], 512):
        n = min(512, out.shape[0] - i)
        out[i:i + n] = _rand(gen, n, Hkv, page, HD, std=std)
    return out


def _int(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    op, page = case["op"], case["page"]
    st = dict(op=op, page=page)
    if op == "qkv":
        n, Hq, Hkv = case["n"], case["Hq"], case["Hkv"]
        heads = Hq + 2 * Hkv
        pages = (n + page - 1) // page + 1
        st.update(Hq=Hq, Hkv=Hkv, qkv=_rand(gen, n, heads * HD),
                  qw=1 + _rand(gen, HD, std=0.1), kw=1 + _rand(gen, HD, std=0.1),
                  k=_pool(gen, pages * page, Hkv, page, 1.0), v=_pool(gen, pages * page, Hkv, page, 1.0),
                  out=torch.zeros(n, Hq, HD, device="cuda", dtype=BF16),
                  inv=1.0 / (THETA ** (torch.arange(0, HD, 2, device="cuda", dtype=torch.float32) / HD)))
        pos = torch.randint(0, case["far"], (case["axes"], n), generator=gen, device="cuda")
        st["pos"] = pos[0].contiguous() if case["axes"] == 1 else pos
        slots = torch.randperm(pages * page, generator=gen, device="cuda")[:n]
        if case["pad"]:
            slots[n - case["pad"]:] = -1
        st.update(slots=slots, live=n - case["pad"])
        return st
    q, past = _lengths(case)
    B = case["B"]
    total = [a + b for a, b in zip(q, past)]
    width = max(1, -(-max(total) // page))
    if op == "plan":
        have = [-(-x // page) for x in past]
        need = sum(-(-x // page) for x in total) - sum(have)
        owned = sum(have)
        order = torch.randperm(owned + need + 16, generator=gen, device="cuda").to(torch.int32)
        j = torch.arange(width, device="cuda")[None]
        h = _int(have, torch.int64)
        at = (h.cumsum(0) - h)[:, None] + j
        table = torch.where(j < h[:, None], order[at.clamp(max=order.numel() - 1)], -1).to(torch.int32)
        st.update(q_lens=_int(q), past=_int(past), table=table.contiguous(), free=order[owned:].contiguous(),
                  n=sum(q) + case["pad"], delta=torch.randint(-500, 500, (B,), generator=gen, device="cuda"))
        return st
    Hq, Hkv = case["Hq"], case["Hkv"]
    counts = [-(-x // page) for x in total]
    pages = sum(counts) + 1
    perm = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    c = _int(counts, torch.int64)
    j = torch.arange(width, device="cuda")[None]
    at = (c.cumsum(0) - c)[:, None] + j
    st["table"] = torch.where(j < c[:, None], perm[at.clamp(max=pages - 1)], -1).to(torch.int32).contiguous()
    st.update(k=_pool(gen, pages * page, Hkv, page, 1.0), v=_pool(gen, pages * page, Hkv, page, 1.0),
              kv_lens=_int(total), max_kv=max(total))
    if op == "decode":
        st["q"] = _rand(gen, B, Hq, HD, std=1.5)
    else:
        n = sum(q)
        cu = [0]
        for x in q:
            cu.append(cu[-1] + x)
        st.update(q=_rand(gen, n, Hq, HD, std=1.5), cu_q=_int(cu), max_q=max(q))
    return st


# --------------------------------------------------------------------------
# the operators
# --------------------------------------------------------------------------
def run(state):
    s = state
    if own:
        ops = _ops()
        if s["op"] == "plan":
            p = ops.ragged_plan(s["q_lens"], s["past"], s["table"], page_tokens=s["page"], n_tokens=s["n"],
                                free_pages=s["free"], rope_delta=s["delta"])
            return dict(table=s["table"], cu_q=p.cu_q, kv_lens=p.kv_lens, requests=p.requests,
                        positions=p.positions, slots=p.slots, counts=p.counts)
        if s["op"] == "qkv":
            q = ops.qkv_norm_rope_ragged(s["qkv"], s["qw"], s["kw"], s["pos"], s["inv"], s["slots"], s["k"], s["v"],
                                         Hq=s["Hq"], Hkv=s["Hkv"], mrope_section=SECTION, eps=EPS, out=s["out"])
            return dict(q=q, k=s["k"], v=s["v"])
        if s["op"] == "decode":
            return ops.attn_decode_ragged(s["q"], s["k"], s["v"], s["table"], s["kv_lens"])
        return ops.attn_prefill_ragged(s["q"], s["k"], s["v"], s["table"], s["cu_q"], s["kv_lens"])
    return dict(plan=_plan, qkv=_qkv, decode=_decode, prefill=_prefill)[s["op"]](s)


def _plan(s):
    page, n, table = s["page"], s["n"], s["table"]
    q, past = s["q_lens"].long(), s["past"].long()
    total = q + past
    have, want = (past + page - 1) // page, (total + page - 1) // page
    need = want - have
    first = need.cumsum(0) - need
    j = torch.arange(table.shape[1], device=table.device)[None]
    fresh = (j >= have[:, None]) & (j < want[:, None])
    at = (first[:, None] + j - have[:, None]).clamp(0, s["free"].numel() - 1)
    table.copy_(torch.where(fresh, s["free"][at], table))
    ends = q.cumsum(0)
    t = torch.arange(n, device=table.device)
    live = t < ends[-1]
    req = torch.searchsorted(ends, t, right=True).clamp(max=q.numel() - 1)
    pos = past[req] + t - (ends - q)[req]
    pages = table[req, (pos // page).clamp(0, table.shape[1] - 1)].long()
    cu = torch.zeros(q.numel() + 1, device=table.device, dtype=torch.int32)
    cu[1:] = ends
    return dict(table=table, cu_q=cu, kv_lens=total.int(),
                requests=torch.where(live, req, -1).int(), positions=torch.where(live, pos + s["delta"][req], 0),
                slots=torch.where(live, pages * page + pos % page, -1),
                counts=torch.stack((ends[-1], need.sum())).int())


def _qkv(s):
    Hq, Hkv = s["Hq"], s["Hkv"]
    n = s["qkv"].shape[0]
    x = s["qkv"].view(n, Hq + 2 * Hkv, HD).float()
    j = torch.arange(HD // 2, device=x.device)
    axis = torch.where((j % 3 == 1) & (j < 3 * SECTION[1]), 1, torch.where((j % 3 == 2) & (j < 3 * SECTION[2]), 2, 0))
    pos = s["pos"].expand(3, n) if s["pos"].dim() == 1 else s["pos"]
    ang = pos.double()[axis].T * s["inv"].double()              # angles of far positions need 64 bits
    cos, sin = ang.cos().float().repeat(1, 2)[:, None], ang.sin().float().repeat(1, 2)[:, None]
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    w = torch.cat((s["qw"].float().expand(Hq, HD), s["kw"].float().expand(Hkv, HD)))
    y = (x * r)[:, :Hq + Hkv] * w
    half = torch.cat((-y[..., HD // 2:], y[..., :HD // 2]), -1)
    y = (y * cos + half * sin).to(BF16)
    live, page = s["live"], s["page"]                           # padding comes last
    slot = s["slots"][:live]
    s["out"][:live] = y[:live, :Hq]
    s["k"][slot // page, :, slot % page] = y[:live, Hq:]
    s["v"][slot // page, :, slot % page] = x[:live, Hq + Hkv:].to(BF16)
    return dict(q=s["out"], k=s["k"], v=s["v"])


def _gather(s, pool):
    """[B, Hkv, L, 128] in 32 bits: each request's rows in order, whatever lies past its end."""
    t = s["table"].clamp(min=0).long()
    B, W = t.shape
    x = pool[t].transpose(1, 2)
    return x.reshape(B, pool.shape[1], W * s["page"], HD)[:, :, :max(1, s["max_kv"])].float()


def _softmax(sc):
    """Softmax over the last axis; a row with nothing to attend to gives zeros."""
    m = sc.amax(-1, keepdim=True).clamp(min=-3e38)
    p = sc.sub_(m).exp_()
    return p.div_(p.sum(-1, keepdim=True).clamp(min=1e-30))


def _decode(s):
    k, v = _gather(s, s["k"]), _gather(s, s["v"])
    B, Hq, _ = s["q"].shape
    Hkv = k.shape[1]
    q = s["q"].float().view(B, Hkv, Hq // Hkv, HD) / math.sqrt(HD)
    off = torch.arange(k.shape[2], device=k.device)[None] >= s["kv_lens"][:, None]
    sc = (q @ k.transpose(-1, -2)).masked_fill_(off[:, None, None], -math.inf)
    return (_softmax(sc) @ v).view(B, Hq, HD).to(BF16)


def _prefill(s):
    k, v = _gather(s, s["k"]), _gather(s, s["v"])
    n, Hq, _ = s["q"].shape
    B, Hkv, L, _ = k.shape
    G, M = Hq // Hkv, max(1, s["max_q"])
    cu = s["cu_q"].long()
    lens = cu[1:] - cu[:-1]
    i = torch.arange(M, device=k.device)[None]
    at = (cu[:-1, None] + i).clamp(max=n - 1)
    live = i < lens[:, None]
    q = s["q"].float()[at].view(B, M, Hkv, G, HD).permute(0, 2, 3, 1, 4) / math.sqrt(HD)
    qpos = s["kv_lens"].long()[:, None] - lens[:, None] + i
    off = torch.arange(L, device=k.device) > torch.where(live, qpos, -1)[..., None]
    sc = (q.reshape(B, Hkv, G * M, HD) @ k.transpose(-1, -2)).view(B, Hkv, G, M, L).masked_fill_(off[:, None, None], -math.inf)
    o = (_softmax(sc).view(B, Hkv, G * M, L) @ v).view(B, Hkv, G, M, HD).permute(0, 3, 1, 2, 4).reshape(B, M, Hq, HD)
    t = torch.arange(n, device=k.device)
    req = torch.searchsorted(cu[1:], t, right=True)
    return o[req, t - cu[req]].to(BF16)


# --------------------------------------------------------------------------
# what an operator cannot do without
# --------------------------------------------------------------------------
def work(case):
    op = case["op"]
    if op == "qkv":
        n, heads = case["n"] - case["pad"], case["Hq"] + 2 * case["Hkv"]
        return dict(bytes=n * (2 * heads * HD * 2 + 8 * case["axes"]) + case["n"] * 8 + 3 * 256,
                    flops=n * (case["Hq"] + case["Hkv"]) * HD * 8)
    q, past = _lengths(case)
    page, B = case["page"], case["B"]
    total = [a + b for a, b in zip(q, past)]
    if op == "plan":
        n = sum(q) + case["pad"]
        need = sum(-(-x // page) for x in total) - sum(-(-x // page) for x in past)
        read = sum(-(-t // page) - p // page for t, p, m in zip(total, past, q) if m) - need   # part-filled last pages
        return dict(bytes=B * (4 + 4 + 8 + 4 + 4) + need * 8 + read * 4 + n * (4 + 8 + 8), flops=n * 4)
    Hq, Hkv = case["Hq"], case["Hkv"]
    pages = sum(-(-x // page) for x in total)
    if op == "decode":
        return dict(bytes=sum(total) * Hkv * HD * 4 + B * Hq * HD * 4 + B * 4 + pages * 4,
                    flops=sum(total) * Hq * HD * 4)
    pairs = sum(m * p + m * (m + 1) // 2 for m, p in zip(q, past))
    kv = sum(t for t, m in zip(total, q) if m)
    return dict(bytes=kv * Hkv * HD * 4 + sum(q) * Hq * HD * 4 + B * 8 + pages * 4, flops=pairs * Hq * HD * 4)


# --------------------------------------------------------------------------
# the definition in 64 bits
# --------------------------------------------------------------------------
def exact(case, seed):
    op, page = case["op"], case["page"]
    s = prepare(case, seed)
    if op == "plan":
        return None                       # whole numbers: compared for equality
    if op == "qkv":
        n, Hq, Hkv = case["n"], case["Hq"], case["Hkv"]
        x = s["qkv"].double().reshape(n, Hq + 2 * Hkv, HD)
        inv = s["inv"].double()
        pos = s["pos"].double().reshape(-1, n)
        ang = torch.empty(n, HD // 2, dtype=torch.float64, device=x.device)
        for f in range(HD // 2):
            a = 1 if f % 3 == 1 and f < 3 * SECTION[1] else 2 if f % 3 == 2 and f < 3 * SECTION[2] else 0
            ang[:, f] = pos[a if pos.shape[0] == 3 else 0] * inv[f]
        q, k, v = s["out"].double(), s["k"].double(), s["v"].double()
        slots = s["slots"].cpu().tolist()
        rows = [t for t in range(n) if slots[t] >= 0]
        at = torch.tensor([slots[t] for t in rows], device=x.device)
        rows = torch.tensor(rows, device=x.device)
        for h in range(Hq + Hkv):
            w = (s["qw"] if h < Hq else s["kw"]).double()
            y = x[:, h] / (x[:, h].pow(2).sum(-1, keepdim=True) / HD + EPS).sqrt() * w
            lo, hi = y[:, :HD // 2], y[:, HD // 2:]
            z = torch.cat((lo * ang.cos() - hi * ang.sin(), hi * ang.cos() + lo * ang.sin()), 1)[rows]
            if h < Hq:
                q[rows, h] = z
            else:
                k[at // page, h - Hq, at % page] = z
        for h in range(Hkv):
            v[at // page, h, at % page] = x[rows, Hq + Hkv + h]
        return dict(q=q, k=k, v=v)
    qn, past = _lengths(case)
    Hq, Hkv = case["Hq"], case["Hkv"]
    G = Hq // Hkv
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    first = 0
    for b, (m, p) in enumerate(zip(qn, past)):
        L = m + p
        rows = 1 if op == "decode" else m
        at = b if op == "decode" else first
        first += m
        if L == 0 or rows == 0:
            continue
        ids = s["table"][b, :-(-L // page)].long()
        for h in range(Hkv):
            k = s["k"][ids, h].reshape(-1, HD)[:L].double()
            v = s["v"][ids, h].reshape(-1, HD)[:L].double()
            for g in range(G):
                sc = s["q"][at:at + rows, h * G + g].double() @ k.T / HD ** 0.5
                if rows > 1:
                    seen = torch.arange(p, L, device="cuda")
                    sc = torch.where(torch.arange(L, device="cuda")[None] <= seen[:, None], sc, -torch.inf)
                out[at:at + rows, h * G + g] = torch.softmax(sc, -1) @ v
    return out
