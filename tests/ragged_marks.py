"""Workloads of the ragged attentions whose answers count keys.

A query row of zeros gives every key it sees the probability 1 / n exactly, and
a V row holds a single 1, in the dim of its 64-key tile.  An output value is
then (keys seen in the tiles of its dim) / n: whole numbers up to the one
division and the rounding to bf16, so a tile that is lost, doubled or taken from
another request moves a value by far more than the bound, however long the
request is.
"""
import torch

from tests import ragged_oracle as ora

HD, TILE = 128, 64


def dim_of(tile, head):
    return (tile + 17 * head) % HD


def pool(lens, Hkv, page, seed=0, width=None):
    """K with random finite rows and V with the marks; every row past a request's
    length is NaN.  (k, v, table)."""
    k, v, table = ora.make_pool(lens, Hkv, page, seed=seed, stale=float("nan"), width=width)
    for b, n in enumerate(lens):
        if n == 0:
            continue
        pos = torch.arange(n)
        pages = torch.tensor(table[b], dtype=torch.long)[pos // page]
        for h in range(Hkv):
            rows = torch.zeros(n, HD)
            rows[pos, dim_of(pos // TILE, h)] = 1.0
            v[pages, h, pos % page] = rows.to(torch.bfloat16)
    return k, v, table


def counts(n, head):
    """Keys of positions [0, n) in the tiles of each dim, fp64 [128]."""
    pos = torch.arange(n)
    return torch.bincount(dim_of(pos // TILE, head), minlength=HD).double()


def expected(seen, Hq, Hkv):
    """fp64 [rows, Hq, 128] for rows that see seen[i] keys (0: zeros)."""
    out = torch.zeros(len(seen), Hq, HD, dtype=torch.float64)
    for i, n in enumerate(seen):
        if n > 0:
            for h in range(Hkv):
                out[i, h * (Hq // Hkv):(h + 1) * (Hq // Hkv)] = counts(n, h) / n
    return out


def bound(want):
    """One rounding to bf16 and two in fp32 (the reciprocal, the product)."""
    return want.abs() * (ora.BF16_HALF + 2.0 ** -22)
