"""The counting workloads tell any lost or doubled tile (no GPU)."""
import pytest
import torch

from tests import ragged_marks as mk


@pytest.mark.parametrize("n", [1, 64, 700, 4097, 9000, 17009, 20000, 30000, 32768])
@pytest.mark.parametrize("tile", [64, 128])
def test_every_lost_or_doubled_tile_passes_the_bound(n, tile):
    if n <= tile:
        return                                    # nothing is left without its only tile
    c = mk.counts(n, 0)
    want = c / n
    tol = mk.bound(want)
    assert float(c.sum()) == n
    first = torch.arange(0, n, tile)
    lost = torch.zeros(len(first), mk.HD, dtype=torch.float64)
    for part in range(tile // mk.TILE):           # keys of each tile by dim
        at = first + part * mk.TILE
        lost[torch.arange(len(first)), mk.dim_of(at // mk.TILE, 0)] += \
            (n - at).clamp(0, mk.TILE).double()
    size = lost.sum(1, keepdim=True)
    for got in ((c - lost) / (n - size), (c + lost) / (n + size),  # with its share of the sum
                (c - lost) / n, (c + lost) / n):                   # and without
        over = ((got - want).abs() - tol).amax(1)
        assert float(over.min()) > 0, int(over.argmin())


def test_expected_rows_and_heads():
    w = mk.expected([0, 1, 65, 130], 4, 2)
    assert w.shape == (4, 4, 128) and not w[0].any()
    assert w[1, 0, 0] == 1 and w[1, 2, 17] == 1
    assert w[2, 0, 0] == 64 / 65 and w[2, 0, 1] == 1 / 65 and w[3, 3, 18] == 64 / 130
    assert torch.allclose(w[1:].sum(-1), torch.ones(3, 4, dtype=torch.float64))
