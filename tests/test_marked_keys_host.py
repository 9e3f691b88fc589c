"""CPU: what the marked keys of _marked.py tell: a tile left out, counted twice or
moved past its row's end, and a part of the keys lost, are each far over the bound
that the attention's outputs are held to."""

from __future__ import annotations

import pytest
import torch

from _marked import BOUND, TILE, shares, worst


@pytest.mark.parametrize("n", [40, 700, 9000, 20000, 33000])
def test_a_lost_or_repeated_tile_is_seen(n):
    g = torch.Generator().manual_seed(n)
    q, k = 2 * torch.randn(3, 64, generator=g), torch.randn(n, 64, generator=g)
    pos = torch.tensor([n - 1, n - 2, n - 3])
    ref = shares(q, k, pos)
    assert 0.012 < BOUND < 0.015 and float((ref.sum(-1) - 1).abs().max()) < 1e-12
    assert worst(ref.to(torch.bfloat16), ref) <= 2.0 ** -8 / BOUND
    tiles = -(-n // TILE)
    for tile in sorted({0, 1, tiles // 2, tiles - 1}):
        for times in (0.0, 2.0):
            count = torch.ones(n, dtype=torch.float64)
            count[tile * TILE:(tile + 1) * TILE] = times
            assert worst(shares(q, k, pos, count), ref) > 5, (tile, times)
    for a, b in ((n // 2, n), (0, n // 4), (n // 3, n // 3 + 256)):  # a part of a split row
        count = torch.ones(n, dtype=torch.float64)
        count[a:b] = 0.0
        assert worst(shares(q, k, pos, count), ref) > 5, (a, b)
    if n <= 512 * TILE:  # a key of one position too many: one of its tile's 32 at least (a third of that at 33000)
        assert worst(shares(q, k, pos + 1)[1:], ref[1:]) > 1
