"""GPU parity of dsa_mla_chunk where a token's first position with a row lies anywhere in a tile: pages that no
tile divides, the first of them (or any) without a row, tokens that attend one such position alone."""
from __future__ import annotations

import pytest
import torch

from _chunk import Chunk, attend64, bf16, check_chunk, gen
from test_chunk_gpu import cache_of, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("many", [False, True], ids=["few", "many"])
@pytest.mark.parametrize("bs,gone", [(4, 1), (4, 9), (7, 1), (12, 3), (20, 1), (100, 1), (28, 1), (60, 2)])
@pytest.mark.parametrize("ns", [1, 2])
def test_first_pages_without_a_row(dev, fp8, many, bs, gone, ns):
    """Every token of a sequence, so that each number of positions from none on is attended."""
    g = gen(bs * 10 + gone, dev)
    n = bs * gone + 41
    c = Chunk(g, [n, 1, 1, 1] + ([2400] if many else []), [n, n, bs * gone + 1, bs * gone + 5] + ([2400] if many else []), bs, spare=1)
    c.table[:4, :gone] = torch.tensor([-1, c.rows // bs + 1, 2 ** 31 - 1, -(2 ** 31)], dtype=torch.int32, device=dev)[:, None]
    q, kv = bf16(g, c.T, 16, 576), cache_of(g, c, fp8)
    out, lse = run(c, q, kv, num_splits=ns)
    check_chunk(c, out, lse, attend64(c, q, kv, True), fp8)


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("T,H", [(8, 5), (40, 16), (2600, 16)])
@pytest.mark.parametrize("keep", [0.02, 0.3, 0.9])
def test_single_positions_without_a_row(dev, fp8, T, H, keep):
    """Pages of one row, of which few, some or most are there."""
    g = gen(int(100 * keep) + T, dev)
    c = Chunk(g, [T, 3], [T + 5, 70], 1, spare=1)
    c.table[torch.rand(c.table.shape, generator=g, device=dev) > keep] = -1
    q, kv = bf16(g, c.T, H, 576), cache_of(g, c, fp8)
    for ns in (0, 1, 3):
        out, lse = run(c, q, kv, num_splits=ns)
        check_chunk(c, out, lse, attend64(c, q, kv, True), fp8, f"ns={ns}")
