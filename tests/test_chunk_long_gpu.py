"""GPU parity of dsa_mla_chunk over long contexts in which a large share of the weight lies in many positions
of tiny probability each, which 16-bit probabilities must not lose.

The contexts name few cache rows through many table entries, so that the 64-bit result is a sum over the
distinct rows, each with the number of positions that have it."""
from __future__ import annotations

import pytest
import torch

from _chunk import E4M3, SM_SCALE, gen, latent64
from opfoundry_amd import dsa

pytestmark = pytest.mark.gpu

PAGE = 64


def long_case(dev, fp8, pages, at, gap):
    """(cache, table, counts): `pages` pages of 64 positions; every row's score is 0 but for the first of page
    `at`, which lies `gap` above (q = 8 in the first rotated value), has zero values and stands alone.  Pages
    0 and `at` are their own, all others one and the same."""
    g = gen(pages + at, dev)
    nope = (0.5 + torch.rand((3 * PAGE, 512), generator=g, device=dev))
    k = torch.zeros((3 * PAGE, 576), dtype=torch.bfloat16, device=dev)
    k[:, :512] = nope.to(torch.bfloat16)
    sink = PAGE
    k[sink, :512], k[sink, 512] = 0, gap / (8 * SM_SCALE)
    if fp8:
        rows = torch.zeros((3 * PAGE, 656), dtype=torch.uint8, device=dev)
        rows[:, :512] = (nope * 100).to(E4M3).view(torch.uint8)
        rows[sink, :512] = 0
        rows[:, 512:528] = torch.full((3 * PAGE, 4), 0.01, device=dev).view(torch.uint8)
        rows[:, 528:] = k[:, 512:].contiguous().view(torch.uint8)
        k = rows
    table = torch.full((1, pages), 2, dtype=torch.int32, device=dev)
    table[0, 0] = 0
    table[0, at] = 1
    count = torch.zeros(3 * PAGE, dtype=torch.float64, device=dev)
    for e in (0, 1, 2):
        count[e * PAGE:(e + 1) * PAGE] = float((table == e).sum())
    return k, table, count


def check_long(dev, fp8, pages, at, gap, T, H, ns):
    k, table, count = long_case(dev, fp8, pages, at, gap)
    n = pages * PAGE
    q = torch.zeros((T, H, 576), dtype=torch.bfloat16, device=dev)
    q[..., 512] = 8.0
    indptr, lens = (torch.tensor(v, dtype=torch.int32, device=dev) for v in ([0, T], [n]))
    out, lse = dsa.mla_chunk(q, k, indptr, lens, SM_SCALE, block_table=table, block_size=PAGE, causal=False, num_splits=ns)
    torch.cuda.synchronize()
    x = latent64(k)
    s = (q[0, 0].double()[None] * x).sum(1) * SM_SCALE
    has = count > 0
    z = torch.logsumexp(s[has] + count[has].log(), 0)
    p = torch.where(has, count * torch.exp(s - z), 0.0)
    o = p @ x[:, :512]                               # all values are >= 0: this is sum p |v| too
    # Steps of fp32 sums, relative: a lane adds two sums of a row's P a tile of 32 positions to its running one,
    # and the products with V two more to each output's, 2^-24 of it at most each time.
    sums = n / 16 * 2.0 ** -24
    # P rounded (bf16 2^-8, fp16 2^-11) and, in fp16, below its normal range off by 2^-11 of a row's sum in all (the
    # first tile's maximum is attended); V rounded twice (2^-11 each, 656-byte rows); the output's rounding.  The
    # scores are exact products (one term), off by three steps of 2^-24 of the largest, 2^5 at most.
    big = float(x[has, :512].abs().max())
    rel = (3 * 2.0 ** -11 if fp8 else 2.0 ** -8) + 2.0 ** -15 + 2.0 ** -8 + 2 * sums
    bound = rel * o + (2.0 ** -11 * big if fp8 else 0.0)
    worst = float(((out.double() - o).abs() / bound).max())
    assert worst <= 1, f"O off by {worst} of its bound"
    worst = float(((lse.double() - z).abs() / (2.0 ** -15 + sums + 2.0 ** -20 * (1 + z.abs()))).max())
    assert worst <= 1, f"LSE off by {worst} of its bound"


# the sink's weight against all others' together is n e^-gap: 2^20 positions 17.5 below it are 1 to 38,
# and their P against its 1 is 2^-25.2, nothing in fp16
LONG = [
    # pages, the sink's page, gap
    (1 << 14, 1, 17.5),
    (1 << 14, 9000, 17.5),              # it comes late: the rows start again with their largest score
    (1 << 14, 9000, 4.0),               # ... or do not
    (1 << 11, 1, 16.0),
    ((1 << 8) + 1, 200, 10.0),          # just past 2^14 positions
    (1 << 8, 1, 17.0),                  # and at them
    (1 << 8, 200, 10.8),                # P grows to 2^15.6, which fp16 holds
    (1 << 8, 200, 11.2),                # ... and to 2^16.2, which it does not
]


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("ns", [0, 1, 3])
@pytest.mark.parametrize("pages,at,gap", LONG)
def test_many_positions_far_below_one(dev, fp8, pages, at, gap, ns):
    check_long(dev, fp8, pages, at, gap, 2, 16, ns)


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("pages,at,gap", [LONG[0], LONG[1], LONG[4]])
def test_many_positions_far_below_one_of_many_rows(dev, fp8, pages, at, gap):
    """Over 128 blocks of 128 rows, as many workgroups as run at once on 256 CUs two rounds of the 32-row ones."""
    check_long(dev, fp8, pages, at, gap, 1100, 16, 1)
