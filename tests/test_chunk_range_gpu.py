"""GPU parity of dsa_mla_chunk over values whose sum passes the range of fp32 although their mean does not."""
from __future__ import annotations

import pytest
import torch

from _chunk import SM_SCALE, Chunk, attend64, bf16, gen
from opfoundry_amd import dsa

pytestmark = pytest.mark.gpu


def check_large(c, q, kv, ns):
    out, lse = dsa.mla_chunk(q, kv, c.indptr, c.seq_lens, SM_SCALE, **c.kw, num_splits=ns)
    torch.cuda.synchronize()
    assert bool(torch.isfinite(out).all()) and bool(torch.isfinite(lse).all())
    o, l, A, E, N = attend64(c, q, kv, True)
    # P and the output rounded to bf16, fp32 sums, scores (their error E)
    rel = 2.0 ** -8 + 2.0 ** -17 + E[..., None]
    assert bool(((out.double() - o).abs() <= rel * A + 2.0 ** -8 * o.abs()).all())
    assert bool(((lse.double() - l).abs() <= E + 2.0 ** -20 * (1 + l.abs())).all())


@pytest.mark.parametrize("tokens", [2, 3000], ids=["few", "many"])
@pytest.mark.parametrize("ns", [0, 1, 2])
def test_values_near_the_largest(dev, tokens, ns):
    """Equal scores over values of 2^126 to 1.5 x 2^127, all of one sign: their sum is infinite, their mean is not."""
    g = gen(41, dev)
    c = Chunk(g, [tokens], [tokens + 200], 64)
    q = bf16(g, c.T, 16, 576)
    q[..., :512] = 0
    kv = ((0.5 + torch.rand((c.rows, 576), generator=g, device=dev)) * 2.0 ** 127).to(torch.bfloat16)
    kv[:, 512:] = 0
    check_large(c, q, kv, ns)


@pytest.mark.parametrize("tokens", [2, 3000], ids=["few", "many"])
@pytest.mark.parametrize("ns", [0, 1, 2])
@pytest.mark.parametrize("rise", [8.0, 26.0, 55.0])
def test_large_values_behind_lower_scores(dev, tokens, ns, rise):
    """Scores that rise after the first tile by 8 nats (2^11), 26 (2^37) or 55 (2^79), values of 2^120 of both signs."""
    g = gen(42, dev)
    c = Chunk(g, [tokens], [tokens + 200], 64)
    q = torch.zeros((c.T, 16, 576), dtype=torch.bfloat16, device=dev)
    q[..., 512] = 8.0
    kv = (torch.randn((c.rows, 576), generator=g, device=dev).clamp(-4, 4) * 2.0 ** 120).to(torch.bfloat16)
    kv[:, 512:] = 0
    late = torch.tensor([c.row(0, j) for j in range(100, c.lens[0])], device=dev)
    kv[late, 512] = rise / (8 * SM_SCALE)
    check_large(c, q, kv, ns)
