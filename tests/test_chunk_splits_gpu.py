"""GPU parity of dsa_mla_chunk's automatic splits, which the device sizes from the lengths of up to 64
sequences: ragged batches of both kernels, loose bounds of the lengths, sequences without tokens or
positions, the counts on both sides of 64 sequences, lengths that change under a captured graph."""
from __future__ import annotations

import random

import pytest
import torch

from _chunk import SM_SCALE, Chunk, attend64, bf16, check_chunk, gen
from opfoundry_amd import dsa
from test_chunk_gpu import cache_of, run

pytestmark = pytest.mark.gpu


def splits(c, H, kv, **kw):
    q = torch.empty((c.T, H, 576), dtype=torch.bfloat16, device=kv.device)
    out = torch.empty((c.T, H, 512), dtype=torch.bfloat16, device=kv.device)
    return dsa.chunk_num_splits(dsa.make_chunk_args(q, kv, c.indptr, c.seq_lens, SM_SCALE, out, None, **c.kw, **kw))


CASES = [
    # new, lens, H, bound (None: the table's), causal
    ([1], [1501], 128, None, True),
    ([1], [70], 128, 60000, True),
    ([1, 1], [5000, 1], 16, None, True),
    ([1, 0, 1, 2], [3000, 500, 31, 2], 16, None, True),
    ([0, 1, 0], [700, 2900, 0], 8, None, True),
    ([3, 1, 4, 2, 1, 3, 2, 4], [4100, 33, 2000, 1, 999, 3000, 64, 1500], 16, None, True),
    ([3, 1, 4, 2, 1, 3, 2, 4], [4100, 33, 2000, 1, 999, 3000, 64, 1500], 16, 300000, True),
    ([40, 1, 99, 7], [1500, 900, 2000, 7], 40, None, True),
    ([200, 3, 150], [2500, 2000, 150], 64, None, True),
    ([200, 3, 150], [2500, 2000, 150], 64, None, False),
    ([5, 5], [3, 4000], 16, None, True),             # a sequence with more tokens than positions
    ([2, 2], [0, 2000], 16, None, True),             # ... and one without any
]


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("new,lens,H,bound,causal", CASES)
def test_ragged(dev, fp8, new, lens, H, bound, causal):
    g = gen(sum(lens) + H, dev)
    c = Chunk(g, new, lens, 64, first=1, pad=2, spare=1)
    q, kv = bf16(g, c.T, H, 576), cache_of(g, c, fp8)
    kw = dict(causal=causal, max_kv_len=bound or max(lens))
    print(f"[case] new={new} lens={lens} H={H} fp8={fp8} at most {splits(c, H, kv, **kw)} splits", flush=True)
    out, lse = run(c, q, kv, **kw)
    check_chunk(c, out, lse, attend64(c, q, kv, causal), fp8)
    again = run(c, q, kv, **kw)
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("B", [2, 5, 16, 63, 64, 65, 100])
@pytest.mark.parametrize("H,hi,most", [(16, 1, 3000), (40, 4, 1200), (128, 2, 700)])
def test_batches(dev, fp8, B, H, hi, most):
    """Batches on both sides of 64 sequences, a quarter of them without tokens; at least one case of each is split."""
    rng = random.Random(B * 1000 + H)
    new = [rng.randint(1, hi) if rng.random() < 0.75 else 0 for _ in range(B)]
    new[0] = 1
    lens = [rng.randint(1, most) for _ in range(B)]
    g = gen(B + H, dev)
    c = Chunk(g, new, lens, 32)
    q, kv = bf16(g, c.T, H, 576), cache_of(g, c, fp8, poison=False)
    print(f"[case] B={B} H={H} fp8={fp8} at most {splits(c, H, kv)} splits", flush=True)
    out, lse = run(c, q, kv)
    check_chunk(c, out, lse, attend64(c, q, kv, True), fp8)


def test_pages_that_end_before_the_bound(dev):
    """Positions past the block table have no row: the splits cover those that have."""
    g = gen(31, dev)
    c = Chunk(g, [1, 2, 1], [900, 2500, 1300], 64)
    c.blocks = 16
    c.table = c.table[:, :16].contiguous()
    c.kw["block_table"] = c.table
    q, kv = bf16(g, c.T, 16, 576), cache_of(g, c, False)
    out, lse = run(c, q, kv, max_kv_len=5000)
    check_chunk(c, out, lse, attend64(c, q, kv, True), False)


def test_longer_than_its_bound_is_nan_among_others(dev):
    g = gen(32, dev)
    c = Chunk(g, [1, 2, 1], [900, 2500, 1300], 64)
    q, kv = bf16(g, c.T, 16, 576), cache_of(g, c, False)
    out, lse = run(c, q, kv, max_kv_len=2000)
    check_chunk(c, out, lse, attend64(c, q, kv, True, max_len=2000), False)


def test_lengths_that_grow_under_a_graph(dev):
    """One captured decode step with a bound of the longest context: each replay reads the lengths of its
    time, and gives the bits of the eager call."""
    g = gen(33, dev)
    c = Chunk(g, [1, 1, 1], [4000, 4000, 4000], 64)
    q, kv = bf16(g, c.T, 16, 576), cache_of(g, c, True)
    lens = torch.ones(3, dtype=torch.int32, device=dev)

    def step():
        return dsa.mla_chunk(q, kv, c.indptr, lens, SM_SCALE, **c.kw, max_kv_len=4000)

    step()
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out, lse = step()
    for now in ([1, 1, 1], [40, 1, 700], [4000, 3, 2000], [4000, 4000, 4000], [0, 5, 64]):
        lens.copy_(torch.tensor(now, dtype=torch.int32))
        out.zero_()
        gr.replay()
        eager = step()
        torch.cuda.synchronize()
        assert torch.equal(out, eager[0]) and torch.equal(lse, eager[1]), now
        c.lens = now
        check_chunk(c, out, lse, attend64(c, q, kv, True), True, str(now))


@pytest.mark.parametrize("tokens", [2, 3000], ids=["few", "many"])
@pytest.mark.parametrize("ns", [1, 2])
def test_large_values_behind_a_low_first_tile(dev, tokens, ns):
    """Scores that rise by 55 (2^80) after the first tile, values of 2^60: the answer is of 2^60, and a sum
    kept against the first tile's maximum would pass the range of fp32."""
    g = gen(34, dev)
    c = Chunk(g, [tokens], [tokens + 200], 64)
    H = 16
    q = torch.zeros((c.T, H, 576), dtype=torch.bfloat16, device=dev)
    q[..., 512:] = 8.0
    kv = bf16(g, c.rows, 576, scale=2.0 ** 60)
    kv[:, 512:] = 0.0
    late = torch.tensor([c.row(0, j) for j in range(100, c.lens[0])], device=dev)
    kv[late, 512:] = 1.5
    out, lse = run(c, q, kv, num_splits=ns)
    assert bool(torch.isfinite(out).all())
    o, l, A, E, N = attend64(c, q, kv, True)
    # (fp32 sums of values of both signs: 2^-24 a term of sum p |v|, which attends all of them alike)
    rel = 2.0 ** -8 + 2.0 ** -17 + E[..., None]
    assert bool(((out.double() - o).abs() <= rel * A + 2.0 ** -8 * o.abs()).all())
    assert bool(((lse.double() - l).abs() <= E + 2.0 ** -20 * (1 + l.abs())).all())
