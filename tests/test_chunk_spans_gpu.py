"""GPU parity of dsa_mla_chunk's 32-row kernel over more positions than one read of the block table covers
(512 positions where pages are no whole tiles, 16384 where they are), and of the calls in front of it with
more sequences than a wave has lanes."""
from __future__ import annotations

import pytest
import torch

from _chunk import SM_SCALE, Chunk, attend64, bf16, check_chunk, cos_sin, gen, near_bf16, norm64, rope64
from opfoundry_amd import dsa
from test_chunk_gpu import cache_of, run
from test_prep_gpu import check_row, empty_cache, slack

pytestmark = pytest.mark.gpu

SPANS = [
    # new, lens, block size, heads
    ([3, 2], [1300, 513], 1, 16),
    ([3, 2], [1300, 1024], 48, 5),
    ([2], [17001], 64, 16),
    ([1, 4], [33000, 16385], 128, 8),
]


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("new,lens,bs,H", SPANS)
@pytest.mark.parametrize("ns", [1, 2])
def test_several_spans(dev, fp8, new, lens, bs, H, ns):
    g = gen(sum(lens) + bs, dev)
    c = Chunk(g, new, lens, bs, spare=1)
    q, kv = bf16(g, c.T, H, 576), cache_of(g, c, fp8)
    out, lse = run(c, q, kv, num_splits=ns)
    check_chunk(c, out, lse, attend64(c, q, kv, True), fp8)


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("n,bs", [(1300, 48), (17001, 64)])
def test_rows_start_again_over_several_spans(dev, fp8, n, bs):
    """Scores that rise by 50 nats from the first position to the last: past what the first tile's maximum serves."""
    g = gen(n, dev)
    c = Chunk(g, [2], [n], bs)
    q, kv = bf16(g, c.T, 16, 576), cache_of(g, c, fp8)
    rope = kv[:, 528:].view(torch.bfloat16) if fp8 else kv[:, 512:]
    at = torch.tensor([c.row(0, j) for j in range(n)], device=dev)
    rope[at, 0] = (torch.linspace(0, 50, n, device=dev) / (8 * SM_SCALE)).to(torch.bfloat16)
    q[..., 512] = 8.0
    for ns in (1, 3):
        out, lse = run(c, q, kv, num_splits=ns)
        check_chunk(c, out, lse, attend64(c, q, kv, True), fp8, f"ns={ns}")


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("n,bs", [(1300, 48), (17001, 64)])
def test_spans_without_pages(dev, fp8, n, bs):
    """The first span has no page, and one in the middle of what follows."""
    g = gen(n + 1, dev)
    c = Chunk(g, [2], [n], bs)
    first = (512 if bs % 32 else 16384) // bs + 1
    c.table[0, :first] = -1
    c.table[0, first + 2:first + 4] = c.rows // bs + 7
    q, kv = bf16(g, c.T, 16, 576), cache_of(g, c, fp8)
    for ns in (1, 2):
        out, lse = run(c, q, kv, num_splits=ns)
        check_chunk(c, out, lse, attend64(c, q, kv, True), fp8, f"ns={ns}")


def ragged(B):
    new = [(0, 1, 3, 1, 2)[b % 5] for b in range(B)]
    return new, [n + 7 * b % 50 for b, n in enumerate(new)]


@pytest.mark.parametrize("fmt", ["bf16", "fp8", "v4fp8"])
@pytest.mark.parametrize("B", [63, 64, 65, 1003])
def test_append_with_index_keys_of_many_sequences(dev, fmt, B):
    """Four tokens' index keys to a wave: of several sequences, and past the last token where T % 4 != 0."""
    g = gen(B, dev)
    new, lens = ragged(B)
    c = Chunk(g, new, lens, 16, first=1, pad=2, spare=1)
    W = 512 if fmt == "v4fp8" else 576
    x, ik = bf16(g, c.T, W), bf16(g, c.T, 128)
    iw, ib, cs = torch.randn(128, generator=g, device=dev), torch.randn(128, generator=g, device=dev), cos_sin(64, dev)
    cache, icache = empty_cache(fmt, c.rows, dev), torch.full((c.rows, 128), 9.0, dtype=torch.bfloat16, device=dev)
    dsa.kv_append(x, cache if len(cache) > 1 else cache[0], c.indptr, c.seq_lens, cs, **c.kw, norm="rms", index_k=ik,
                  index_cache=icache, index_norm="layer", index_weight=iw, index_bias=ib)
    torch.cuda.synchronize()
    tok = list(c.tokens())
    at = torch.tensor([c.row(b, p) for _, b, p in tok], device=dev)
    ts, ps = torch.tensor([t for t, _, _ in tok], device=dev), torch.tensor([p for _, _, p in tok], device=dev)
    check_row(fmt, cache, at, rope64(norm64(x[ts], "rms", 512, 1e-6), W - 64, cs[ps], "interleaved"))
    iy = rope64(norm64(ik[ts], "layer", 128, 1e-6, iw, ib), 0, cs[ps], "halves")
    near_bf16(icache[at], iy, slack(iy))
    rest = torch.ones(c.rows, dtype=torch.bool, device=dev)
    rest[at] = False
    assert bool((icache[rest] == 9).all())
    for t, was in zip(cache, empty_cache(fmt, c.rows, dev)):
        assert torch.equal(t[rest], was[rest])


@pytest.mark.parametrize("D", [128, 512, 576])
@pytest.mark.parametrize("B", [64, 65, 1003])
def test_norm_and_rotation_by_the_positions_of_many_sequences(dev, D, B):
    g = gen(D + B, dev)
    new, lens = ragged(B)
    c = Chunk(g, new, lens, 16, first=2, pad=3)
    cs = cos_sin(64, dev)
    q, k = bf16(g, c.T, 9, D), bf16(g, c.T, 1, D)
    qo, ko = torch.full_like(q, 5.0), torch.full_like(k, 5.0)
    dsa.qk_norm_rope(q, cs, k=k, k_norm="rms", q_indptr=c.indptr, seq_lens=c.seq_lens, q_out=qo, k_out=ko)
    torch.cuda.synchronize()
    off, nd = (0 if D == 128 else D - 64), min(D, 512)
    ts, ps = (torch.tensor(v, device=dev) for v in zip(*[(t, p) for t, _, p in c.tokens()]))
    for x, o, n in ((q, qo, "none"), (k, ko, "rms")):
        y = torch.full_like(x, 5.0).double()
        y[ts] = rope64(norm64(x[ts], n, nd, 1e-6), off, cs[ps][:, None], "interleaved")
        near_bf16(o, y, slack(y))
