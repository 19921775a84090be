"""GPU parity of dsa_mla_chunk against a 64-bit reference (tests/_chunk.py): ragged chunks from one
token on, empty sequences, rows before and behind the sequences, pages of every kind, positions
without a row, causal and full masks, tokens that attend nothing, head counts that do and do not
divide a block of rows, splits, strides, the largest offsets, streams and graphs.

Calls of few rows run in workgroups of 32 rows, calls of many in workgroups of 128 (more than 256 of
them always do); `many` adds a sequence of enough tokens to a case, which so runs on the other kernel."""
from __future__ import annotations

import math

import pytest
import torch

from _chunk import SM_SCALE, Chunk, attend64, bf16, check_chunk, fp8_rows, gen
from opfoundry_amd import abi, dsa

pytestmark = pytest.mark.gpu


def cache_of(g, c, fp8, poison=True):
    """The cache's rows; those that no position of a sequence has hold NaN."""
    kv = fp8_rows(g, c.rows) if fp8 else bf16(g, c.rows, 576)
    if poison:
        used = torch.zeros(c.rows, dtype=torch.bool, device=g.device)
        for b in range(c.B):
            at = [r for r in (c.row(b, j) for j in range(c.lens[b])) if r >= 0]
            used[torch.tensor(at, dtype=torch.long, device=g.device)] = True
        kv[~used] = 0xFF if fp8 else float("nan")
    return kv


def run(c, q, kv, **kw):
    out = torch.full((c.T, q.shape[1], 512), 7.0, dtype=torch.bfloat16, device=q.device)
    lse = torch.full((c.T, q.shape[1]), 7.0, dtype=torch.float32, device=q.device)
    dsa.mla_chunk(q, kv, c.indptr, c.seq_lens, SM_SCALE, out, lse, **c.kw, **kw)
    torch.cuda.synchronize()
    other = torch.ones(c.T, dtype=torch.bool, device=q.device)
    other[c.first:c.first + sum(c.new)] = False
    assert bool((out[other] == 7).all()) and bool((lse[other] == 7).all()), "rows of no sequence were written"
    return out, lse


def with_many(new, lens, H, many, n=None):
    """The case with a sequence in front that fills over 300 blocks of 128 rows."""
    n = n or -(-300 * 128 // H)
    return ([n] + new, [n + 9] + lens) if many else (new, lens)


CASES = [
    # new, lens, H, causal, block_size, num_splits, first, pad
    ([1], [1], 128, True, 64, 0, 0, 0),
    ([1], [1500], 128, True, 64, 0, 0, 0),
    ([1], [33], 1, True, 64, 1, 0, 0),
    ([2, 1, 3, 1], [700, 33, 129, 1], 16, True, 64, 0, 0, 0),
    ([3, 0, 5], [31, 40, 5], 40, True, 64, 1, 2, 3),
    ([0, 0], [10, 0], 16, True, 64, 0, 0, 4),
    ([70, 1, 40], [300, 257, 40], 40, True, 64, 0, 0, 0),
    ([20], [20], 128, True, 64, 1, 0, 0),
    ([20], [20], 128, True, 64, 3, 0, 0),
    ([130], [461], 3, True, 64, 1, 0, 1),
    ([9, 8], [100, 64], 96, False, 64, 2, 0, 0),
    ([5], [3], 16, True, 64, 1, 0, 0),          # more tokens than positions: the first attend nothing
    ([5], [3], 16, True, 64, 2, 0, 0),
    ([4, 4], [50, 1], 200, True, 16, 0, 0, 0),
    ([6], [1000], 17, True, 1, 4, 0, 0),        # pages of one row
    ([6], [1000], 17, True, 48, 64, 0, 0),      # pages that no tile divides, the most splits
    ([33], [2113], 64, True, 128, 0, 0, 0),
    ([64], [640], 32, True, 256, 1, 0, 0),
]


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("new,lens,H,causal,bs,ns,first,pad", CASES)
@pytest.mark.parametrize("many", [False, True], ids=["few", "many"])
def test_parity(dev, fp8, new, lens, H, causal, bs, ns, first, pad, many):
    if many and H < 16:
        H, ns = H + 32, min(ns, 2)
    ns = min(ns, 3) if many else ns
    new, lens = with_many(new, lens, H, many)
    g = gen(len(new) * 1000 + H + sum(lens), dev)
    c = Chunk(g, new, lens, bs, first=first, pad=pad, spare=1)
    q, kv = bf16(g, c.T, H, 576), cache_of(g, c, fp8)
    print(f"[case] new={new} lens={lens} H={H} bs={bs} ns={ns} fp8={fp8}", flush=True)
    out, lse = run(c, q, kv, causal=causal, num_splits=ns)
    check_chunk(c, out, lse, attend64(c, q, kv, causal), fp8)


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
def test_many_sequences(dev, fp8):
    """More sequences than one read of their starts covers, several of them without tokens."""
    g = gen(5, dev)
    B = 4200
    new = [(b * 7) % 3 if b % 50 == 0 else 0 for b in range(B)]
    lens = [5 + b % 90 if new[b] else 0 for b in range(B)]
    c = Chunk(g, new, lens, 32, first=1, pad=2)
    q, kv = bf16(g, c.T, 5, 576), cache_of(g, c, fp8, poison=False)
    for ns in (1, 2):
        out, lse = run(c, q, kv, num_splits=ns)
        check_chunk(c, out, lse, attend64(c, q, kv, True), fp8, f"ns={ns}")


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("ns", [1, 3])
@pytest.mark.parametrize("many", [False, True], ids=["few", "many"])
def test_positions_without_a_row(dev, fp8, ns, many):
    """Table entries outside the cache (the first page of one sequence, all of another, a middle page
    of a third) and sequences longer than their table row: skipped, never read."""
    g = gen(6, dev)
    extra = [1700] if many else []                  # 1700 tokens of 24 heads over 384 positions that have pages
    c = Chunk(g, [4, 3, 2, 5] + extra, [200, 150, 130, 400] + extra, 32)
    c.blocks = 12                                   # 384 positions: the ends of the longer ones have no page
    c.table = c.table[:, :12].contiguous()
    c.table[0, 0], c.table[0, 5] = c.rows // 32, -1
    c.table[1, :] = 2 ** 31 - 1
    c.table[2, 1:4] = -(2 ** 31)
    c.kw["block_table"] = c.table
    q, kv = bf16(g, c.T, 24, 576), cache_of(g, c, fp8)
    out, lse = run(c, q, kv, num_splits=ns, max_kv_len=max(c.lens))
    ref = attend64(c, q, kv, True)
    assert bool(torch.isinf(ref[1][4:7]).all())
    check_chunk(c, out, lse, ref, fp8)


@pytest.mark.parametrize("ns", [1, 2])
@pytest.mark.parametrize("many", [False, True], ids=["few", "many"])
def test_longer_than_its_bound_is_nan(dev, ns, many):
    g = gen(7, dev)
    new, lens = ([2, 2] + [1] * 2500, [100, 300] + [40] * 2500) if many else ([2, 2], [100, 300])
    c = Chunk(g, new, lens, 64)
    q, kv = bf16(g, c.T, 16, 576), cache_of(g, c, False)
    out, lse = run(c, q, kv, num_splits=ns, max_kv_len=256)
    check_chunk(c, out, lse, attend64(c, q, kv, True, max_len=256), False)


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("many", [False, True], ids=["few", "many"])
def test_flat_caches_and_strides(dev, fp8, many):
    """Flat caches of padded rows, q and out with gaps, an 8-byte aligned out."""
    g = gen(8, dev)
    c = Chunk(g, *(([3, 7, 2000], [90, 129, 2001]) if many else ([3, 7], [90, 129])), None, flat=2001 if many else 129)
    q = bf16(g, c.T, 24, 640)[:, 2:22, 16:592]
    wide = fp8_rows(g, c.rows) if fp8 else bf16(g, c.rows, 576)
    kv = torch.full((c.rows, 704 if fp8 else 640), 0xFF if fp8 else float("nan"), dtype=wide.dtype, device=dev)
    kv[:, :wide.shape[1]] = wide
    kv = kv[:, :wide.shape[1]]
    for off in (0, 4):
        big = torch.full((c.T, 22, 544), 3.0, dtype=torch.bfloat16, device=dev)
        out = big[:, 1:21, off:512 + off]
        _, lse = dsa.mla_chunk(q, kv, c.indptr, c.seq_lens, SM_SCALE, out, **c.kw, num_splits=1 + off // 2)
        torch.cuda.synchronize()
        check_chunk(c, out, lse, attend64(c, q, kv, True), fp8)
        assert bool((big[:, 0] == 3).all()) and bool((big[:, 21] == 3).all()) and bool((big[..., 512 + off:] == 3).all())


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("many", [False, True], ids=["few", "many"])
def test_scores_of_every_size(dev, fp8, many):
    """Scores that rise far above the first positions' (a running maximum that grows late), lie far below
    zero, differ by hundreds, and queries of every magnitude."""
    g = gen(9, dev)
    c = Chunk(g, *(([40, 1, 5000], [700, 650, 5000]) if many else ([40, 1], [700, 650])), 64)
    q, kv = bf16(g, c.T, 8, 576), cache_of(g, c, fp8)
    q[:, 0] *= 100
    q[:, 1] *= 1e-3
    q[:, 2] *= 1e-30
    q[:, 3] *= 3e4
    ramp = torch.linspace(-400, 400, 700, device=dev)
    rope = kv[:, 528:].view(torch.bfloat16) if fp8 else kv[:, 512:]
    for b in range(2):
        at = torch.tensor([c.row(b, j) for j in range(c.lens[b])], device=dev)
        rope[at, 0] = (ramp[:len(at)] / 10).to(torch.bfloat16)
    q[:, 4, 512], q[:, 5, 512], q[:, 6, 512] = 138.0, -138.0, 1000.0
    for ns in (1, 4):
        out, lse = run(c, q, kv, num_splits=ns)
        check_chunk(c, out, lse, attend64(c, q, kv, True), fp8, f"ns={ns}")


@pytest.mark.parametrize("ns", [1, 2])
@pytest.mark.parametrize("many", [False, True], ids=["few", "many"])
def test_scale_out_of_range_is_nan(dev, ns, many):
    """A 656-byte row whose scale is 128 or more, negative or NaN: NaN for the tokens that attend it."""
    g = gen(10, dev)
    for bad in (128.0, -0.5, float("nan"), float("inf")):
        c = Chunk(g, *(([6, 2, 2400], [300, 80, 2400]) if many else ([6, 2], [300, 80])), 64)
        q, kv = bf16(g, c.T, 16, 576), cache_of(g, c, True)
        ref = attend64(c, q, kv, True)
        kv[c.row(0, 296), 516:520] = torch.tensor([bad], device=dev).view(torch.uint8)
        out, lse = run(c, q, kv, num_splits=ns)
        hit = torch.zeros(c.T, dtype=torch.bool, device=dev)
        hit[2:6] = True                                     # tokens 2..5 are positions 296..299
        assert bool(torch.isnan(out[hit]).all()) and bool(torch.isnan(lse[hit]).all())
        ref[0][hit], ref[1][hit] = float("nan"), float("nan")
        check_chunk(c, out, lse, ref, True)


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("ns", [1, 2])
@pytest.mark.parametrize("value", ["nan", "inf", "-inf"])
@pytest.mark.parametrize("many", [False, True], ids=["few", "many"])
def test_values_that_are_not_finite_stay_with_their_tokens(dev, fp8, ns, value, many):
    """A row with a NaN or infinity, in NoPE or RoPE: the tokens of the same block of rows that do not
    attend it are as if it were not there."""
    g = gen(15, dev)
    for place in (3, 515):
        c = Chunk(g, *(([9, 4, 2400], [300, 70, 2400]) if many else ([9, 4], [300, 70])), 64)
        q, kv = bf16(g, c.T, 16, 576), cache_of(g, c, fp8)
        ref = attend64(c, q, kv, True)
        hit = c.row(0, 295)                                     # tokens 4 .. 8 are positions 295 .. 299
        if fp8 and place < 512:
            kv[hit, place] = 0x7F                               # e4m3 has no infinity
        else:
            rope = kv[:, 528:].view(torch.bfloat16) if fp8 else kv
            rope[hit, place - 512 if fp8 else place] = float(value)
        out, lse = run(c, q, kv, num_splits=ns)
        if value == "nan":
            assert bool(torch.isnan(out[4:9]).all()) and bool(torch.isnan(lse[4:9]).all())
        for x in ref[:2]:
            x[4:9] = float("nan")
        out[4:9], lse[4:9] = float("nan"), float("nan")
        check_chunk(c, out, lse, ref, fp8, f"{place} {value}")


def test_scale_must_be_positive_and_finite(dev):
    g = gen(16, dev)
    c = Chunk(g, [2], [70], 64)
    q, kv = bf16(g, 2, 16, 576), cache_of(g, c, False)
    for scale in (0.0, -0.1, math.inf, math.nan):
        with pytest.raises(abi.DsaError) as e:
            dsa.mla_chunk(q, kv, c.indptr, c.seq_lens, scale, **c.kw)
        assert e.value.code == -3


def test_cache_past_two_gigabytes(dev):
    """Rows whose byte offset passes 32 bits."""
    g = gen(11, dev)
    rows = (5 << 30) // 1152 // 64 * 64
    c = Chunk(g, [3], [200], 64)
    c.rows = rows
    c.table[0, :] = torch.tensor([rows // 64 - 1, 1, rows // 64 - 3, 2], dtype=torch.int32, device=dev)
    kv = torch.empty((rows, 576), dtype=torch.bfloat16, device=dev)
    for j in range(256):
        kv[c.row(0, j)] = bf16(g, 576)
    q = bf16(g, 3, 16, 576)
    out, lse = run(c, q, kv)
    check_chunk(c, out, lse, attend64(c, q, kv, True), False)


def test_repeats_its_bits_on_other_streams_and_in_graphs(dev):
    """The same call twice, on a side stream, and two captured graphs of different calls replayed in turn
    with eager work between, each with the workspace that its capture held."""
    g = gen(12, dev)
    c = Chunk(g, [2, 9], [900, 1300], 64)
    q, kv = bf16(g, c.T, 16, 576), cache_of(g, c, False)
    q2 = bf16(g, c.T, 16, 576)
    want, want2 = run(c, q, kv, num_splits=4), run(c, q2, kv, num_splits=2)
    again = run(c, q, kv, num_splits=4)
    assert torch.equal(want[0], again[0]) and torch.equal(want[1], again[1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    o, l = dsa.mla_chunk(q, kv, c.indptr, c.seq_lens, SM_SCALE, **c.kw, num_splits=4, stream=side)
    side.synchronize()
    assert torch.equal(o, want[0]) and torch.equal(l, want[1])
    graphs = []
    for x, ns in ((q, 4), (q2, 2)):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            res = dsa.mla_chunk(x, kv, c.indptr, c.seq_lens, SM_SCALE, **c.kw, num_splits=ns)
        graphs.append((gr, res))
    for _ in range(3):
        for (gr, res), w in zip(graphs, (want, want2)):
            res[0].zero_()
            gr.replay()
            eager = dsa.mla_chunk(q, kv, c.indptr, c.seq_lens, SM_SCALE, **c.kw, num_splits=4)
            torch.cuda.synchronize()
            assert torch.equal(res[0], w[0]) and torch.equal(res[1], w[1])
            assert torch.equal(eager[0], want[0])


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("B", [3, 330])
def test_agrees_with_the_sparse_decode_of_every_position(dev, fp8, B):
    """Contexts no longer than the top-k: mla_decode over a list of every position attends the same rows."""
    g = gen(13, dev)
    H, s_q = 128, 2
    lens = [700, 64, 1025] if B == 3 else [2 + 7 * b % 300 for b in range(B)]
    c = Chunk(g, [s_q] * B, lens, 64)
    q, kv = bf16(g, c.T, H, 576), cache_of(g, c, fp8)
    out, lse = run(c, q, kv)
    idx = torch.full((B, s_q, max(lens)), -1, dtype=torch.int32, device=dev)
    for b in range(B):
        idx[b, :, :lens[b]] = torch.arange(lens[b], dtype=torch.int32, device=dev)
    od, ld = dsa.mla_decode(q.view(B, s_q, H, 576), kv, idx, SM_SCALE, seq_lens=c.seq_lens, causal=True, **c.kw)
    torch.cuda.synchronize()
    ref = attend64(c, q, kv, True)
    check_chunk(c, out, lse, ref, fp8)
    # Both approximate the same O, so they differ by at most the sum of their bounds: two roundings of the
    # output (2 * 2^-8 |O|; a fixed bar would demand equal bf16 values where |O| >= 4), two of P (bf16 2^-8,
    # fp16 2^-11), fp16 V twice (656-byte rows), the fp32 error E of both scores, and for the sparse path's
    # K in fp16 scores off by up to 2^-11 of big = max_j sum |q k| sm_scale (E = 2^-17 big), which a
    # probability and its sum both carry.
    o, l, A, E, N = ref
    k16 = 2.0 ** -11 * E * 2.0 ** 17 if fp8 else torch.zeros_like(E)
    rel = 4 * 2.0 ** -11 if fp8 else 2 * 2.0 ** -8
    bound = (rel + 2.0 ** -16 + 2 * E + 2 * k16)[..., None] * A + 2 * 2.0 ** -8 * o.abs() + 2.0 ** -23 * (1 + N)
    assert bool(((od.view(c.T, H, 512).double() - out.double()).abs() <= bound).all())
    assert bool(((ld.view(c.T, H).double() - lse.double()).abs() <= 2 * E + k16 + 2.0 ** -19 * (1 + l.abs())).all())


def test_refuses_tensors_of_another_kind(dev):
    g = gen(14, dev)
    c = Chunk(g, [2], [70], 64)
    q, kv = bf16(g, 2, 16, 576), cache_of(g, c, False)

    def call(q=q, kv=kv, indptr=c.indptr, lens=c.seq_lens, **kw):
        return dsa.mla_chunk(q, kv, indptr, lens, SM_SCALE, **{**c.kw, **kw})

    for bad in (dict(q=q.float()), dict(indptr=c.indptr.long())):
        with pytest.raises(TypeError):
            call(**bad)
    for bad in (dict(q=q.cpu()), dict(indptr=c.indptr[:1]), dict(q=q[..., :512]), dict(block_size=None, kv=kv),
                dict(block_table=c.table.view(-1)), dict(out=torch.empty((2, 16, 576), dtype=torch.bfloat16, device=dev)),
                dict(lse=torch.empty((2, 17), device=dev))):
        with pytest.raises(ValueError):
            call(**bad)
    for bad, code in ((dict(num_splits=65), -6), (dict(block_size=0), -2), (dict(max_kv_len=-1), -2)):
        with pytest.raises(abi.DsaError) as e:
            call(**bad)
        assert e.value.code == code
    assert math.isfinite(float(call()[1].sum()))
