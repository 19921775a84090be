"""GPU parity of each kernel on 400-byte rows (16, 32 and 128 heads or rows a workgroup, over lists and dense) where a
split is longer than a span of 2048 entries or positions: other rows in each span, scores that make rows start again, and rows
that are not finite in every kind of place.  Each case asserts the kernel that it runs in (tests/_fp4_kernels.py)."""
from __future__ import annotations

import math

import pytest
import torch

import _fp4
from _chunk import SM_SCALE, Chunk, attend64, bf16, gen, i32
from _fp4_kernels import BLOCK_SIZE, CHUNKS, KERNELS, LISTS
from opfoundry_amd import dsa
from test_chunk_gpu import run
from test_fp4_gpu import cache_of

pytestmark = pytest.mark.gpu

ROWS = 6000


def lists_of(g, T, n, holes=True):
    """(indices [T, n], the valid entries of each): distinct rows in any order; every fifth token has entries that are not valid
    strewn in, and token 0 half as many valid ones."""
    dev = g.device
    idx = torch.stack([torch.randperm(ROWS, generator=g, device=dev)[:n] for _ in range(T)]).to(torch.int32)
    if holes:
        out = torch.rand((T, n), generator=g, device=dev) < 0.3
        out[torch.arange(T, device=dev) % 5 != 1] = False
        out[0] = torch.rand(n, generator=g, device=dev) < 0.5
        idx = torch.where(out, torch.where(idx % 2 == 0, -1, ROWS + 5), idx).to(torch.int32)
    return idx, [[j for j in x if 0 <= j < ROWS] for x in idx.tolist()]


def attend_lists(q, kv, idx, ns, heads, causal_entry):
    """The call by either entry point, in the kernel `heads` where it is unsplit."""
    T = q.shape[0]
    if causal_entry:
        a = dsa.make_prefill_args(q, kv, idx, SM_SCALE, q, None, num_splits=ns)
        assert ns != 1 or dsa.prefill_group_heads(a) == heads
        o, l = dsa.mla_prefill(q, kv, idx, SM_SCALE, num_splits=ns)
    else:
        sl = i32([ROWS] * T, q.device)
        a = dsa.make_decode_args(q[:, None], kv, idx[:, None], SM_SCALE, q[:, None], None, seq_lens=sl, num_splits=ns)
        assert ns != 1 or dsa.decode_group_heads(a) == heads
        o, l = dsa.mla_decode(q[:, None], kv, idx[:, None], SM_SCALE, seq_lens=sl, num_splits=ns)
        o, l = o[:, 0], l[:, 0]
    torch.cuda.synchronize()
    return o, l


def loud(q):
    """Queries of every magnitude, and some that look at RoPE's first value."""
    for h, f in enumerate((100, 1e-3, 1e-30, 3e4)):
        q[:, h] *= f
    q[:, 4, 512], q[:, 5, 512], q[:, 6, 512] = 138.0, -138.0, 1000.0
    return q


@pytest.mark.parametrize("heads", KERNELS)
def test_lists_of_several_spans(dev, heads):
    T, H, n = LISTS[heads]
    g = gen(70 + heads, dev)
    kv, q = _fp4.rows(g, ROWS), bf16(g, T, H, 576)
    idx, lists = lists_of(g, T, n)
    at, ref = _fp4.attend_lists64(q, _fp4.as_bf16(kv), lists, H)
    for ns, prefill in ((1, False), (1, True), (2, False), (0, True)):
        o, l = attend_lists(q, kv, idx, ns, heads, prefill)
        _fp4.check(at, o, l, ref, f"ns={ns}")


@pytest.mark.parametrize("heads", KERNELS)
@pytest.mark.parametrize("rising", [True, False], ids=["rising", "shuffled"])
def test_lists_whose_rows_start_again(dev, heads, rising):
    """The largest scores in the last span (rising entries), or anywhere."""
    T, H, n = LISTS[heads]
    g = gen(80 + heads, dev)
    kv, q = _fp4.rows(g, ROWS), loud(bf16(g, T, H, 576))
    kv[:, 272:].view(torch.bfloat16)[:, 0] = torch.linspace(-40, 40, ROWS, device=dev).to(torch.bfloat16)
    idx, lists = lists_of(g, T, n, holes=not rising)
    if rising:
        idx = idx.sort(1).values.contiguous()
        lists = idx.tolist()
    at, ref = _fp4.attend_lists64(q, _fp4.as_bf16(kv), lists, H)
    for ns in (1, 2):
        o, l = attend_lists(q, kv, idx, ns, heads, rising)
        _fp4.check(at, o, l, ref, f"ns={ns}")


@pytest.mark.parametrize("heads", KERNELS)
def test_lists_with_rows_that_are_not_finite(dev, heads):
    """In the first span, in a later one and in the last tile, which is filled up: their tokens are NaN and no others."""
    T, H, n = LISTS[heads]
    n -= 9                                                       # (the last tile has 3 entries)
    g = gen(90 + heads, dev)
    kv, q = _fp4.rows(g, ROWS + 3), bf16(g, T, H, 576)
    kv[ROWS, 260] = 255
    kv[ROWS + 1, 272:274] = torch.tensor([0xC0, 0x7F], dtype=torch.uint8, device=dev)
    kv[ROWS + 2, 259], kv[ROWS + 2, 48:64] = 254, 0x77          # 6 x 2^127 in all of a group
    idx, lists = lists_of(g, T, n, holes=False)
    at, ref = _fp4.attend_lists64(q, _fp4.as_bf16(kv), lists, H)
    hit = {0: (2100, ROWS), 1: (17, ROWS + 1), 2: (n - 1, ROWS + 2), 3: (n - 2, ROWS), 4: (2048, ROWS + 2), T - 1: (4096, ROWS + 1)}
    for t, (e, row) in hit.items():
        idx[t, e] = row
        for x in ref[:2]:
            x[t] = float("nan")
    sl = i32([ROWS + 3] * T, dev)
    for ns in (1, 3):
        a = dsa.make_decode_args(q[:, None], kv, idx[:, None], SM_SCALE, q[:, None], None, seq_lens=sl, num_splits=ns)
        assert ns != 1 or dsa.decode_group_heads(a) == heads
        o, l = dsa.mla_decode(q[:, None], kv, idx[:, None], SM_SCALE, seq_lens=sl, num_splits=ns)
        torch.cuda.synchronize()
        _fp4.check(at, o[:, 0], l[:, 0], ref, f"ns={ns}")


def chunk_of(g, rows):
    new, lens, H = CHUNKS[rows]
    c = Chunk(g, new, lens, BLOCK_SIZE, spare=1)
    return c, bf16(g, c.T, H, 576), cache_of(g, c)


def attend(c, q, kv, ns, rows):
    out = torch.empty((c.T, q.shape[1], 512), dtype=torch.bfloat16, device=q.device)
    a = dsa.make_chunk_args(q, kv, c.indptr, c.seq_lens, SM_SCALE, out, None, num_splits=ns, **c.kw)
    assert ns != 1 or dsa.chunk_group_rows(a) == rows
    return run(c, q, kv, num_splits=ns)


@pytest.mark.parametrize("rows", KERNELS)
def test_chunks_of_several_spans(dev, rows):
    c, q, kv = chunk_of(gen(100 + rows, dev), rows)
    ref = attend64(c, q, _fp4.as_bf16(kv), True)
    for ns in (1, 2, 0):
        out, lse = attend(c, q, kv, ns, rows)
        _fp4.check(c, out, lse, ref, f"ns={ns}")


@pytest.mark.parametrize("rows", KERNELS)
def test_chunks_whose_rows_start_again(dev, rows):
    g = gen(110 + rows, dev)
    c, q, kv = chunk_of(g, rows)
    loud(q)
    rope = kv[:, 272:].view(torch.bfloat16)
    for b, n in enumerate(c.lens):
        at = torch.tensor([c.row(b, j) for j in range(n)], device=dev)
        ramp = torch.linspace(-40, 40, n, device=dev)
        rope[at, 0] = (ramp if b % 2 == 0 else ramp[torch.randperm(n, generator=g, device=dev)]).to(torch.bfloat16)
    ref = attend64(c, q, _fp4.as_bf16(kv), True)
    for ns in (1, 2):
        out, lse = attend(c, q, kv, ns, rows)
        _fp4.check(c, out, lse, ref, f"ns={ns}")


@pytest.mark.parametrize("rows", KERNELS)
def test_chunks_with_rows_that_are_not_finite(dev, rows):
    """A NaN scale in the second span of sequence 0, which all its tokens attend, and a NaN in RoPE at the last position but
    one of the last sequence, which its last two tokens attend."""
    c, q, kv = chunk_of(gen(120 + rows, dev), rows)
    clean = attend64(c, q, _fp4.as_bf16(kv), True)
    last = c.B - 1
    kv[c.row(0, 2100), 259] = 255
    kv[c.row(last, c.lens[last] - 2), 274:276] = torch.tensor([0xC0, 0x7F], dtype=torch.uint8, device=dev)
    for x in clean[:2]:
        x[:c.new[0]], x[c.T - 2:] = float("nan"), float("nan")
    for ns in (1, 2):
        out, lse = attend(c, q, kv, ns, rows)
        _fp4.check(c, out, lse, clean, f"ns={ns}")


@pytest.mark.parametrize("rows", KERNELS)
@pytest.mark.parametrize("at", [5, 2100, -2], ids=["first", "span", "last"])
def test_chunks_with_a_value_past_bf16s_largest(dev, rows, at):
    """Scale byte 253 under one code of 6 (6 x 2^126, infinity in bf16) at dim 100.  By the definition a head whose query is
    positive there has a score of +inf, O and LSE not finite; one whose query is negative a probability of 0, and NaN (0 times
    infinity) at that dim.  In a tile that some rows do not attend, such a row counts as NaN: all of O and LSE may be NaN.
    What is finite is what it is without that row; tokens that do not attend it are as ever."""
    g = gen(130 + rows, dev)
    c, q, kv = chunk_of(g, rows)
    b = c.B - 1
    p = at if at >= 0 else c.lens[b] - 2
    if p >= c.lens[b] - c.new[b] and at >= 0 or p >= c.lens[b]:
        b, p = 0, at
    q[..., 100] = torch.where(q[..., 100] == 0, 1.0, q[..., 100].float()).to(torch.bfloat16)
    hit = c.row(b, p)
    kv[hit, 259], kv[hit, 48:64], kv[hit, 50] = 253, 0, 0x07
    # (without the row: a code of 0 in its place, and the row left out of the sums)
    first = c.first + sum(c.new[:b])
    tokens = [t for t in range(first, first + c.new[b]) if c.lens[b] - c.new[b] + t - first >= p]
    without = kv.clone()
    without[hit, 259] = 0
    bare = _fp4.as_bf16(without)
    ref = list(attend64(c, q, bare, True))
    for t in tokens:
        rest = [c.row(b, j) for j in range(c.lens[b] - c.new[b] + t - first + 1) if j != p]
        _, one = _fp4.attend_lists64(q[t:t + 1], bare, [rest], q.shape[1])
        for x, y in zip(ref, one):
            x[t] = y[0]
    for ns in (1, 2):
        out, lse = attend(c, q, kv, ns, rows)
        o, l = out[tokens], lse[tokens]
        up = q[tokens][..., 100] > 0
        assert bool(o[..., 100].isnan().all()), "an infinite value was left out"
        assert not bool(torch.isfinite(o[up]).any()) and not bool(torch.isfinite(l[up]).any())
        want = [x.clone() for x in ref]
        want[0][tokens] = torch.where(torch.isfinite(o), want[0][tokens], math.nan)
        want[1][tokens] = torch.where(torch.isfinite(l), want[1][tokens], math.nan)
        out[tokens], lse[tokens] = torch.where(torch.isfinite(o), o, math.nan), torch.where(torch.isfinite(l), l, math.nan)
        _fp4.check(c, out, lse, want, f"ns={ns}")
