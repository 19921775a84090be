"""GPU parity of 400-byte rows (DSA_KV_MXFP4): their writing and reading back (kv_append, kv_read, the latter
for every format), dense attention (mla_chunk) and attention over lists (mla_decode, mla_prefill) against
64-bit references (tests/_chunk.py, tests/_fp4.py)."""
from __future__ import annotations

import math

import pytest
import torch

import _fp4
from _chunk import E4M3, SM_SCALE, Chunk, attend64, bf16, cos_sin, fp8_rows, gen, i32, near_bf16, norm64, rope64
from opfoundry_amd import abi, dsa
from test_chunk_gpu import CASES, run, with_many

pytestmark = pytest.mark.gpu


def used_rows(c):
    used = torch.zeros(c.rows, dtype=torch.bool, device=c.indptr.device)
    for b in range(c.B):
        at = [r for r in (c.row(b, j) for j in range(c.lens[b])) if r >= 0]
        used[torch.tensor(at, dtype=torch.long, device=used.device)] = True
    return used


def cache_of(g, c, poison=True):
    """400-byte rows; those that no position of a sequence has hold NaN."""
    kv = _fp4.rows(g, c.rows)
    if poison:
        kv[~used_rows(c)] = 0xFF
    return kv


# ------------------------------------------------------------------ reading back

def streams(g, fmt, n):
    """A cache of n rows of a format, and its values (float64)."""
    dev = g.device
    if fmt == "fp4":
        r = _fp4.rows(g, n)
        return r, _fp4.values(r)
    if fmt in ("bf16", "v4"):
        r = bf16(g, n, 576 if fmt == "bf16" else 512)
        return r, r.double()
    if fmt == "fp8":
        r = fp8_rows(g, n)
        scale = r[:, 512:528].contiguous().view(torch.float32).double().repeat_interleave(128, 1)
        return r, torch.cat([r[:, :512].contiguous().view(E4M3).double() * scale,
                             r[:, 528:].contiguous().view(torch.bfloat16).double()], 1)
    width = 512 if fmt == "mx" else 448
    codes = torch.randn((n, width), generator=g, device=dev).to(E4M3)
    e = torch.randint(1, 250, (n, width // 32), generator=g, device=dev)
    rope = bf16(g, n, 64)
    val = torch.cat([codes.double() * torch.exp2(e.double() - 127).repeat_interleave(32, 1), rope.double()], 1)
    if fmt == "mx":
        return (codes.view(torch.uint8), e.to(torch.uint8), rope), val
    nope = torch.full((n, 512), 0xFF, dtype=torch.uint8, device=dev)
    nope[:, :448], nope[:, 448:462] = codes.view(torch.uint8), e.to(torch.uint8)
    return (nope, rope), val


def read_want(c, val):
    want = torch.full((c.T, val.shape[1]), 7.0, dtype=torch.float64, device=val.device)
    for t, b, p in c.tokens():
        r = c.row(b, p)
        want[t] = val[r] if r >= 0 else 0.0
    return want


READS = [([1], [1], 64, 0, 0), ([1], [1500], 64, 0, 3), ([333, 0, 7, 64], [333, 10, 100, 64], 64, 2, 1),
         ([3, 9], [2, 9], 16, 0, 0), ([130, 65], [400, 70], 48, 1, 0), ([9], [1000], 1, 0, 0), ([0, 0], [5, 0], 64, 0, 2)]


@pytest.mark.parametrize("fmt", ["fp4", "bf16", "fp8", "mx", "v4", "v4fp8"])
@pytest.mark.parametrize("new,lens,bs,first,pad", READS)
def test_read(dev, fmt, new, lens, bs, first, pad):
    g = gen(len(new) * 100 + sum(lens), dev)
    c = Chunk(g, new, lens, bs, first=first, pad=pad, spare=1)
    cache, val = streams(g, fmt, c.rows)
    width = val.shape[1]
    want = read_want(c, val)
    big = torch.full((c.T, width + 24), 7.0, dtype=torch.bfloat16, device=dev)
    out = big[:, 8:8 + width]
    assert dsa.kv_read(cache, c.indptr, c.seq_lens, out=out, **c.kw) is out
    torch.cuda.synchronize()
    assert bool((big[:, :8] == 7).all()) and bool((big[:, 8 + width:] == 7).all())
    # one rounding of the fp32 product (itself within 2^-24): all but 656-byte rows are exact in bf16
    if fmt == "fp8":
        near_bf16(out, want, 0.0 + 2.0 ** -23 * float(want.abs().max()))
    else:
        assert torch.equal(out.double(), want.to(torch.bfloat16).double())


def test_read_every_code(dev):
    """All 16 codes under all 256 scale bytes."""
    kv = torch.zeros((256, 400), dtype=torch.uint8, device=dev)
    kv[:, :256] = torch.arange(256, dtype=torch.uint8, device=dev)
    kv[:, 256:272] = torch.arange(256, dtype=torch.uint8, device=dev)[:, None]
    out = dsa.kv_read(kv, i32([0, 256], dev), i32([256], dev), 256)
    torch.cuda.synchronize()
    want = _fp4.values(kv).to(torch.bfloat16)
    assert torch.equal(out.isnan(), want.isnan()) and bool(out[255, :512].isnan().all())
    assert torch.equal(out[:255].view(torch.int16), want[:255].view(torch.int16))


def test_read_of_positions_without_a_row_and_padded_rows(dev):
    g = gen(3, dev)
    c = Chunk(g, [70, 40, 30], [70, 60, 200], 16, spare=1)
    c.blocks = 8                                      # positions from 128 on have no page
    c.table = c.table[:, :8].contiguous()
    c.table[0, 1], c.table[1, :] = -1, 2 ** 31 - 1
    c.kw["block_table"] = c.table
    big = torch.full((c.rows, 448), 0xFF, dtype=torch.uint8, device=dev)
    big[:, :400] = _fp4.rows(g, c.rows)
    kv = big[:, :400]
    out = dsa.kv_read(kv, c.indptr, c.seq_lens, c.T, **c.kw)
    torch.cuda.synchronize()
    want = read_want(c, _fp4.values(kv))
    assert torch.equal(out.double(), want) and bool((want[70:] == 0).all()) and bool((want[:16] != 0).any())


def test_read_flat_and_many_sequences(dev):
    g = gen(4, dev)
    new = [b % 5 for b in range(150)]
    c = Chunk(g, new, [n + b % 3 for b, n in enumerate(new)], None, flat=7, first=1, pad=2)
    kv = _fp4.rows(g, c.rows)
    out = torch.full((c.T, 576), 7.0, dtype=torch.bfloat16, device=dev)
    dsa.kv_read(kv.view(150, 7, 400), c.indptr, c.seq_lens, out=out, **c.kw)
    torch.cuda.synchronize()
    assert torch.equal(out.double(), read_want(c, _fp4.values(kv)))


# ------------------------------------------------------------------ writing

def test_append_gives_the_nearest_codes(dev):
    """Without a norm or a rotation the bytes are the definition's: groups of every magnitude, ties, zeros, values
    below the normal range, the largest, infinities and NaN."""
    g = gen(5, dev)
    x = bf16(g, 200, 576)
    x *= torch.exp2(torch.randint(-130, 120, (200, 1), generator=g, device=dev).float()).to(torch.bfloat16)
    x[0] = 0
    x[1, :32], x[1, 32:64] = 1e-40, -0.0
    x[2, :512] = torch.arange(512, device=dev).to(torch.bfloat16) / 64
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0], device=dev)
    x[3, :32] = torch.cat([ties, -ties, ties * (1 + 2 ** -7), ties * (1 - 2 ** -7)])[:32].clamp(-6, 6).to(torch.bfloat16)
    x[4, :512] = math.inf
    x[6, :512] = (torch.linspace(-1, 1, 512, device=dev) * 3.3895e38).to(torch.bfloat16)
    x[5, 7], x[5, 40], x[5, 511] = math.nan, math.inf, -math.inf
    c = Chunk(g, [200], [230], 64, spare=1)
    kv = torch.full((c.rows, 400), 0xA5, dtype=torch.uint8, device=dev)
    before = kv.clone()
    dsa.kv_append(x, kv, c.indptr, c.seq_lens, None, style=None, **c.kw)
    torch.cuda.synchronize()
    at = torch.tensor([c.row(0, 30 + t) for t in range(200)], device=dev)
    codes, scales = _fp4.pack(x[:, :512].double())
    assert torch.equal(kv[at][:, 256:272], scales)
    # (the code of a zero's sign is the value's own)
    assert torch.equal(kv[at][:, :256], codes)
    assert torch.equal(kv[at][:, 272:].contiguous().view(torch.int16), x[:, 512:].contiguous().view(torch.int16))
    before[at] = kv[at]
    assert torch.equal(before, kv), "other rows were written"
    back = dsa.kv_read(kv, c.indptr, c.seq_lens, 200, **c.kw)
    torch.cuda.synchronize()
    assert bool(back[4, :512].isnan().all()) and bool(torch.isfinite(back[6]).all()) and bool(back[5, :64].isnan().all()) and bool(back[5, 480:512].isnan().all())
    assert bool(torch.isfinite(back[5, 64:480]).all())


@pytest.mark.parametrize("new,lens,bs", [([1], [1500], 64), ([2, 0, 3], [2, 9, 100], 64), ([70, 130], [200, 130], 16)])
@pytest.mark.parametrize("style", ["interleaved", "halves"])
def test_append_with_norm_and_rotation(dev, new, lens, bs, style):
    """Codes are the nearest of the 64-bit values but where those lie within the fp32 work's error of a border
    (32 additions and a few roundings more: 2^-18 of a value; of an exponent's border likewise)."""
    g = gen(sum(lens), dev)
    c = Chunk(g, new, lens, bs, first=1, pad=2)
    kv = torch.zeros((c.rows, 400), dtype=torch.uint8, device=dev)
    x, w, cs = bf16(g, c.T, 576), 1 + 0.1 * torch.randn(512, generator=g, device=dev), cos_sin(max(lens), dev)
    dsa.kv_append(x, kv, c.indptr, c.seq_lens, cs, weight=w, eps=1e-6, style=style, **c.kw)
    back = dsa.kv_read(kv, c.indptr, c.seq_lens, c.T, **c.kw)
    torch.cuda.synchronize()
    for t, b, p in c.tokens():
        y = rope64(norm64(x[t], "rms", 512, 1e-6, w), 512, cs[p], style)
        near_bf16(back[t, 512:], y[512:], 2.0 ** -20 * float(x[t, 512:].double().abs().max()))
        row = kv[c.row(b, p)]
        want = []
        for f in (1 - 2.0 ** -18, 1.0, 1 + 2.0 ** -18):
            v = y[None, :512] * f
            codes, s = _fp4.pack(v)
            want.append(_fp4.values(torch.cat([codes[0], s[0], row[272:]]))[:512])
        got = _fp4.values(row)[:512]
        assert bool(((got == want[0]) | (got == want[1]) | (got == want[2])).all())


# ------------------------------------------------------------------ dense attention

@pytest.mark.parametrize("new,lens,H,causal,bs,ns,first,pad", CASES)
@pytest.mark.parametrize("many", [False, True], ids=["few", "many"])
def test_chunk_parity(dev, new, lens, H, causal, bs, ns, first, pad, many):
    if many and H < 16:
        H, ns = H + 32, min(ns, 2)
    ns = min(ns, 3) if many else ns
    new, lens = with_many(new, lens, H, many)
    g = gen(len(new) * 1000 + H + sum(lens), dev)
    c = Chunk(g, new, lens, bs, first=first, pad=pad, spare=1)
    q, kv = bf16(g, c.T, H, 576), cache_of(g, c)
    print(f"[case] new={new} lens={lens} H={H} bs={bs} ns={ns}", flush=True)
    out, lse = run(c, q, kv, causal=causal, num_splits=ns)
    _fp4.check(c, out, lse, attend64(c, q, _fp4.as_bf16(kv), causal))


@pytest.mark.parametrize("ns", [1, 3])
@pytest.mark.parametrize("many", [False, True], ids=["few", "many"])
def test_chunk_positions_without_a_row(dev, ns, many):
    g = gen(6, dev)
    extra = [1700] if many else []
    c = Chunk(g, [4, 3, 2, 5] + extra, [200, 150, 130, 400] + extra, 32)
    c.blocks = 12
    c.table = c.table[:, :12].contiguous()
    c.table[0, 0], c.table[0, 5] = c.rows // 32, -1
    c.table[1, :] = 2 ** 31 - 1
    c.table[2, 1:4] = -(2 ** 31)
    c.kw["block_table"] = c.table
    q, kv = bf16(g, c.T, 24, 576), cache_of(g, c)
    out, lse = run(c, q, kv, num_splits=ns, max_kv_len=max(c.lens))
    _fp4.check(c, out, lse, attend64(c, q, _fp4.as_bf16(kv), True))


@pytest.mark.parametrize("ns", [1, 2])
@pytest.mark.parametrize("many", [False, True], ids=["few", "many"])
def test_chunk_longer_than_its_bound_is_nan(dev, ns, many):
    g = gen(7, dev)
    new, lens = ([2, 2] + [1] * 2500, [100, 300] + [40] * 2500) if many else ([2, 2], [100, 300])
    c = Chunk(g, new, lens, 64)
    q, kv = bf16(g, c.T, 16, 576), cache_of(g, c)
    out, lse = run(c, q, kv, num_splits=ns, max_kv_len=256)
    _fp4.check(c, out, lse, attend64(c, q, _fp4.as_bf16(kv), True, max_len=256))


@pytest.mark.parametrize("many", [False, True], ids=["few", "many"])
def test_chunk_flat_caches_and_strides(dev, many):
    g = gen(8, dev)
    c = Chunk(g, *(([3, 7, 2000], [90, 129, 2001]) if many else ([3, 7], [90, 129])), None, flat=2001 if many else 129)
    q = bf16(g, c.T, 24, 640)[:, 2:22, 16:592]
    wide = torch.full((c.rows, 448), 0xFF, dtype=torch.uint8, device=dev)
    wide[:, :400] = _fp4.rows(g, c.rows)
    kv = wide[:, :400]
    for off in (0, 4):
        big = torch.full((c.T, 22, 544), 3.0, dtype=torch.bfloat16, device=dev)
        out = big[:, 1:21, off:512 + off]
        _, lse = dsa.mla_chunk(q, kv, c.indptr, c.seq_lens, SM_SCALE, out, **c.kw, num_splits=1 + off // 2)
        torch.cuda.synchronize()
        _fp4.check(c, out, lse, attend64(c, q, _fp4.as_bf16(kv), True))
        assert bool((big[:, 0] == 3).all()) and bool((big[:, 21] == 3).all()) and bool((big[..., 512 + off:] == 3).all())


@pytest.mark.parametrize("many", [False, True], ids=["few", "many"])
def test_chunk_scores_of_every_size(dev, many):
    """A running maximum that grows late, scores far below zero, queries of every magnitude."""
    g = gen(9, dev)
    c = Chunk(g, *(([40, 1, 5000], [700, 650, 5000]) if many else ([40, 1], [700, 650])), 64)
    q, kv = bf16(g, c.T, 8, 576), cache_of(g, c)
    for h, f in enumerate((100, 1e-3, 1e-30, 3e4)):
        q[:, h] *= f
    ramp = torch.linspace(-400, 400, 700, device=dev)
    rope = kv[:, 272:].view(torch.bfloat16)
    for b in range(2):
        at = torch.tensor([c.row(b, j) for j in range(c.lens[b])], device=dev)
        rope[at, 0] = (ramp[:len(at)] / 10).to(torch.bfloat16)
    q[:, 4, 512], q[:, 5, 512], q[:, 6, 512] = 138.0, -138.0, 1000.0
    for ns in (1, 4):
        out, lse = run(c, q, kv, num_splits=ns)
        _fp4.check(c, out, lse, attend64(c, q, _fp4.as_bf16(kv), True), f"ns={ns}")


@pytest.mark.parametrize("ns", [1, 2])
@pytest.mark.parametrize("many", [False, True], ids=["few", "many"])
def test_chunk_values_that_are_not_finite_stay_with_their_tokens(dev, ns, many):
    """A NaN scale, a scale under which some codes pass bf16's largest value, and a NaN in RoPE; a scale that high
    whose codes are small is a row like others."""
    g = gen(15, dev)
    for what in ("scale", "high", "rope", "small"):
        c = Chunk(g, *(([9, 4, 2400], [300, 70, 2400]) if many else ([9, 4], [300, 70])), 64)
        q, kv = bf16(g, c.T, 16, 576), cache_of(g, c)
        hit = c.row(0, 295)                                     # tokens 4 .. 8 are positions 295 .. 299
        if what == "scale":
            kv[hit, 259] = 255
        elif what == "rope":
            kv[hit, 274:276] = torch.tensor([0xC0, 0x7F], dtype=torch.uint8, device=dev)
        else:
            kv[hit, 259] = 253
            kv[hit, 48:64] = 0
            kv[hit, 50] = 0x07 if what == "high" else 0x00
            q[..., 96:128] = 0 if what == "small" else q[..., 96:128]
        ref = attend64(c, q, _fp4.as_bf16(kv), True)
        out, lse = run(c, q, kv, num_splits=ns)
        if what in ("scale", "rope"):
            assert bool(torch.isnan(out[4:9]).all()) and bool(torch.isnan(lse[4:9]).all())
        if what != "small":
            for x in ref[:2]:
                x[4:9] = float("nan")
            out[4:9], lse[4:9] = float("nan"), float("nan")
        _fp4.check(c, out, lse, ref, what)


def test_chunk_cache_past_four_gigabytes(dev):
    g = gen(11, dev)
    n = (5 << 30) // 400 // 64 * 64
    c = Chunk(g, [3], [200], 64)
    c.rows = n
    c.table[0, :] = torch.tensor([n // 64 - 1, 1, n // 64 - 3, 2], dtype=torch.int32, device=dev)
    kv = torch.empty((n, 400), dtype=torch.uint8, device=dev)
    at = torch.tensor([c.row(0, j) for j in range(256)], device=dev)
    kv[at] = _fp4.rows(g, 256)
    q = bf16(g, 3, 16, 576)
    out, lse = run(c, q, kv)
    few = torch.zeros((256, 576), dtype=torch.bfloat16, device=dev)
    few[:] = _fp4.as_bf16(kv[at])
    c2, ref = _fp4.attend_lists64(q, few, [range(198), range(199), range(200)], 16)
    _fp4.check(c2, out, lse, ref)
    back = dsa.kv_read(kv, i32([0, 200], dev), c.seq_lens, 200, **c.kw)
    idx = torch.arange(200, dtype=torch.int32, device=dev).expand(1, 3, 200).contiguous()
    o, l = dsa.mla_decode(q[None], kv, idx, SM_SCALE, seq_lens=c.seq_lens, causal=True, **c.kw)
    torch.cuda.synchronize()
    assert torch.equal(back, few[:200])
    _fp4.check(c2, o[0], l[0], ref)


def test_chunk_repeats_its_bits_on_other_streams_and_in_graphs(dev):
    g = gen(12, dev)
    c = Chunk(g, [2, 9], [900, 1300], 64)
    q, kv, q2 = bf16(g, c.T, 16, 576), cache_of(g, c), bf16(g, c.T, 16, 576)
    want, want2 = run(c, q, kv, num_splits=4), run(c, q2, kv, num_splits=2)
    again = run(c, q, kv, num_splits=4)
    assert torch.equal(want[0], again[0]) and torch.equal(want[1], again[1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    o, l = dsa.mla_chunk(q, kv, c.indptr, c.seq_lens, SM_SCALE, **c.kw, num_splits=4, stream=side)
    r = dsa.kv_read(kv, c.indptr, c.seq_lens, c.T, **c.kw, stream=side)
    side.synchronize()
    assert torch.equal(o, want[0]) and torch.equal(l, want[1])
    assert torch.equal(r, dsa.kv_read(kv, c.indptr, c.seq_lens, c.T, **c.kw))
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


# ------------------------------------------------------------------ attention over lists

class Lists:
    """B sequences of s_q tokens, lists of topk entries: shuffled positions, some twice, some not valid."""

    def __init__(self, g, lens, s_q, topk, bs, causal, holes=True, flat=0):
        dev = g.device
        self.B, self.s_q, self.lens = len(lens), s_q, lens
        blocks = max(1, -(-max(lens) // bs)) if bs else 0
        self.rows = (self.B * blocks + 1) * bs if bs else self.B * flat
        self.table = torch.randperm(self.B * blocks + 1, generator=g, device=dev)[:self.B * blocks].to(torch.int32).view(self.B, -1) if bs else None
        idx = torch.full((self.B, s_q, topk), -1, dtype=torch.int32)
        cg = torch.Generator().manual_seed(int(torch.randint(0, 2 ** 30, (1,), generator=g, device=dev)))
        table = self.table.cpu() if bs else None
        self.lists = []
        for b in range(self.B):
            for t in range(s_q):
                n = min(topk, lens[b])
                if n:
                    at = torch.randperm(lens[b], generator=cg)[:n].to(torch.int32)
                    if holes and n > 4:
                        at[1], at[2], at[3] = at[0], -1, lens[b] + 3
                    idx[b, t, :n] = at
                limit = lens[b] - s_q + t + 1 if causal else lens[b]
                rows = []
                for j in idx[b, t].tolist():
                    if 0 <= j < min(limit, lens[b]):
                        rows.append(int(table[b, j // bs]) * bs + j % bs if bs else b * flat + j)
                self.lists.append(rows)
        self.indices, self.seq_lens = idx.to(dev), i32(lens, dev)
        self.kw = dict(block_table=self.table, block_size=bs) if bs else dict(kv_batch_stride=flat)


DECODES = [
    # lens, s_q, H, topk, block_size, causal, num_splits
    ([1500], 1, 128, 2048, 64, True, 0), ([4000, 3000], 1, 128, 2048, 64, True, 0), ([1], 1, 16, 64, 64, True, 0),
    ([0, 40], 1, 16, 64, 64, False, 0), ([0, 40], 2, 16, 64, 64, True, 3), ([700, 33, 5], 3, 40, 512, 64, True, 0),
    ([700, 33, 5], 3, 40, 512, 48, True, 7), ([300] * 9, 2, 96, 128, 1, True, 1), ([2500], 1, 1, 2500, 64, False, 1),
    ([5000], 2, 200, 4321, 128, True, 0), ([5000], 2, 17, 4321, 64, True, 64), ([90] * 70, 1, 128, 100, 64, True, 0),
    ([200] * 300, 1, 64, 64, 64, True, 0), ([600] * 130, 2, 16, 256, 64, True, 0), ([33], 1, 33, 33, 64, True, 2),
]


@pytest.mark.parametrize("lens,s_q,H,topk,bs,causal,ns", DECODES)
def test_decode_parity(dev, lens, s_q, H, topk, bs, causal, ns):
    g = gen(sum(lens) + H, dev)
    c = Lists(g, lens, s_q, topk, bs, causal)
    kv = _fp4.rows(g, c.rows)
    q = bf16(g, c.B * s_q, H, 576)
    print(f"[case] lens={lens[:4]} s_q={s_q} H={H} topk={topk} bs={bs} ns={ns}", flush=True)
    o, l = dsa.mla_decode(q.view(c.B, s_q, H, 576), kv, c.indices, SM_SCALE, seq_lens=c.seq_lens, causal=causal, num_splits=ns, **c.kw)
    torch.cuda.synchronize()
    at, ref = _fp4.attend_lists64(q, _fp4.as_bf16(kv), c.lists, H)
    _fp4.check(at, o.view(-1, H, 512), l.view(-1, H), ref)


@pytest.mark.parametrize("N,ctx,H,topk", [(1, 0, 128, 64), (5, 900, 128, 512), (70, 3, 16, 48), (300, 50, 40, 200), (40, 2100, 128, 2048)])
@pytest.mark.parametrize("ns", [0, 1, 3])
def test_prefill_parity(dev, N, ctx, H, topk, ns):
    g = gen(N + ctx + H, dev)
    kv = _fp4.rows(g, ctx + N)
    q = bf16(g, N, H, 576)
    idx = torch.full((N, topk), -1, dtype=torch.int32, device=dev)
    lists = []
    for i in range(N):
        n = min(topk, ctx + N)
        at = torch.randperm(ctx + N, generator=g, device=dev)[:n]        # (some lie after the token: not attended)
        idx[i, :n] = at.to(torch.int32)
        lists.append([j for j in at.tolist() if j <= ctx + i])
    o, l = dsa.mla_prefill(q, kv, idx, SM_SCALE, causal=True, causal_offset=ctx, num_splits=ns)
    torch.cuda.synchronize()
    at, ref = _fp4.attend_lists64(q, _fp4.as_bf16(kv), lists, H)
    _fp4.check(at, o, l, ref)


def test_decode_strides_flat_caches_and_bad_pages(dev):
    g = gen(21, dev)
    H, s_q = 24, 2
    c = Lists(g, [300, 200], s_q, 96, None, True, flat=300)
    wide = torch.full((c.rows, 416), 0xFF, dtype=torch.uint8, device=dev)
    wide[:, :400] = _fp4.rows(g, c.rows)
    kv = wide[:, :400]
    q = bf16(g, 2, s_q, H + 3, 600)[:, :, 1:H + 1, 8:584]
    at, ref = _fp4.attend_lists64(q.reshape(-1, H, 576), _fp4.as_bf16(kv), c.lists, H)
    for ns in (1, 2):
        big = torch.full((2, s_q, H + 2, 528), 3.0, dtype=torch.bfloat16, device=dev)
        out = big[:, :, 1:H + 1, 4:516]
        _, l = dsa.mla_decode(q, kv, c.indices, SM_SCALE, out, seq_lens=c.seq_lens, causal=True, num_splits=ns, **c.kw)
        torch.cuda.synchronize()
        _fp4.check(at, out.reshape(-1, H, 512), l.view(-1, H), ref)
        assert bool((big[:, :, 0] == 3).all()) and bool((big[..., :4] == 3).all()) and bool((big[..., 516:] == 3).all())
    # table entries outside the cache: skipped, never read
    c = Lists(g, [300, 200], s_q, 96, 16, True, holes=False)
    kv = _fp4.rows(g, c.rows)
    c.table[0, ::2], c.table[1, :] = -1, 2 ** 31 - 1
    lists = [[int(c.table[t // s_q, j // 16]) * 16 + j % 16 for j in c.indices[t // s_q, t % s_q].tolist()
              if 0 <= j < c.lens[t // s_q] - s_q + t % s_q + 1 and t < s_q and (j // 16) % 2] for t in range(4)]
    q = bf16(g, 4, H, 576)
    o, l = dsa.mla_decode(q.view(2, s_q, H, 576), kv, c.indices, SM_SCALE, seq_lens=c.seq_lens, causal=True, **c.kw)
    torch.cuda.synchronize()
    at, ref = _fp4.attend_lists64(q, _fp4.as_bf16(kv), lists, H)
    _fp4.check(at, o.view(-1, H, 512), l.view(-1, H), ref)
    assert bool((o[1] == 0).all()) and bool(torch.isinf(l[1]).all())


@pytest.mark.parametrize("ns", [1, 4])
@pytest.mark.parametrize("H", [16, 128])
def test_decode_scores_of_every_size(dev, ns, H):
    g = gen(22, dev)
    for T in (2, 320):
        kv = _fp4.rows(g, 1024)
        kv[:, 272:].view(torch.bfloat16)[:, 0] = torch.linspace(-40, 40, 1024, device=dev).to(torch.bfloat16)
        q = bf16(g, T, H, 576)
        for h, f in enumerate((100, 1e-3, 1e-30, 3e4)):
            q[:, h] *= f
        q[:, 4, 512], q[:, 5, 512], q[:, 6, 512] = 138.0, -138.0, 1000.0
        n = 700 if T == 2 else 160
        idx = torch.stack([torch.randperm(1024, generator=g, device=dev)[:n].sort().values for _ in range(T)]).to(torch.int32)
        o, l = dsa.mla_decode(q[:, None], kv, idx[:, None], SM_SCALE, seq_lens=i32([1024] * T, dev), num_splits=ns)
        torch.cuda.synchronize()
        at, ref = _fp4.attend_lists64(q, _fp4.as_bf16(kv), idx.tolist(), H)
        _fp4.check(at, o.view(T, H, 512), l.view(T, H), ref)


def test_decode_of_rows_that_are_not_finite(dev):
    """Only the tokens whose lists name such a row are NaN."""
    g = gen(23, dev)
    kv = _fp4.rows(g, 500)
    kv[100, 260], kv[101, 272:274] = 255, torch.tensor([0xC0, 0x7F], dtype=torch.uint8, device=dev)
    q = bf16(g, 6, 40, 576)
    idx = torch.stack([torch.randperm(100, generator=g, device=dev)[:75] for _ in range(6)]).to(torch.int32)
    at, ref = _fp4.attend_lists64(q, _fp4.as_bf16(kv), idx.tolist(), 40)
    idx[1, 70], idx[4, 3] = 100, 101
    for x in ref[:2]:
        x[1], x[4] = float("nan"), float("nan")
    for ns in (1, 2):
        o, l = dsa.mla_decode(q[:, None], kv, idx[:, None], SM_SCALE, seq_lens=i32([500] * 6, dev), num_splits=ns)
        torch.cuda.synchronize()
        _fp4.check(at, o.view(6, 40, 512), l.view(6, 40), ref)


def test_decode_in_graphs_on_streams_and_without_a_workspace(dev):
    g = gen(24, dev)
    H = 128
    c = Lists(g, [3000, 2500], 1, 2048, 64, True)
    kv, q = _fp4.rows(g, c.rows), bf16(g, 2, 1, H, 576)
    call = lambda **kw: dsa.mla_decode(q, kv, c.indices, SM_SCALE, seq_lens=c.seq_lens, causal=True, **c.kw, **kw)  # noqa: E731
    want = call()
    a = dsa.make_decode_args(q, kv, c.indices, SM_SCALE, *want, seq_lens=c.seq_lens, causal=True, **c.kw)
    assert dsa.decode_num_splits(a) > 1
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = call()
    side.synchronize()
    torch.cuda.synchronize()
    assert torch.equal(other[0], want[0]) and torch.equal(other[1], want[1])
    o, l = torch.empty_like(want[0]), torch.empty_like(want[1])
    a.out, a.lse = o.data_ptr(), l.data_ptr()
    import ctypes
    assert abi.load_library().dsa_mla_decode_noalloc(ctypes.byref(a), torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    assert torch.equal(o, want[0]) and torch.equal(l, want[1])
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        res = call()
    for _ in range(3):
        res[0].zero_()
        gr.replay()
        eager = call(num_splits=2)
        torch.cuda.synchronize()
        assert torch.equal(res[0], want[0]) and torch.equal(res[1], want[1]) and bool(torch.isfinite(eager[0]).all())


# ------------------------------------------------------------------ together

def test_a_serving_run(dev):
    """A prompt in two chunks and three decode steps on one 4-bit cache: rows appended, dense attention over them,
    the same as attention over lists of every position, and as the bf16 rows that are read back."""
    g = gen(31, dev)
    H, bs = 16, 64
    lens, cs = [0, 0], cos_sin(400, dev)
    table = torch.randperm(12, generator=g, device=dev).to(torch.int32).view(2, 6)
    kw = dict(block_table=table, block_size=bs)
    kv = torch.full((12 * bs, 400), 0xFF, dtype=torch.uint8, device=dev)
    w = 1 + 0.1 * torch.randn(512, generator=g, device=dev)
    for new in ([100, 33], [120, 200], [1, 1], [1, 2], [2, 1]):
        lens = [a + b for a, b in zip(lens, new)]
        T = sum(new)
        indptr, sl = i32([0, new[0], T], dev), i32(lens, dev)
        dsa.kv_append(bf16(g, T, 576), kv, indptr, sl, cs, weight=w, **kw)
        q = bf16(g, T, H, 576)
        o, l = dsa.mla_chunk(q, kv, indptr, sl, SM_SCALE, **kw)
        rows = dsa.kv_read(kv, i32([0, lens[0], sum(lens)], dev), sl, sum(lens), **kw)
        torch.cuda.synchronize()
        assert bool(torch.isfinite(rows).all())
        lists, flat = [], []
        for b in range(2):
            for i in range(new[b]):
                n = lens[b] - new[b] + i + 1
                lists.append(list(range(b * lens[0], b * lens[0] + n)))
                flat.append([int(table[b, j // bs]) * bs + j % bs for j in range(n)])
        c, ref = _fp4.attend_lists64(q, rows, lists, H)
        _fp4.check(c, o, l, ref, str(new))
        idx = torch.full((T, max(lens)), -1, dtype=torch.int32, device=dev)
        for t, f in enumerate(flat):
            idx[t, :len(f)] = i32(f, dev)
        o2, l2 = dsa.mla_prefill(q, kv, idx, SM_SCALE)
        torch.cuda.synchronize()
        _fp4.check(c, o2, l2, ref, str(new))


def test_refuses_tensors_of_another_kind(dev):
    g = gen(32, dev)
    kv, ip, sl = _fp4.rows(g, 128), i32([0, 70], dev), i32([70], dev)
    for bad, err in ((dict(rows=None), ValueError), (dict(rows=71, out=torch.empty((70, 576), dtype=torch.bfloat16, device=dev)), ValueError),
                     (dict(out=torch.empty((70, 512), dtype=torch.bfloat16, device=dev)), ValueError),
                     (dict(out=torch.empty((70, 576), device=dev)), TypeError), (dict(cache=kv[:, :399]), ValueError),
                     (dict(cache=kv.cpu()), ValueError), (dict(q_indptr=ip.long()), TypeError)):
        with pytest.raises(err):
            dsa.kv_read(**{**dict(cache=kv, q_indptr=ip, seq_lens=sl, rows=70), **bad})
    with pytest.raises(abi.DsaError) as e:      # rows of out over one another
        dsa.kv_read(kv, ip, sl, out=torch.empty((70, 576), dtype=torch.bfloat16, device=dev)[:1].expand(70, 576))
    assert e.value.code == -7
    big = torch.empty((1000, 576), dtype=torch.bfloat16, device=dev)
    with pytest.raises(abi.DsaError) as e:      # out over the cache it reads
        dsa.kv_read(big, ip, sl, out=big[500:570])
    assert e.value.code == -7
    for scale in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(abi.DsaError) as e:
            dsa.mla_decode(bf16(g, 1, 1, 16, 576), kv, torch.zeros((1, 1, 4), dtype=torch.int32, device=dev), scale, seq_lens=sl)
        assert e.value.code == -3
    with pytest.raises(abi.DsaError) as e:
        dsa.mla_decode_csr(bf16(g, 1, 16, 576), kv, i32([0, 4], dev), i32([0, 1, 2, 3], dev), SM_SCALE, max_kv_len=4)
    assert e.value.code == -4


# ------------------------------------------------------------------ the ends of the ranges

def test_calls_of_nothing(dev):
    """No tokens, no entries, no new rows: the outputs of tokens that attend nothing, and nothing else."""
    g = gen(41, dev)
    kv, ip, sl = _fp4.rows(g, 128), i32([0, 2], dev), i32([70], dev)
    assert dsa.kv_read(kv, i32([0, 0], dev), sl, 0).shape == (0, 576)
    o, l = dsa.mla_chunk(bf16(g, 0, 16, 576), kv, i32([0, 0], dev), sl, SM_SCALE)
    assert o.shape == (0, 16, 512) and l.shape == (0, 16)
    for H in (16, 40, 128):
        q = bf16(g, 3, H, 576)
        for topk, ns in ((0, 0), (0, 3), (5, 0), (300, 0), (300, 4)):
            none = torch.full((3, topk), -1, dtype=torch.int32, device=dev)
            for o, l in (dsa.mla_decode(q[:, None], kv, none[:, None], SM_SCALE, seq_lens=i32([128] * 3, dev), num_splits=ns),
                         dsa.mla_prefill(q, kv, none, SM_SCALE, causal=True, causal_offset=100, num_splits=ns)):
                torch.cuda.synchronize()
                assert bool((o == 0).all()) and bool((l == math.inf).all())
        o, l = dsa.mla_prefill(q[:0], kv, torch.zeros((0, 5), dtype=torch.int32, device=dev), SM_SCALE)
        assert o.shape == (0, H, 512) and l.shape == (0, H)
        o, l = dsa.mla_chunk(q[:2], kv, ip, i32([0], dev), SM_SCALE)           # a sequence without positions
        torch.cuda.synchronize()
        assert bool((o == 0).all()) and bool((l == math.inf).all())
    # no new rows: the cache stays as it was
    before = kv.clone()
    dsa.kv_append(bf16(g, 4, 576), kv, i32([0, 0], dev), sl, style=None)
    torch.cuda.synchronize()
    assert torch.equal(kv, before)


@pytest.mark.parametrize("H", [16, 40, 128])
def test_one_position_many_times(dev, H):
    """n times the same entry: its values, and a sum of n."""
    g = gen(42, dev)
    kv, q = _fp4.rows(g, 64), bf16(g, 2, H, 576)
    lists = [[17] * 2500, [3] * 64 + [63]]
    idx = torch.full((2, 2500), -1, dtype=torch.int32, device=dev)
    for t, x in enumerate(lists):
        idx[t, :len(x)] = i32(x, dev)
    at, ref = _fp4.attend_lists64(q, _fp4.as_bf16(kv), lists, H)
    for ns in (0, 1, 5):
        o, l = dsa.mla_prefill(q, kv, idx, SM_SCALE, num_splits=ns)
        torch.cuda.synchronize()
        _fp4.check(at, o, l, ref)


@pytest.mark.parametrize("T,H,n", [(300, 32, 100), (260, 64, 70), (3, 48, 130), (520, 20, 33)])
def test_lists_of_few_heads(dev, T, H, n):
    g = gen(43, dev)
    kv, q = _fp4.rows(g, 900), bf16(g, T, H, 576)
    idx = torch.randint(0, 900, (T, n), generator=g, device=dev).to(torch.int32)
    at, ref = _fp4.attend_lists64(q, _fp4.as_bf16(kv), idx.tolist(), H)
    for ns in (0, 1, 2):
        o, l = dsa.mla_prefill(q, kv, idx, SM_SCALE, num_splits=ns)
        torch.cuda.synchronize()
        _fp4.check(at, o, l, ref)


def test_append_and_read_in_a_graph(dev):
    """A captured step writes and reads what its buffers hold at each replay, with eager calls between."""
    g = gen(44, dev)
    c = Chunk(g, [3, 1], [500, 64], 64, pad=2)
    kv, cs = torch.zeros((c.rows, 400), dtype=torch.uint8, device=dev), cos_sin(600, dev)
    x, w = bf16(g, c.T, 576), 1 + 0.1 * torch.randn(512, generator=g, device=dev)
    step = lambda: (dsa.kv_append(x, kv, c.indptr, c.seq_lens, cs, weight=w, **c.kw),            # noqa: E731
                    dsa.kv_read(kv, c.indptr, c.seq_lens, c.T, **c.kw))[1]
    step()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out = step()
    for seed in (1, 2, 3):
        x.copy_(bf16(gen(seed, dev), c.T, 576))
        c.seq_lens.copy_(i32([500 - seed, 64 - seed], dev))
        out.fill_(9.0)
        gr.replay()
        torch.cuda.synchronize()
        got, cache = out.clone(), kv.clone()
        kv.zero_()
        want = step()
        torch.cuda.synchronize()
        assert torch.equal(got[:4], want[:4]) and bool((got[4:] == 9).all())
        at = torch.tensor([c.row(b, n - seed - k) for b, n, k in ((0, 500, 1), (0, 500, 2), (0, 500, 3), (1, 64, 1))], device=dev)
        assert torch.equal(cache[at], kv[at]) and bool((got[:4] != 0).any())


def test_two_graphs_with_one_workspace(dev):
    """A program's own workspace, of the larger call, under two captured calls in turn."""
    g = gen(45, dev)
    c = Chunk(g, [2, 9], [900, 1300], 64)
    ls = Lists(g, [1300, 1200], 1, 700, 64, True)
    kv, kv2 = cache_of(g, c), _fp4.rows(g, ls.rows)
    q, q2 = bf16(g, c.T, 16, 576), bf16(g, 2, 1, 128, 576)
    ws = torch.empty(64 << 20, dtype=torch.uint8, device=dev)
    calls = (lambda **k: dsa.mla_chunk(q, kv, c.indptr, c.seq_lens, SM_SCALE, num_splits=4, **c.kw, **k),
             lambda **k: dsa.mla_decode(q2, kv2, ls.indices, SM_SCALE, seq_lens=ls.seq_lens, causal=True, num_splits=3, **ls.kw, **k))
    want = [f() for f in calls]
    graphs = []
    for f in calls:
        f(workspace=ws)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            res = f(workspace=ws)
        graphs.append((gr, res))
    for _ in range(3):
        ws.fill_(0xFF)
        for (gr, res), w in zip(graphs, want):
            res[0].zero_()
            gr.replay()
            calls[0](workspace=ws)
            torch.cuda.synchronize()
            assert torch.equal(res[0], w[0]) and torch.equal(res[1], w[1])


@pytest.mark.parametrize("T,H", [(256, 128), (300, 40), (2, 128)])
@pytest.mark.parametrize("scale", [255, 254])
def test_rows_that_are_not_finite_at_a_lists_end(dev, T, H, scale):
    """In a list's last tile, which is filled up, as anywhere else: the tokens that name such a row are NaN."""
    g = gen(46, dev)
    kv, q = _fp4.rows(g, 300), bf16(g, T, H, 576)
    kv[200, 259], kv[200, 48:64] = scale, 0x77          # of dims 96 .. 127: NaN, or 6 x 2^127
    kv[201, 272:274] = torch.tensor([0x80, 0x7F], dtype=torch.uint8, device=dev)
    idx = torch.stack([torch.randperm(200, generator=g, device=dev)[:70] for _ in range(T)]).to(torch.int32)
    lists = idx.tolist()
    if T > 2:
        lists[2] = lists[2][:69]
    at, ref = _fp4.attend_lists64(q, _fp4.as_bf16(kv), lists, H)
    idx[0, 66], idx[1, 3] = 200, 200
    for x in ref[:2]:
        x[0], x[1] = float("nan"), float("nan")
    if T > 2:
        idx[2, 69], idx[T - 1, 0] = 201, 200
        for x in ref[:2]:
            x[T - 1] = float("nan")
            # (an infinite RoPE value, which V does not have: a score of +inf, whose weight is exp(inf - inf), or of
            # -inf, whose weight is 0)
            x[2, q[2, :, 512] > 0] = float("nan")
    for ns in (1, 2):
        o, l = dsa.mla_prefill(q, kv, idx, SM_SCALE, num_splits=ns)
        torch.cuda.synchronize()
        _fp4.check(at, o, l, ref)
