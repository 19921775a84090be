"""GPU parity of dsa_qk_norm_rope and dsa_kv_append against 64-bit references (tests/_chunk.py), and the
run of the operators as a serving step uses them."""
from __future__ import annotations

import pytest
import torch

from _chunk import E4M3, SM_SCALE, Chunk, attend64, bf16, check_chunk, cos_sin, gen, i32, near_bf16, norm64, rope64
from opfoundry_amd import dsa

pytestmark = pytest.mark.gpu

# fp32 work before the one rounding: at most 32 steps of 2^-24 (the tree of a row's sum, the root, the products)
# of the largest terms that a value is made of; twice the row's largest value bounds them
STEPS = 32 * 2.0 ** -24 * 2


def slack(y):
    return STEPS * float(y.abs().nan_to_num().max()) if y.numel() else 0.0


PREP = [
    # D, T, H, Hk, q_norm, k_norm, norm_dim, rot_off, style, inverse
    (576, 1, 128, 1, "none", "rms", 512, 512, "interleaved", False),
    (576, 5, 3, 2, "rms", "layer", 512, 0, "halves", False),
    (576, 3, 17, 0, "rms", "none", 64, 512, "halves", True),
    (512, 1, 1, 1, "rms", "rms", 512, 448, "interleaved", False),
    (512, 67, 40, 1, "rms", "rms", 512, 448, "interleaved", False),
    (512, 7, 9, 3, "layer", "none", 448, 448, "halves", True),
    (512, 4, 8, 0, "none", "none", 512, 448, "interleaved", True),
    (512, 4, 8, 1, "rms", "rms", 8, 64, None, False),
    (128, 1, 64, 1, "none", "layer", 128, 0, "halves", False),
    (128, 301, 33, 5, "layer", "rms", 128, 64, "interleaved", False),
    (128, 2, 1, 0, "rms", "none", 64, 0, "halves", False),
]


@pytest.mark.parametrize("D,T,H,Hk,qn,kn,nd,off,style,inverse", PREP)
def test_norm_and_rotation(dev, D, T, H, Hk, qn, kn, nd, off, style, inverse):
    g = gen(D + T + H, dev)
    cs = cos_sin(5000, dev)
    pos = torch.randint(0, 5000, (T,), generator=g, device=dev).to(torch.int32)
    q = bf16(g, T, H + 2, D + 24)[:, 1:H + 1, 8:D + 8]          # strides of a view
    k = bf16(g, T, Hk, D, scale=30.0) if Hk else None
    wb = [torch.randn(nd, generator=g, device=dev) for _ in range(4)]
    kw = {}
    if qn != "none":
        kw.update(q_weight=wb[0], q_bias=wb[1] if qn == "layer" else None)
    if kn != "none":
        kw.update(k_weight=wb[2], k_bias=wb[3] if kn == "layer" else None)
    if Hk:
        kw.update(k=k, k_norm=kn)
    q0, k0 = q.clone(), k.clone() if Hk else None
    print(f"[case] D={D} T={T} H={H} Hk={Hk} {qn} {kn} nd={nd} off={off} {style}", flush=True)
    qo, ko = dsa.qk_norm_rope(q, cs, pos, q_norm=qn, norm_dim=nd, rot_off=off, style=style, inverse=inverse, **kw)
    torch.cuda.synchronize()
    assert torch.equal(q, q0) and (not Hk or torch.equal(k, k0))
    turn = cs[pos.long()][:, None]
    y = rope64(norm64(q, qn, nd, 1e-6, kw.get("q_weight"), kw.get("q_bias")), off, turn, style, inverse)
    near_bf16(qo, y, slack(y))
    if Hk:
        y = rope64(norm64(k, kn, nd, 1e-6, kw.get("k_weight"), kw.get("k_bias")), off, turn, style, inverse)
        near_bf16(ko, y, slack(y))
    else:
        assert ko is None


def test_norm_of_values_far_from_zero_and_tiny(dev):
    """A layer norm whose mean is 200 times its spread; an RMS norm of zeros and of values near 2^-60."""
    g = gen(3, dev)
    x = (bf16(g, 6, 4, 128).float() + 200).to(torch.bfloat16)
    y = norm64(x, "layer", 128, 1e-6)
    out, _ = dsa.qk_norm_rope(x, style=None, q_norm="layer")
    # the mean of 128 values near 200 is off by at most 8 steps of 2^-24 of it, and the spread is about 1
    near_bf16(out, y, slack(y) + 8 * 2.0 ** -24 * 200 / 0.5)
    z = torch.zeros((2, 1, 512), dtype=torch.bfloat16, device=dev)
    z[1] = bf16(g, 1, 512, scale=2.0 ** -60)
    out, _ = dsa.qk_norm_rope(z, style=None, q_norm="rms")
    y = norm64(z, "rms", 512, 1e-6)
    near_bf16(out, y, slack(y))


def test_unknown_positions_and_rows_of_no_sequence(dev):
    """A position outside the table: NaN rotated values, the others as ever.  Positions of the chunk:
    rows before and behind the sequences stay."""
    g = gen(4, dev)
    cs = cos_sin(50, dev)
    q = bf16(g, 6, 5, 512)
    pos = i32([0, 49, 50, -1, 2 ** 31 - 1, 7], dev)
    out, _ = dsa.qk_norm_rope(q, cs, pos, q_norm="rms")
    y = rope64(norm64(q, "rms", 512, 1e-6), 448, cs[pos.long().clamp(0, 49)][:, None], "interleaved")
    y[2:5, :, 448:] = float("nan")
    near_bf16(out, y, slack(y))
    c = Chunk(g, [2, 0, 3], [20, 0, 3], 64, first=1, pad=2)
    q, k = bf16(g, c.T, 20, 576), bf16(g, c.T, 1, 576)
    qo, ko = torch.full_like(q, 5.0), torch.full_like(k, 5.0)
    dsa.qk_norm_rope(q, cs, k=k, k_norm="rms", q_indptr=c.indptr, seq_lens=c.seq_lens, q_out=qo, k_out=ko)
    torch.cuda.synchronize()
    for x, o, n in ((q, qo, "none"), (k, ko, "rms")):
        y = torch.full_like(x, 5.0).double()
        for t, b, p in c.tokens():
            y[t] = rope64(norm64(x[t], n, 512, 1e-6), 512, cs[p], "interleaved")
        near_bf16(o, y, slack(y))


def test_in_place_and_empty(dev):
    g = gen(5, dev)
    cs = cos_sin(64, dev)
    for D, H in ((576, 11), (512, 16), (128, 37)):
        x = bf16(g, 9, H, D)
        pos = torch.arange(9, dtype=torch.int32, device=dev)
        want, _ = dsa.qk_norm_rope(x, cs, pos, q_norm="rms", style="halves")
        y = x.clone()
        dsa.qk_norm_rope(y, cs, pos, q_norm="rms", style="halves", q_out=y)
        assert torch.equal(y, want)
        y = x.clone()
        plain, _ = dsa.qk_norm_rope(x, cs, pos)
        dsa.qk_norm_rope(y, cs, pos, q_out=y)
        assert torch.equal(y, plain)
    assert dsa.qk_norm_rope(bf16(g, 0, 4, 512), cs, i32([], dev))[0].shape == (0, 4, 512)
    assert dsa.qk_norm_rope(bf16(g, 3, 0, 512), cs, i32([1, 2, 3], dev))[0].shape == (3, 0, 512)


# ------------------------------------------------------------------ append

def empty_cache(fmt, rows, dev):
    u8 = torch.uint8
    if fmt in ("bf16", "v4"):
        return (torch.full((rows, 576 if fmt == "bf16" else 512), 9.0, dtype=torch.bfloat16, device=dev),)
    if fmt == "fp8":
        return (torch.full((rows, 656), 0x5A, dtype=u8, device=dev),)
    rope = torch.full((rows, 64), 9.0, dtype=torch.bfloat16, device=dev)
    nope = torch.full((rows, 512), 0x5A, dtype=u8, device=dev)
    return (nope, torch.full((rows, 16), 0x5A, dtype=u8, device=dev), rope) if fmt == "mx" else (nope, rope)


def near_e4m3(codes, want, what):
    """codes (bytes) are `want` (in units of the scale) rounded once after fp32 work (32 steps)."""
    got = codes.view(E4M3).double()
    bound = torch.maximum(2.0 ** -4 * want.abs(), torch.full_like(want, 2.0 ** -10)) + 448 * 64 * 2.0 ** -24
    assert bool(((got - want).abs() <= bound).all()), what


def check_row(fmt, cache, at, y):
    """The written rows `at` against the values y [n, 576 or 512]."""
    split = y.shape[1] - 64
    near = slack(y)
    if fmt in ("bf16", "v4"):
        near_bf16(cache[0][at], y, near)
        return
    if fmt == "fp8":
        r = cache[0][at]
        sc = r[:, 512:528].contiguous().view(torch.float32).double()
        amax = y[:, :512].view(-1, 4, 128).abs().amax(2)
        assert bool(((sc - amax / 448).abs() <= 40 * 2.0 ** -24 * amax / 448).all())
        unit = torch.where(sc > 0, sc, torch.ones_like(sc)).repeat_interleave(128, 1)
        near_e4m3(r[:, :512].contiguous(), y[:, :512] / unit, fmt)
        near_bf16(r[:, 528:].contiguous().view(torch.bfloat16), y[:, 512:], near)
        return
    n = split // 32
    by = cache[1][at] if fmt == "mx" else cache[0][at][:, 448:462]
    amax = y[:, :split].reshape(-1, n, 32).abs().amax(2)
    e = by.double() - 127
    # the least power of two at or above amax / 448, but for fp32 work of amax
    some = amax > 0
    assert bool((amax[some] <= 448 * torch.exp2(e[some]) * (1 + 2.0 ** -18)).all())
    assert bool((amax[some] > 224 * torch.exp2(e[some]) * (1 - 2.0 ** -18)).all()) and bool((e[~some] == 0).all())
    near_e4m3(cache[0][at][:, :split].contiguous(), y[:, :split] / torch.exp2(e).repeat_interleave(32, 1), fmt)
    near_bf16(cache[-1][at], y[:, split:], near)


@pytest.mark.parametrize("fmt", ["bf16", "fp8", "v4", "mx", "v4fp8"])
@pytest.mark.parametrize("new,lens,bs,norm,style,first,pad", [
    ([1], [1], 64, True, "interleaved", 0, 0),
    ([1], [777], 64, True, "interleaved", 0, 0),
    ([3, 0, 5, 70], [3, 9, 40, 200], 16, True, "halves", 2, 3),
    ([40], [2000], 48, False, None, 0, 0),
    ([9, 9], [64, 128], 1, False, "interleaved", 0, 1),
])
def test_append(dev, fmt, new, lens, bs, norm, style, first, pad):
    g = gen(sum(lens) + bs, dev)
    c = Chunk(g, new, lens, bs, first=first, pad=pad, spare=2)
    W = 512 if fmt in ("v4", "v4fp8") else 576
    x = bf16(g, c.T, W + 8)[:, :W]
    x[:, 100:140] *= 2.0 ** -20
    if norm is False:
        x[:, 256:384] = 0
    w = 1 + 0.2 * torch.randn(512, generator=g, device=dev) if norm else None
    ik, iw, ib = bf16(g, c.T, 128), torch.randn(128, generator=g, device=dev), torch.randn(128, generator=g, device=dev)
    cache, icache = empty_cache(fmt, c.rows, dev), torch.full((c.rows, 128), 9.0, dtype=torch.bfloat16, device=dev)
    before = [t.clone() for t in cache]
    cs = cos_sin(2100, dev)
    print(f"[case] append {fmt} new={new} lens={lens} bs={bs}", flush=True)
    dsa.kv_append(x, cache if len(cache) > 1 else cache[0], c.indptr, c.seq_lens, cs, **c.kw, weight=w, style=style,
                  index_k=ik, index_cache=icache, index_norm="layer", index_weight=iw, index_bias=ib)
    torch.cuda.synchronize()
    tok = list(c.tokens())
    at = torch.tensor([c.row(b, p) for _, b, p in tok], device=dev)
    ts, ps = torch.tensor([t for t, _, _ in tok], device=dev), torch.tensor([p for _, _, p in tok], device=dev)
    y = rope64(norm64(x[ts], "rms" if norm else "none", 512, 1e-6, w), W - 64, cs[ps], style)
    check_row(fmt, cache, at, y)
    iy = rope64(norm64(ik[ts], "layer", 128, 1e-6, iw, ib), 0, cs[ps], "halves")
    near_bf16(icache[at], iy, slack(iy))
    rest = torch.ones(c.rows, dtype=torch.bool, device=dev)
    rest[at] = False
    for t, was in zip(cache, before):
        assert torch.equal(t[rest], was[rest]), "a row of no token was written"
    if fmt == "v4fp8":
        assert bool((cache[0][:, 462:] == 0x5A).all())
    assert bool((icache[rest] == 9).all())


def test_append_gives_the_quantiser_s_bytes(dev):
    """656-byte rows of ready values: the bytes of dsa_kv_quantize_fp8, whatever the values."""
    g = gen(20, dev)
    x = bf16(g, 200, 576) * torch.exp2(torch.randint(-30, 30, (200, 576), generator=g, device=dev)).to(torch.bfloat16)
    x[3, :128], x[4, 5], x[5, 300], x[6, 0:512] = 0, float("inf"), float("nan"), -0.0
    x[7] *= 2.0 ** -100
    x[8] = (x[8].float().clamp(-2, 2) * 2.0 ** -126).to(torch.bfloat16)
    x[9, 7], x[9, 200] = float("-inf"), 3e38
    want = dsa.quantize_kv_fp8(x.contiguous())
    c = Chunk(g, [200], [200], None, flat=200)
    got = torch.zeros((200, 656), dtype=torch.uint8, device=dev)
    dsa.kv_append(x, got, c.indptr, c.seq_lens, **c.kw, style=None)
    torch.cuda.synchronize()
    assert torch.equal(got, want)


def test_append_power_of_two_scales_exactly(dev):
    """MXFP8 of ready values: the scale bytes and codes by exact arithmetic, NaN codes for NaN values."""
    g = gen(21, dev)
    x = bf16(g, 64, 576) * torch.exp2(torch.randint(-60, 60, (64, 18), generator=g, device=dev)).to(
        torch.bfloat16).repeat_interleave(32, 1)
    x[0, :32], x[1, :32], x[2, 3], x[3, :32] = 0, 448.0, float("nan"), 450.0
    c = Chunk(g, [64], [64], 32)
    cache = empty_cache("mx", c.rows, dev)
    dsa.kv_append(x, cache, c.indptr, c.seq_lens, **c.kw, style=None)
    torch.cuda.synchronize()
    at = torch.tensor([c.row(0, p) for p in range(64)], device=dev)
    v = x[:, :512].double().view(64, 16, 32)
    amax = v.abs().nan_to_num().amax(2)
    e = torch.where(amax > 0, torch.ceil(torch.log2(amax / 448)), torch.zeros_like(amax))
    assert torch.equal(cache[1][at].double(), e + 127)
    codes = (v * torch.exp2(-e)[..., None]).float().view(64, 512).to(E4M3)
    got = cache[0][at].view(E4M3)
    assert torch.equal(torch.isnan(got.float()), torch.isnan(codes.float()))
    assert torch.equal(got.float().nan_to_num(), codes.float().nan_to_num())
    assert torch.equal(cache[2][at], x[:, 512:])


def test_append_skips_positions_without_a_row(dev):
    """Entries outside the cache, positions past the table's row, negative positions, a flat cache's end."""
    g = gen(22, dev)
    c = Chunk(g, [6, 4, 3], [6, 70, 1], 32)           # the last sequence: two tokens before position 0
    c.blocks = 2                                       # positions from 64 on have no page
    c.table = c.table[:, :2].contiguous()
    c.table[0, 0] = -1
    cache = torch.full((c.rows, 576), 9.0, dtype=torch.bfloat16, device=dev)
    x = bf16(g, c.T, 576)
    dsa.kv_append(x, cache, c.indptr, c.seq_lens, block_table=c.table, block_size=32, style=None)
    torch.cuda.synchronize()
    want = torch.full_like(cache, 9.0)
    want[c.row(2, 0)] = x[12]
    assert torch.equal(cache, want)
    f = Chunk(g, [3, 2], [10, 9], None, flat=8)
    cache = torch.full((16, 576), 9.0, dtype=torch.bfloat16, device=dev)
    x = bf16(g, 5, 576)
    dsa.kv_append(x, cache, f.indptr, f.seq_lens, kv_batch_stride=8, style=None)
    torch.cuda.synchronize()
    want = torch.full_like(cache, 9.0)
    want[7], want[15] = x[0], x[3]
    assert torch.equal(cache, want)


def test_append_past_two_gigabytes_and_padded_rows(dev):
    g = gen(23, dev)
    rows = (5 << 30) // 1280
    c = Chunk(g, [2], [rows], None, flat=0)
    cache = torch.empty((rows, 640), dtype=torch.bfloat16, device=dev)
    cache[-3:] = 9.0
    x = bf16(g, 2, 576)
    dsa.kv_append(x, cache[:, :576], c.indptr, c.seq_lens, style=None)
    torch.cuda.synchronize()
    assert torch.equal(cache[-2:, :576], x) and bool((cache[-3] == 9).all()) and bool((cache[-2:, 576:] == 9).all())


def test_append_many_sequences_and_unknown_position(dev):
    """5000 sequences, one token each in every third; a table of angles shorter than the positions."""
    g = gen(24, dev)
    B = 5000
    new = [1 if b % 3 == 0 else 0 for b in range(B)]
    lens = [1 + b % 40 for b in range(B)]
    c = Chunk(g, new, lens, 8)
    x, cs = bf16(g, c.T, 576), cos_sin(30, dev)
    cache = torch.zeros((c.rows, 576), dtype=torch.bfloat16, device=dev)
    dsa.kv_append(x, cache, c.indptr, c.seq_lens, cs, **c.kw)
    torch.cuda.synchronize()
    tok = list(c.tokens())
    at = torch.tensor([c.row(b, p) for _, b, p in tok], device=dev)
    ps = torch.tensor([p for _, _, p in tok], device=dev)
    y = rope64(x.double(), 512, cs[ps.clamp(max=29)], "interleaved")
    y[ps >= 30, 512:] = float("nan")
    near_bf16(cache[at], y, slack(y))


# ------------------------------------------------------------------ together

@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
def test_serving_steps(dev, fp8):
    """A layer's three steps over ragged sequences: a prompt chunk, another, single tokens.  Each norms and
    rotates its queries, appends its latent rows, and attends the cache; the result is that of one pass over
    all tokens' rows.  The index keys feed the scorer and the selection, which below the top-k keeps every
    position, so the sparse decode of the last step agrees."""
    g = gen(30, dev)
    B, H, bs = 3, 16, 32
    steps = [[20, 0, 70], [5, 33, 64], [1, 1, 1]]
    total = [sum(s[b] for s in steps) for b in range(B)]
    cs = cos_sin(256, dev)
    w, iw, ib = (1 + 0.1 * torch.randn(n, generator=g, device=dev) for n in (512, 128, 128))
    blocks = -(-max(total) // bs)
    table = torch.randperm(B * blocks, generator=g, device=dev).to(torch.int32).view(B, blocks)
    cache = torch.zeros((B * blocks, bs, 656 if fp8 else 576), dtype=torch.uint8 if fp8 else torch.bfloat16, device=dev)
    icache = torch.zeros((B * blocks, bs, 128), dtype=torch.bfloat16, device=dev)
    done = [0] * B
    for new in steps:
        done = [d + n for d, n in zip(done, new)]
        c = Chunk(g, new, done, bs)
        c.table, c.blocks, c.rows = table, blocks, B * blocks * bs
        c.kw = dict(block_table=table)                     # the page size comes from the cache's shape
        chunk = dict(q_indptr=c.indptr, seq_lens=c.seq_lens)
        q, x, ik = bf16(g, c.T, H, 576), bf16(g, c.T, 576), bf16(g, c.T, 128)
        qr, _ = dsa.qk_norm_rope(q, cs, **chunk)
        dsa.kv_append(x, cache, c.indptr, c.seq_lens, cs, block_table=table, weight=w, index_k=ik, index_cache=icache,
                      index_norm="layer", index_weight=iw, index_bias=ib)
        out, lse = dsa.mla_chunk(qr, cache, c.indptr, c.seq_lens, SM_SCALE, block_table=table)
        torch.cuda.synchronize()
        flat = cache.view(-1, cache.shape[-1])
        check_chunk(c, out, lse, attend64(c, qr, flat, True), fp8)
        # the rows just written hold the normed and rotated values
        tok = list(c.tokens())
        at = torch.tensor([c.row(b, p) for _, b, p in tok], device=dev)
        ps = torch.tensor([p for _, _, p in tok], device=dev)
        check_row("fp8" if fp8 else "bf16", (flat,), at, rope64(norm64(x, "rms", 512, 1e-6, w), 512, cs[ps], "interleaved"))
    iq = bf16(g, B, 32, 128)
    iqr, _ = dsa.qk_norm_rope(iq, cs, i32([n - 1 for n in total], dev), style="halves")
    scores = dsa.indexer_scores(iqr.view(B, 1, 32, 128), torch.rand((B, 1, 32), generator=g, device=dev), icache,
                                c.seq_lens, block_table=table, causal=True, n_cols=256)
    idx = dsa.topk_indices(scores.view(B, -1), 256, c.seq_lens).view(B, 1, 256)
    so, _ = dsa.mla_decode(qr.view(B, 1, H, 576), cache, idx, SM_SCALE, seq_lens=c.seq_lens, block_table=table, causal=True)
    torch.cuda.synchronize()
    # the same rows attended twice: the bound of tests/test_chunk_gpu.py's comparison with the sparse decode
    o, _, A, E, N = attend64(c, qr, flat, True)
    k16 = 2.0 ** -11 * E * 2.0 ** 17 if fp8 else torch.zeros_like(E)
    rel = 4 * 2.0 ** -11 if fp8 else 2 * 2.0 ** -8
    bound = (rel + 2.0 ** -16 + 2 * E + 2 * k16)[..., None] * A + 2 * 2.0 ** -8 * o.abs() + 2.0 ** -23 * (1 + N)
    assert bool(((so.view(B, H, 512).double() - out.double()).abs() <= bound).all())


def test_steps_replay_in_a_graph(dev):
    """The three operators captured once, replayed as the sequences grow: lengths and rows are read on the
    device, so a replay follows them."""
    g = gen(31, dev)
    B, H, bs = 4, 16, 16
    cs = cos_sin(128, dev)
    table = torch.randperm(B * 8, generator=g, device=dev).to(torch.int32).view(B, 8)
    cache = torch.zeros((B * 8, bs, 576), dtype=torch.bfloat16, device=dev)
    indptr, lens = i32(list(range(B + 1)), dev), i32([3, 40, 77, 1], dev)
    q, x = torch.zeros((B, H, 576), dtype=torch.bfloat16, device=dev), torch.zeros((B, 576), dtype=torch.bfloat16, device=dev)

    def step():
        qr, _ = dsa.qk_norm_rope(q, cs, q_indptr=indptr, seq_lens=lens)
        dsa.kv_append(x, cache, indptr, lens, cs, block_table=table)
        return dsa.mla_chunk(qr, cache, indptr, lens, SM_SCALE, block_table=table)

    step()
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out, lse = step()
    for _ in range(4):
        lens += 1
        q.copy_(bf16(g, B, H, 576))
        x.copy_(bf16(g, B, 576))
        gr.replay()
        torch.cuda.synchronize()
        got, got_l = out.clone(), lse.clone()
        o, l = step()
        torch.cuda.synchronize()
        assert torch.equal(o, got) and torch.equal(l, got_l)
