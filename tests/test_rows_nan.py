"""A NaN among a token's latent values is a NaN in its cache row, whatever the values beside it: a group of
a 656-byte row in which nothing else is larger than zero has scale 0 and keeps its NaN codes, so that every
token that attends the row is NaN, as with the other formats.  (An RMS norm makes such groups: one NaN under
it makes all 512 values NaN, one infinity itself NaN and the others 0.)"""
from __future__ import annotations

import numpy as np
import pytest
import torch

import oracle
from _chunk import E4M3, SM_SCALE, Chunk, bf16, cos_sin, gen, norm64, rope64
from opfoundry_amd import dsa

NAN, INF = float("nan"), float("inf")


def odd_rows():
    """fp32 rows of 576: groups of NaNs only, of both signs; a NaN among zeros; a NaN among values; an infinity."""
    rng = np.random.default_rng(5)
    x = oracle.bf16_to_f32(oracle.normal_bf16(rng, (8, 576)))
    x[0, :512] = NAN
    x[1, 128:256] = NAN
    x[1, 130] = -NAN
    x[2, :128], x[2, 17] = 0.0, NAN
    x[3, 384:512], x[3, 400] = -0.0, -NAN
    x[4, 300] = NAN
    x[5, 5] = INF
    x[6, :512] = 0.0
    x[7, 560] = NAN                                  # a rotated value, no part of any group
    return x


def test_oracle_rows_keep_nan():
    x = odd_rows()
    rows = oracle.quantize_rows_656(x)
    back = oracle.dequant_rows_656(rows)
    want = np.isnan(x)
    want[5, :128] |= np.isinf(x[5, :128])            # inf / inf; the group's scale is infinite
    with np.errstate(invalid="ignore"):
        got = np.isnan(back)
    got[5, :128] &= want[5, :128]                    # (0 times that scale: NaN too)
    assert np.array_equal(got, want)
    scale = rows[:, 512:528].copy().view(np.float32)
    assert scale[0].tolist() == [0.0] * 4 and scale[1, 1] == scale[2, 0] == scale[3, 3] == 0.0
    assert (rows[0, :512] & 0x7F == 0x7F).all() and (rows[1, 128:256] & 0x7F == 0x7F).all()
    assert rows[1, 130] == rows[3, 400] == 0xFF and rows[2, 17] == 0x7F
    # everything else of a group without a value is a plain zero, as in a group of zeros
    assert (np.delete(rows[2, :128], 17) == 0).all() and (np.delete(rows[3, 384:512], 16) == 0).all()
    assert (rows[6, :528] == 0).all()


@pytest.mark.gpu
def test_quantiser_keeps_nan(dev):
    x = odd_rows()
    src = torch.from_numpy(oracle.bf16_bits(x).view(np.int16)).view(torch.bfloat16).to(dev)
    got = dsa.quantize_kv_fp8(src)
    torch.cuda.synchronize()
    assert np.array_equal(got.cpu().numpy(), oracle.quantize_rows_656(x))
    c = Chunk(gen(0, dev), [8], [8], None, flat=8)
    rows = torch.zeros((8, 656), dtype=torch.uint8, device=dev)
    dsa.kv_append(src, rows, c.indptr, c.seq_lens, **c.kw, style=None)
    torch.cuda.synchronize()
    assert torch.equal(rows, got)


def values_of(fmt, cache, at):
    """The values that rows `at` of a cache hold, as readers take them."""
    if fmt in ("bf16", "v4"):
        return cache[0][at].double()
    n = {"fp8": 512, "mx": 512, "v4fp8": 448}[fmt]
    codes = cache[0][at][:, :n].contiguous().view(E4M3).double()
    if fmt == "fp8":
        r = cache[0][at]
        scale = r[:, 512:528].contiguous().view(torch.float32).double().repeat_interleave(128, 1)
        return torch.cat([codes * scale, r[:, 528:].contiguous().view(torch.bfloat16).double()], 1)
    by = cache[1][at] if fmt == "mx" else cache[0][at][:, 448:462]
    return torch.cat([codes * torch.exp2(by.double() - 127).repeat_interleave(32, 1), cache[-1][at].double()], 1)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["bf16", "fp8", "v4", "mx", "v4fp8"])
@pytest.mark.parametrize("weighted", [False, True], ids=["plain", "weight"])
def test_append_keeps_nan(dev, fmt, weighted):
    """NaN exactly where the norm and rotation of the definition give one."""
    u8, W = torch.uint8, 512 if fmt in ("v4", "v4fp8") else 576
    g = gen(6, dev)
    c = Chunk(g, [6], [6], None, flat=6)
    cs = cos_sin(6, dev)
    w = 1 + 0.2 * torch.randn(512, generator=g, device=dev) if weighted else None

    def fresh():
        if fmt in ("bf16", "v4"):
            return (torch.zeros((6, W), dtype=torch.bfloat16, device=dev),)
        if fmt == "fp8":
            return (torch.zeros((6, 656), dtype=u8, device=dev),)
        rope, nope = torch.zeros((6, 64), dtype=torch.bfloat16, device=dev), torch.zeros((6, 512), dtype=u8, device=dev)
        return (nope, torch.zeros((6, 16), dtype=u8, device=dev), rope) if fmt == "mx" else (nope, rope)

    def cached(x, **kw):
        cache = fresh()
        dsa.kv_append(x, cache if len(cache) > 1 else cache[0], c.indptr, c.seq_lens, cs, **c.kw, **kw)
        torch.cuda.synchronize()
        return values_of(fmt, cache, torch.arange(6, device=dev))

    # under the norm: a NaN, an infinity of each sign, a NaN in the last values, none
    x = bf16(g, 6, W)
    x[0, 100], x[1, 5], x[2, 300], x[3, W - 3], x[4, 511] = NAN, INF, -INF, NAN, NAN
    y = rope64(norm64(x, "rms", 512, 1e-6, w), W - 64, cs, "interleaved")
    got = cached(x, norm="rms", weight=w)
    assert torch.equal(torch.isnan(got), torch.isnan(y)), fmt
    assert bool(torch.isnan(got[:2]).any(1).all()) and bool(torch.isfinite(got[5]).all())
    assert bool((got[1][torch.isfinite(y[1]) & (y[1] == 0)] == 0).all())
    if weighted:
        return
    # without one: groups of NaNs only and NaNs among zeros
    x = bf16(g, 6, W)
    x[0, :128], x[1, 128:384], x[2, 256:288] = NAN, -NAN, NAN
    x[3, :128], x[3, 64] = 0, NAN
    got = cached(x, norm="none", style=None)
    assert torch.equal(torch.isnan(got), torch.isnan(x)), fmt


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("value", [NAN, INF], ids=["nan", "inf"])
@pytest.mark.parametrize("many", [False, True], ids=["few", "many"])
def test_tokens_that_attend_such_a_row_are_nan(dev, fp8, value, many):
    """From the appended token on, by the dense attention of both kernels and by the sparse decode."""
    g = gen(7, dev)
    n, H, hit = 3000 if many else 40, 16, 33
    c = Chunk(g, [n], [n], 64)
    x, cs = bf16(g, n, 576), cos_sin(n, dev)
    x[hit, 70] = value
    cache = torch.zeros((c.rows // 64, 64, 656 if fp8 else 576), dtype=torch.uint8 if fp8 else torch.bfloat16, device=dev)
    dsa.kv_append(x, cache, c.indptr, c.seq_lens, cs, block_table=c.table, norm="rms")
    q = bf16(g, n, H, 576)
    out, lse = dsa.mla_chunk(q, cache, c.indptr, c.seq_lens, SM_SCALE, block_table=c.table)
    torch.cuda.synchronize()
    assert bool(torch.isfinite(out[:hit]).all()) and bool(torch.isfinite(lse[:hit]).all())
    assert bool(torch.isnan(out[hit:]).all()) and bool(torch.isnan(lse[hit:]).all())
    idx = torch.arange(40, dtype=torch.int32, device=dev).view(1, 1, 40)
    for last, bad in ((hit, False), (40, True)):
        od, _ = dsa.mla_decode(q[:1].view(1, 1, H, 576), cache, idx, SM_SCALE, block_table=c.table,
                               seq_lens=torch.tensor([last], dtype=torch.int32, device=dev))
        torch.cuda.synchronize()
        assert bool(torch.isnan(od).all()) if bad else bool(torch.isfinite(od).all()), last
