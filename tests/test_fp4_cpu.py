"""400-byte rows and kv_read without a GPU: what the entries refuse, the calls of nothing, split counts, and the
tests' own codes against the definition."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

import _fp4
from opfoundry_amd import abi

NULL, SHAPE, UNSUPPORTED, FORMAT, WORKSPACE, SPLITS, STRIDE = -1, -2, -3, -4, -5, -6, -7


@pytest.fixture(scope="module")
def lib():
    return abi.load_library()


def _set(a, kw):
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def _read(**kw):
    base = dict(cache=0x100000, cache_rows=640, kv_format=abi.KV_MXFP4, T=3, out=0x10000, out_stride_t=576, q_indptr=0x2004,
                seq_lens=0x3004, block_table=0x4004, block_table_stride=10, table_blocks=10, block_size=64, B=1)
    return _set(abi.KvReadArgs(), {**base, **kw})


MX = dict(kv_format=abi.KV_MXFP8, cache_scale=0x900000, cache_rope=0xa00000)
READ_BAD = [
    (dict(T=-1), SHAPE), (dict(T=2 ** 29), SHAPE), (dict(B=-1), SHAPE), (dict(cache_rows=-1), SHAPE), (dict(cache_rows=2 ** 31), SHAPE),
    (dict(kv_format=-1), FORMAT), (dict(kv_format=6), FORMAT), (dict(block_size=0), SHAPE), (dict(table_blocks=-1), SHAPE),
    (dict(block_size=2 ** 20, table_blocks=2 ** 12), SHAPE), (dict(block_table_stride=-1), STRIDE),
    (dict(block_table=0, kv_batch_stride=-1), STRIDE), (dict(q_indptr=0), NULL), (dict(seq_lens=0), NULL), (dict(out=0), NULL),
    (dict(cache=0), NULL), ({**MX, "cache_scale": 0}, NULL), ({**MX, "cache_rope": 0}, NULL), (dict(stride_row=384), STRIDE),
    (dict(stride_row=408), STRIDE), (dict(kv_format=abi.KV_BF16, stride_row=568), STRIDE), ({**MX, "rope_stride_row": 60}, STRIDE),
    ({**MX, "scale_stride_row": 24}, STRIDE), (dict(cache=0x100008), STRIDE), ({**MX, "cache_scale": 0x900004}, STRIDE),
    (dict(out=0x10008), STRIDE), (dict(out_stride_t=580), STRIDE), (dict(out_stride_t=568), STRIDE), (dict(out_stride_t=-576), STRIDE),
    (dict(kv_format=abi.KV_BF16_D512, out_stride_t=504), STRIDE),
    # out over the cache, its last row, a stream of it
    (dict(out=0x100000), STRIDE), (dict(out=0x100000 + 639 * 400), STRIDE), (dict(out=0x100000 - 3 * 1152 + 16), STRIDE),
    ({**MX, "out": 0x900000 + 16 * 639}, STRIDE), ({**MX, "out": 0xa00000 + 128 * 639}, STRIDE),
]


@pytest.mark.parametrize("kw,code", READ_BAD, ids=[f"{i}" for i in range(len(READ_BAD))])
def test_read_refuses(lib, kw, code):
    assert lib.dsa_kv_read(ctypes.byref(_read(**kw)), None) == code


def test_read_of_nothing(lib):
    assert lib.dsa_kv_read(None, None) == NULL
    for kw in (dict(T=0), dict(B=0), dict(T=0, q_indptr=0, seq_lens=0, cache=0, out=0)):
        assert lib.dsa_kv_read(ctypes.byref(_read(**kw)), None) == 0, kw


def _decode(**kw):
    base = dict(q=0x1000, q_stride_b=128 * 576, q_stride_t=128 * 576, q_stride_h=576, kv_cache=0x10000, kv_total_rows=6400,
                kv_format=abi.KV_MXFP4, block_size=64, block_table=0x4004, block_table_stride=100, seq_lens=0x5004, indices=0x6004,
                idx_stride_b=2048, idx_stride_t=2048, out=0x7008, o_stride_b=128 * 512, o_stride_t=128 * 512, o_stride_h=512,
                B=2, s_q=1, H=128, topk=2048, sm_scale=0.07)
    return _set(abi.DecodeArgs(), {**base, **kw})


DECODE_BAD = [(dict(sm_scale=0.0), UNSUPPORTED), (dict(sm_scale=-1.0), UNSUPPORTED), (dict(sm_scale=math.nan), UNSUPPORTED),
              (dict(sm_scale=math.inf), UNSUPPORTED), (dict(kv_stride_row=384), STRIDE), (dict(kv_stride_row=408), STRIDE),
              (dict(kv_stride_row=2 ** 32), STRIDE), (dict(kv_cache=0x10008), STRIDE), (dict(B=2 ** 20, H=2 ** 10), SHAPE),
              (dict(num_splits=65), SPLITS), (dict(indices=0), NULL), (dict(kv_format=6), FORMAT)]


@pytest.mark.parametrize("kw,code", DECODE_BAD, ids=[f"{i}" for i in range(len(DECODE_BAD))])
def test_decode_refuses(lib, kw, code):
    a, n, size = ctypes.byref(_decode(**kw)), ctypes.c_int32(-5), ctypes.c_size_t(7)
    assert lib.dsa_mla_decode(a, 0x100000, 1 << 40, None) == code
    assert lib.dsa_mla_decode_noalloc(a, None) == code
    assert lib.dsa_mla_decode_num_splits(a, ctypes.byref(n)) == code and n.value == -5
    assert lib.dsa_mla_decode_workspace_size(a, ctypes.byref(size)) == code and size.value == 7


def test_csr_form_refuses_the_format(lib):
    a = abi.CsrArgs()
    a.q, a.kv, a.out, a.kv_indptr, a.kv_indices = 0x1000, 0x10000, 0x7008, 0x2004, 0x3004
    a.B, a.s_q, a.H, a.total_tokens, a.max_kv_len, a.kv_format, a.softmax_scale = 1, 1, 16, 100, 64, abi.KV_MXFP4, 0.07
    size = ctypes.c_size_t(7)
    assert lib.dsa_mla_decode_csr_workspace_size(ctypes.byref(a), ctypes.byref(size)) == FORMAT and size.value == 7


@pytest.mark.parametrize("B", [1, 2, 3, 16, 64, 100, 256, 300, 4000])
@pytest.mark.parametrize("H", [1, 16, 40, 64, 128, 200])
@pytest.mark.parametrize("topk", [0, 1, 100, 2048, 20000])
def test_decode_split_counts(lib, B, H, topk):
    """Every automatic count is one that the call takes, splits nothing below four tiles, and its workspace holds the
    partials; a given count is kept."""
    n, size = ctypes.c_int32(0), ctypes.c_size_t(0)
    a = _decode(B=B, H=H, topk=topk)
    assert lib.dsa_mla_decode_num_splits(ctypes.byref(a), ctypes.byref(n)) == 0
    assert 1 <= n.value <= max(1, min(64, (topk + 127) // 128))
    assert lib.dsa_mla_decode_workspace_size(ctypes.byref(a), ctypes.byref(size)) == 0
    assert size.value == (n.value * B * H * 513 * 4 + 256 if n.value > 1 else 0)
    a.num_splits = 5
    assert lib.dsa_mla_decode_num_splits(ctypes.byref(a), ctypes.byref(n)) == 0 and n.value == 5


def test_chunk_takes_the_format(lib):
    a = abi.ChunkArgs()
    _set(a, dict(q=0x1000, q_stride_t=16 * 576, q_stride_h=576, q_indptr=0x2004, seq_lens=0x3004, kv_cache=0x10000,
                 kv_total_rows=6400, kv_format=abi.KV_MXFP4, block_size=64, block_table=0x4004, block_table_stride=100, out=0x5008,
                 o_stride_t=16 * 512, o_stride_h=512, lse=0x6004, table_blocks=100, T=2, B=1, H=16, causal=1, max_kv_len=6000,
                 num_splits=4, sm_scale=0.07))
    size = ctypes.c_size_t(0)
    assert lib.dsa_mla_chunk_workspace_size(ctypes.byref(a), ctypes.byref(size)) == 0 and size.value == 4 * 2 * 16 * 513 * 4 + 16
    assert lib.dsa_mla_chunk(ctypes.byref(a), 0x100000, size.value - 1, None) == WORKSPACE
    for kw in (dict(kv_stride_row=384), dict(kv_stride_row=408)):
        assert lib.dsa_mla_chunk(ctypes.byref(_set(a, kw)), 0x100000, 1 << 40, None) == STRIDE


def test_the_references_codes():
    """By the definition: nearest values with ties to the even code, the least exponent, values beside borders."""
    for a, code in ((0, 0), (0.25, 0), (0.2500001, 1), (0.75, 2), (0.7499999, 1), (1.25, 2), (1.75, 4), (2.5, 4), (3.5, 6), (5, 6),
                    (5.0000001, 7), (100, 7)):
        assert int(_fp4.nearest(torch.tensor([a], dtype=torch.float64))) == code, a
    for amax, e in ((0, 0), (6, 0), (6.0000001, 1), (3, -1), (3.0000001, 0), (1.5 * 2 ** 127, 125), (3.38e38, 126), (1e-45, -125)):
        assert int(_fp4.exponent(torch.tensor([amax], dtype=torch.float64))) == e, amax
    g = torch.Generator().manual_seed(1)
    x = torch.randn((50, 512), generator=g, dtype=torch.float64)
    codes, scales = _fp4.pack(x)
    r = torch.cat([codes, scales, torch.zeros((50, 128), dtype=torch.uint8)], 1)
    err = (_fp4.values(r)[:, :512] - x).abs()
    # at most half a step: of a value below 2 a quarter, else a quarter of the value, in units of the scale
    scale = torch.exp2(scales.double() - 127).repeat_interleave(32, 1)
    assert bool((err <= torch.maximum(0.25 * scale, 0.25 * x.abs())).all())
    assert torch.equal(_fp4.as_bf16(r).double(), _fp4.values(r))


def test_python_checks_before_a_device():
    from opfoundry_amd import dsa
    assert dsa.kv_format_of(torch.zeros((7, 64, 400), dtype=torch.uint8)) == (abi.KV_MXFP4, 448, 0)
    assert dsa.kv_format_of(torch.zeros((9, 448), dtype=torch.uint8)[:, :400]) == (abi.KV_MXFP4, 9, 448)
    with pytest.raises(ValueError):
        dsa.kv_read(torch.zeros((4, 400), dtype=torch.uint8), torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), 1)
