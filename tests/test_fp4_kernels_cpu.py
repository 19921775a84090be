"""Which kernel calls on 400-byte rows run in, by the library's own answer: the calls of tests/test_fp4_kernels_gpu.py and the
ranges that those queries answer for."""
from __future__ import annotations

import ctypes

import pytest

from _fp4_kernels import BLOCK_SIZE, CHUNKS, KERNELS, LISTS, bound
from opfoundry_amd import abi, dsa
from test_fp4_cpu import DECODE_BAD, _decode, _set


@pytest.fixture(scope="module")
def lib():
    return abi.load_library()


def prefill_args(T, H, topk, ns, **kw):
    return _set(abi.PrefillArgs(), {**dict(q=0x1000, q_stride_n=H * 576, q_stride_h=576, kv=0x10000, kv_rows=6400, kv_format=abi.KV_MXFP4,
                                           indices=0x6004, idx_stride_n=topk, out=0x7008, o_stride_n=H * 512, o_stride_h=512, N=T, H=H,
                                           topk=topk, num_splits=ns, sm_scale=0.07), **kw})


def chunk_args(new, lens, H, ns, **kw):
    blocks = bound(lens) // BLOCK_SIZE
    return _set(abi.ChunkArgs(), {**dict(q=0x1000, q_stride_t=H * 576, q_stride_h=576, q_indptr=0x2004, seq_lens=0x3004, kv_cache=0x10000,
                                         kv_total_rows=640000, kv_format=abi.KV_MXFP4, block_size=BLOCK_SIZE, block_table=0x4004,
                                         block_table_stride=blocks, out=0x5008, o_stride_t=H * 512, o_stride_h=512, lse=0x6004,
                                         table_blocks=blocks, T=sum(new), B=len(new), H=H, causal=1, max_kv_len=bound(lens),
                                         num_splits=ns, sm_scale=0.07), **kw})


@pytest.mark.parametrize("heads", KERNELS)
def test_the_kernel_of_a_list(heads):
    T, H, topk = LISTS[heads]
    a = _decode(B=T, H=H, topk=topk, num_splits=1, q_stride_b=H * 576, q_stride_t=H * 576, o_stride_b=H * 512, o_stride_t=H * 512)
    assert dsa.decode_group_heads(a) == heads
    assert dsa.prefill_group_heads(prefill_args(T, H, topk, 1)) == heads


@pytest.mark.parametrize("rows", KERNELS)
def test_the_kernel_of_a_chunk(rows):
    assert dsa.chunk_group_rows(ctypes.byref(chunk_args(*CHUNKS[rows], 1))) == rows


@pytest.mark.parametrize("fmt,stride,all_of", [(abi.KV_BF16, 0, {32, 64, 128}), (abi.KV_FP8_656, 0, {32, 64, 128}), (abi.KV_MXFP4, 0, {16, 32, 128})])
def test_every_answer_is_a_kernel_and_every_kernel_an_answer(fmt, stride, all_of):
    seen, seen_p, rows = set(), set(), set()
    for T in (1, 2, 16, 40, 64, 100, 160, 200, 256, 300, 1000):
        for H in (1, 16, 33, 64, 96, 128, 200):
            for ns in (0, 1, 3):
                a = _decode(B=T, H=H, num_splits=ns, kv_format=fmt)
                seen.add(dsa.decode_group_heads(a))
                seen_p.add(dsa.prefill_group_heads(prefill_args(T, H, 2048, ns, kv_format=fmt)))
                rows.add(dsa.chunk_group_rows(ctypes.byref(chunk_args([T], [5000], H, ns, kv_format=fmt))))
    assert seen == all_of and seen_p == all_of
    assert rows == ({16, 32, 128} if fmt == abi.KV_MXFP4 else {32, 128})


@pytest.mark.parametrize("kw,code", DECODE_BAD, ids=[f"{i}" for i in range(len(DECODE_BAD))])
def test_the_queries_refuse_what_the_calls_refuse(lib, kw, code):
    n = ctypes.c_int32(-5)
    assert lib.dsa_mla_decode_group_heads(ctypes.byref(_decode(**kw)), ctypes.byref(n)) == code and n.value == -5


def test_the_queries_need_a_place_and_a_call(lib):
    n = ctypes.c_int32(-5)
    for f, a in ((lib.dsa_mla_decode_group_heads, _decode()), (lib.dsa_mla_prefill_group_heads, prefill_args(3, 16, 64, 0)),
                 (lib.dsa_mla_chunk_group_rows, chunk_args([3], [9], 16, 0))):
        assert f(ctypes.byref(a), None) == -1 and f(None, ctypes.byref(n)) == -1 and n.value == -5
        assert f(ctypes.byref(a), ctypes.byref(n)) == 0 and n.value in (16, 32, 128)
        n.value = -5
    assert lib.dsa_mla_prefill_group_heads(ctypes.byref(prefill_args(3, 16, 64, 65)), ctypes.byref(n)) == -6
    assert lib.dsa_mla_chunk_group_rows(ctypes.byref(chunk_args([3], [9], 16, 65)), ctypes.byref(n)) == -6
