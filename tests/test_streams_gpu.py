"""Calls with stream=: outputs and workspaces that they allocate are not handed out again while the call waits or runs, and
their bits are those of a call on the current stream."""
from __future__ import annotations

import pytest
import torch

import _fp4
from _chunk import SM_SCALE, bf16, gen, i32
from opfoundry_amd import dsa

pytestmark = pytest.mark.gpu


def decode(g, dev):
    kv, q = _fp4.rows(g, 3000), bf16(g, 2, 1, 128, 576)
    idx = torch.stack([torch.randperm(3000, generator=g, device=dev)[:2048] for _ in range(2)]).to(torch.int32)[:, None]
    sl = i32([3000, 3000], dev)
    a = dsa.make_decode_args(q, kv, idx, SM_SCALE, q, None, seq_lens=sl)
    assert dsa.decode_num_splits(a) > 1
    return lambda **k: dsa.mla_decode(q, kv, idx, SM_SCALE, seq_lens=sl, **k)


def prefill(g, dev):
    kv, q = bf16(g, 3000, 576), bf16(g, 3, 16, 576)
    idx = torch.stack([torch.randperm(3000, generator=g, device=dev)[:2048] for _ in range(3)]).to(torch.int32)
    assert dsa.prefill_workspace_size(dsa.make_prefill_args(q, kv, idx, SM_SCALE, q, None)) > 0
    return lambda **k: dsa.mla_prefill(q, kv, idx, SM_SCALE, **k)


def csr(g, dev):
    kv, q = bf16(g, 3000, 576), bf16(g, 2, 16, 576)
    ptr, rows = i32([0, 2000, 2100], dev), torch.randint(0, 3000, (2100,), generator=g, device=dev).to(torch.int32)
    return lambda **k: dsa.mla_decode_csr(q, kv, ptr, rows, SM_SCALE, max_kv_len=2000, **k)


def indexer(g, dev):
    q, w, kc, sl = bf16(g, 2, 1, 64, 128), torch.randn((2, 1, 64), generator=g, device=dev), bf16(g, 2000, 128), i32([900, 700], dev)
    return lambda **k: (dsa.indexer_scores(q, w, kc, sl, n_cols=1000, k_batch_stride=1000, **k),)


def topk(g, dev):
    s = torch.randn((5, 4000), generator=g, device=dev)
    return lambda **k: (dsa.topk_indices(s, 300, **k),)


@pytest.mark.parametrize("make", [decode, prefill, csr, indexer, topk])
def test_memory_of_a_call_on_another_stream(dev, make):
    g = gen(61, dev)
    call = make(g, dev)
    want = [x.clone() for x in call()]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for as_handle in (False, True):
        with torch.cuda.stream(side):
            torch.cuda._sleep(100_000_000)              # (the call's kernels wait for this)
        got = call(stream=side.cuda_stream if as_handle else side)
        was, shapes = {x.data_ptr() for x in got}, [(x.shape, x.dtype) for x in got]
        kept = [torch.empty_like(x) for x in got]
        with torch.cuda.stream(side):
            for k, x in zip(kept, got):
                k.copy_(x)
        del got, x
        # what the current stream allocates now is none of the call's memory (and filling it changes nothing)
        others = [torch.full(s, 7, dtype=d, device=dev) for s, d in shapes for _ in range(3)]
        more = torch.full((32 << 20,), 255, dtype=torch.uint8, device=dev)
        assert not side.query(), "the side stream ended before the check"
        assert not was & {x.data_ptr() for x in others} and more.data_ptr() not in was
        side.synchronize()
        torch.cuda.synchronize()
        for k, w in zip(kept, want):
            assert torch.equal(k.view(torch.uint8), w.view(torch.uint8))
