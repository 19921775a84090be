"""dsa_mla_decode_noalloc on 400-byte rows at the limit of its scratch."""
from __future__ import annotations

import ctypes

import pytest
import torch

import _fp4
from _chunk import SM_SCALE, bf16, gen, i32
from opfoundry_amd import abi, dsa

pytestmark = pytest.mark.gpu

# tokens, heads, entries; the split count the call must run with (of the automatic one's partials)
CALLS = [(32, 64, 2048), (64, 32, 2048), (16, 128, 2048), (96, 128, 2048), (64, 64, 2048), (128, 32, 2048)]


def largest(B, H):
    return max(1, (abi.NOALLOC_SCRATCH_BYTES - 256) // (B * H * 513 * 4))


@pytest.mark.parametrize("B,H,topk", CALLS)
def test_an_automatic_count_falls_back_to_the_largest_that_fits(dev, B, H, topk):
    g = gen(B + H, dev)
    kv, q = _fp4.rows(g, 2500), bf16(g, B, 1, H, 576)
    idx = torch.stack([torch.randperm(2500, generator=g, device=dev)[:topk] for _ in range(B)]).to(torch.int32)[:, None]
    sl = i32([2500] * B, dev)
    o, l = torch.full((B, 1, H, 512), 7.0, dtype=torch.bfloat16, device=dev), torch.full((B, 1, H), 7.0, device=dev)
    a = dsa.make_decode_args(q, kv, idx, SM_SCALE, o, l, seq_lens=sl)
    ns = dsa.decode_num_splits(a)
    assert dsa.decode_workspace_size(a) > abi.NOALLOC_SCRATCH_BYTES and 1 <= largest(B, H) < ns
    stream = torch.cuda.current_stream().cuda_stream
    assert abi.load_library().dsa_mla_decode_noalloc(ctypes.byref(a), stream) == 0
    want = dsa.mla_decode(q, kv, idx, SM_SCALE, seq_lens=sl, num_splits=largest(B, H))
    torch.cuda.synchronize()
    assert torch.equal(o, want[0]) and torch.equal(l, want[1])
    at, ref = _fp4.attend_lists64(q[:, 0], _fp4.as_bf16(kv), idx[:, 0].tolist(), H)
    _fp4.check(at, o[:, 0], l[:, 0], ref)
    # a count of the caller's is kept, or refused with the outputs as they were
    o.fill_(7.0)
    a.num_splits = largest(B, H) + 1
    assert abi.load_library().dsa_mla_decode_noalloc(ctypes.byref(a), stream) == (-9 if largest(B, H) + 1 > 1 else 0)
    torch.cuda.synchronize()
    assert bool((o == 7).all())
