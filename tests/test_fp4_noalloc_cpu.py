"""dsa_mla_decode_noalloc on 400-byte rows without a GPU: no automatic split count is refused for its partials' size."""
from __future__ import annotations

import ctypes

import pytest
import torch

from opfoundry_amd import abi
from test_fp4_cpu import _decode

SCRATCH_LIMIT = -9


@pytest.mark.skipif(torch.cuda.is_available(), reason="these calls' addresses are no device's")
@pytest.mark.parametrize("H", [8, 16, 32, 40, 64, 96, 128, 200])
@pytest.mark.parametrize("topk", [300, 2048, 20000])
def test_automatic_counts_fit_the_scratch(H, topk):
    lib = abi.load_library()
    for B in (1, 2, 7, 16, 32, 64, 96, 128, 200, 256, 1000):
        rc = lib.dsa_mla_decode_noalloc(ctypes.byref(_decode(B=B, H=H, topk=topk)), None)
        assert rc != SCRATCH_LIMIT, (B, rc)
    # (a count of the caller's stays, and is refused where it does not fit)
    assert lib.dsa_mla_decode_noalloc(ctypes.byref(_decode(B=64, H=H, topk=topk, num_splits=64)), None) == SCRATCH_LIMIT
