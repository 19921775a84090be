"""Packed argument blocks: values that their fields do not hold reach the library's own checks, or are refused by name."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

from opfoundry_amd import abi, dsa
from test_streams_cpu import DEV, U8, i32, t

BLOCKS = [(abi.DecodeArgs, abi.pack_decode), (abi.PrefillArgs, abi.pack_prefill), (abi.KvReadArgs, abi.pack_read),
          (abi.ChunkArgs, abi.pack_chunk)]
SHAPE, SPLITS, NULL, UNSUPPORTED = -2, -6, -1, -3


@pytest.fixture
def here(monkeypatch):
    """Tensors that say they are on a device, and the library: every call of these tests ends in its checks."""
    monkeypatch.setattr(dsa, "_current_device", lambda: DEV)
    monkeypatch.setattr(dsa, "_raw_stream", lambda d: 0)


def whole(cls):
    return [i for i, (_, c) in enumerate(cls._fields_) if c is ctypes.c_int32]


@pytest.mark.parametrize("cls,pack", BLOCKS, ids=[c.__name__ for c, _ in BLOCKS])
def test_values_past_a_fields_range(cls, pack):
    n = len(cls._fields_)
    base = [0.5 if c is ctypes.c_float else i + 1 for i, (_, c) in enumerate(cls._fields_)]
    for i in whole(cls):
        name = cls._fields_[i][0]
        for v, held in ((2 ** 31 - 1, 2 ** 31 - 1), (2 ** 31, 2 ** 31 - 1), (2 ** 32 + 1, 2 ** 31 - 1), (-2 ** 31 - 1, -2 ** 31)):
            a = cls.from_buffer_copy(pack(*base[:i], v, *base[i + 1:]))
            assert getattr(a, name) == held, (name, v)
            assert all(getattr(a, f) == base[k] for k, (f, _) in enumerate(cls._fields_) if k != i)
        for bad in (1.5, None, "2"):
            with pytest.raises(TypeError, match=name):
                pack(*base[:i], bad, *base[i + 1:])
    for i, (name, c) in enumerate(cls._fields_):
        if c is ctypes.c_int64:
            for bad in (2 ** 63, -2 ** 63 - 1):
                with pytest.raises(ValueError, match=name):
                    pack(*base[:i], bad, *base[i + 1:])
        if c is ctypes.c_void_p:
            assert getattr(cls.from_buffer_copy(pack(*base[:i], None, *base[i + 1:])), name) is None
        if c is ctypes.c_float:
            for v in (1e39, -1e39, math.inf, math.nan):
                got = getattr(cls.from_buffer_copy(pack(*base[:i], v, *base[i + 1:])), name)
                assert got == math.copysign(math.inf, v) or (math.isnan(v) and math.isnan(got))
    assert n == len(base)


@pytest.mark.parametrize("splits", [65, 2 ** 31 - 1, 2 ** 31, 2 ** 32 + 1, -1, -2 ** 31 - 5])
def test_split_counts_past_every_range_are_the_librarys_to_refuse(here, splits):
    q, idx, sl = t(2, 1, 16, 576), i32(*range(8)).view(2, 1, 4), i32(4, 4)
    for kv in (t(64, 576), t(64, 656, dtype=U8), t(64, 400, dtype=U8)):
        for call in (lambda: dsa.mla_decode(q, kv, idx, 0.1, seq_lens=sl, num_splits=splits),
                     lambda: dsa.mla_prefill(q[:, 0], kv, idx[:, 0], 0.1, num_splits=splits),
                     lambda: dsa.mla_chunk(q[:, 0], kv, i32(0, 2), i32(9), 0.1, num_splits=splits),
                     lambda: dsa.decode_num_splits(dsa.make_decode_args(q, kv, idx, 0.1, q, None, seq_lens=sl, num_splits=splits))):
            with pytest.raises(abi.DsaError) as e:
                call()
            assert e.value.code == SPLITS


def test_other_values_past_every_range(here):
    q, kv, ip, sl = t(2, 16, 576), t(64, 400, dtype=U8), i32(0, 2), i32(9)
    for call, code in ((lambda: dsa.mla_chunk(q, kv, ip, sl, 0.1, max_kv_len=2 ** 33), SHAPE),
                       (lambda: dsa.mla_chunk(q, kv, ip, sl, 1e39), UNSUPPORTED),
                       (lambda: dsa.kv_read(kv, ip, sl, 3, block_table=i32(0, 1).view(1, 2), block_size=2 ** 40), SHAPE),
                       (lambda: dsa.mla_prefill(q, kv, i32(0, 1).view(2, 1), 1e39), UNSUPPORTED)):
        with pytest.raises(abi.DsaError) as e:
            call()
        assert e.value.code == code
    with pytest.raises(ValueError, match="kv_batch_stride"):
        dsa.kv_read(kv, ip, sl, 3, kv_batch_stride=2 ** 63)


def test_a_missing_seq_lens_is_the_librarys_to_refuse():
    q, kv, idx = torch.zeros((2, 1, 16, 576), dtype=torch.bfloat16), torch.zeros((64, 576), dtype=torch.bfloat16), torch.zeros((2, 1, 4), dtype=torch.int32)
    a = dsa.make_decode_args(q, kv, idx, 0.1, q, None, seq_lens=None)
    assert a.seq_lens is None
    n = ctypes.c_int32(0)
    assert abi.load_library().dsa_mla_decode_num_splits(ctypes.byref(a), ctypes.byref(n)) == NULL
