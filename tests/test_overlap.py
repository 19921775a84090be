"""Outputs whose rows share memory with one another, or with what the call reads, are refused: workgroups would
race for them.  The host's rules (opfoundry_amd/csrc/dsa_overlap.h, compiled here with g++) against a count of
elements, and the entries' refusals, which come before any launch (no device is touched)."""
from __future__ import annotations

import ctypes
import os
import random
import subprocess

import pytest
import torch

from _chunk import bf16, cos_sin, gen
from opfoundry_amd import abi, dsa
from test_chunk_cpu import _chunk, _prep

HERE = os.path.dirname(os.path.abspath(__file__))
STRIDE = -7


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("overlap") / "liboverlap_check.so")
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-Wall", "-Werror",
                    os.path.join(HERE, "native", "overlap_check.cpp"), "-o", so], check=True)
    L = ctypes.CDLL(so)
    L.rows_within.argtypes = [ctypes.c_int64] * 5
    L.rows_between.argtypes = [ctypes.c_int64] * 9
    return L


def elements(T, H, st, sh, w, at=0):
    return [at + t * st + h * sh + i for t in range(T) for h in range(H) for i in range(w)]


def test_rows_of_one_output(rules):
    rng = random.Random(1)
    seen = {0: 0, 1: 0}
    for _ in range(20000):
        T, H, w = rng.randint(1, 6), rng.randint(1, 6), rng.randint(1, 5)
        st, sh = rng.randint(0, 40), rng.randint(0, 40)
        e = elements(T, H, st, sh, w)
        want = int(len(set(e)) < len(e))
        assert rules.rows_within(T, H, st, sh, w) == want, (T, H, st, sh, w)
        seen[want] += 1
    assert min(seen.values()) > 2000


def test_rows_of_an_output_and_an_input(rules):
    """Never a miss; a false alarm only where the two lie among one another with other strides."""
    rng = random.Random(2)
    seen = {0: 0, 1: 0}
    exact = 0
    for i in range(40000):
        T, Ha, Hb, w = rng.randint(1, 5), rng.randint(1, 5), rng.randint(1, 5), rng.randint(1, 4)
        stb, shb = rng.randint(0, 60), rng.randint(0, 20)
        if rules.rows_within(T, Hb, stb, shb, w):
            continue
        sta, sha = (stb if rng.random() < 0.8 else rng.randint(0, 60)), (shb if rng.random() < 0.7 else rng.randint(0, 20))
        delta = rng.randint(-150, 150)
        a, b = set(elements(T, Ha, sta, sha, w)), set(elements(T, Hb, stb, shb, w, delta))
        want, got = int(bool(a & b)), rules.rows_between(T, Ha, sta, sha, Hb, stb, shb, w, delta)
        same = (T == 1 or sta == stb != 0) and (Ha == 1 or Hb == 1 or sha == shb)
        assert got >= want, (T, Ha, sta, sha, Hb, stb, shb, w, delta)
        if same:
            assert got == want, (T, Ha, sta, sha, Hb, stb, shb, w, delta)
            exact += 1
        if max(a) < min(b) or max(b) < min(a):
            assert got == 0
        seen[want] += 1
    assert min(seen.values()) > 2000 and exact > 10000


def test_layouts_in_use(rules):
    """Dense, by head, a slice of a fused projection, and the largest sizes, without a long search."""
    D = 576
    assert not rules.rows_within(4096, 128, 128 * D, D, D) and not rules.rows_within(4096, 128, D, 4096 * D, D)
    assert not rules.rows_within(2 ** 22, 127, 127 * 512, 512, 512) and not rules.rows_within(1, 128, 0, D, D)
    assert rules.rows_within(2, 2, D, D, D) and rules.rows_within(5, 16, 2 * D, D, D)
    # 128 query heads and a key head of one projection of 129, each in place: they lie between one another
    assert not rules.rows_between(4096, 128, 129 * D, D, 1, 129 * D, D, D, 128 * D)
    assert not rules.rows_between(4096, 1, 129 * D, D, 128, 129 * D, D, D, -128 * D)
    assert rules.rows_between(4096, 128, 129 * D, D, 1, 129 * D, D, D, 127 * D)
    assert rules.rows_between(3, 16, 16 * D, D, 16, 16 * D, D, D, 8)
    big = 2 ** 62
    assert not rules.rows_within(2, 2, big, D, D) and not rules.rows_between(2, 2, big, D, 2, big, D, D, 4 * D)


@pytest.mark.parametrize("kw", [
    dict(o_stride_t=512, o_stride_h=512), dict(o_stride_t=1024, o_stride_h=512), dict(o_stride_t=512, o_stride_h=516),
    dict(o_stride_t=768, o_stride_h=1024, T=3), dict(o_stride_t=15 * 512, o_stride_h=512),
    dict(o_stride_t=16 * 512 - 4, o_stride_h=512),
])
def test_chunk_refuses_an_output_over_itself(kw):
    lib = abi.load_library()
    n, size = ctypes.c_int32(-5), ctypes.c_size_t(7)
    a = ctypes.byref(_chunk(**kw))
    assert lib.dsa_mla_chunk(a, 0x100000, 1 << 40, None) == STRIDE
    assert lib.dsa_mla_chunk_num_splits(a, ctypes.byref(n)) == STRIDE and n.value == -5
    assert lib.dsa_mla_chunk_workspace_size(a, ctypes.byref(size)) == STRIDE and size.value == 7


@pytest.mark.parametrize("kw", [
    dict(o_stride_t=512, o_stride_h=1024), dict(o_stride_t=512, o_stride_h=2 * 512 + 8), dict(o_stride_t=0, T=1),
    dict(o_stride_t=512, o_stride_h=0, H=1), dict(o_stride_t=17 * 512, o_stride_h=512),
    dict(o_stride_t=516, o_stride_h=1032), dict(T=3, H=2, o_stride_t=1024, o_stride_h=512),
])
def test_chunk_takes_outputs_apart(kw):
    lib = abi.load_library()
    n = ctypes.c_int32(-5)
    assert lib.dsa_mla_chunk_num_splits(ctypes.byref(_chunk(**{"T": 2, **kw})), ctypes.byref(n)) == 0 and n.value == 4


K = {"k.x": 0x1000000, "k.stride_t": 576, "k.stride_h": 576, "k.out": 0x2000000, "k.out_stride_t": 576,
     "k.out_stride_h": 576, "k.H": 1, "k.norm": 1, "q.out": 0x100000}
ROW = 2 * 576


@pytest.mark.parametrize("kw", [
    # an output's own rows
    {"q.out": 0x100000, "q.out_stride_t": 576, "q.out_stride_h": 576},
    {"q.out": 0x100000, "q.out_stride_t": 2 * 576},
    {"q.x": 0x100000, "q.out": 0x100000, "q.stride_t": 576, "q.out_stride_t": 576},
    # an output over its input, shifted by less than all of it
    {"q.out": 0x1000 + 16}, {"q.out": 0x1000 + ROW}, {"q.out": 0x1000 - ROW + 0x10}, {"q.out": 0x1000 + 16 * ROW},
    {"q.out": 0x1000 + 2 * ROW, "q.out_stride_t": 18 * 576},
    # ... over the other stream's input or output
    {**K, "k.out": 0x1000}, {**K, "k.out": 0x1000 + 47 * ROW}, {**K, "q.out": 0x1000000 - 47 * ROW},
    {**K, "k.out": 0x100000 + 5 * ROW}, {**K, "k.x": 0x100000 + 16},
])
def test_norm_rope_refuses_outputs_over_what_it_reads(kw):
    assert abi.load_library().dsa_qk_norm_rope(ctypes.byref(_prep(**kw)), None) == STRIDE


@pytest.mark.gpu
@pytest.mark.parametrize("D", [128, 512, 576])
@pytest.mark.parametrize("T", [1, 2, 77])
def test_slices_of_one_buffer(dev, D, T):
    """Queries and a key of one projection, each in place; outputs that take turns with their inputs, by head and
    by stream: as with buffers of their own."""
    g = gen(D + T, dev)
    cs, pos = cos_sin(100, dev), torch.arange(T, dtype=torch.int32, device=dev)
    kw = dict(q_norm="rms", k_norm="layer", style="halves")
    x = bf16(g, T, 18, D)
    want = dsa.qk_norm_rope(x[:, :17].clone(), cs, pos, k=x[:, 17:].clone(), **kw)
    fused = x.clone()
    dsa.qk_norm_rope(fused[:, :17], cs, pos, k=fused[:, 17:], q_out=fused[:, :17], k_out=fused[:, 17:], **kw)
    torch.cuda.synchronize()
    assert torch.equal(fused[:, :17], want[0]) and torch.equal(fused[:, 17:], want[1])
    turns = torch.zeros((T, 36, D), dtype=torch.bfloat16, device=dev)
    turns[:, 0::2] = x
    dsa.qk_norm_rope(turns[:, 0:34:2], cs, pos, k=turns[:, 34:35], q_out=turns[:, 1:34:2], k_out=turns[:, 35:], **kw)
    torch.cuda.synchronize()
    assert torch.equal(turns[:, 0::2], x) and torch.equal(turns[:, 1:34:2], want[0]) and torch.equal(turns[:, 35:], want[1])
    with pytest.raises(abi.DsaError) as e:
        dsa.qk_norm_rope(fused[:, :17], cs, pos, q_out=fused[:, 1:])
    assert e.value.code == STRIDE
