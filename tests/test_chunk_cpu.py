"""The chunk operators (include/dsa_chunk.h) without a GPU: the rules of sequences, pages, blocks and
splits that their kernels apply (opfoundry_amd/csrc/dsa_seq.h, compiled here with g++), the layout of
their argument structs against the C compiler's, and the refusals of every entry point, which come
before any launch (no device is touched)."""
from __future__ import annotations

import ctypes
import math
import os
import subprocess

import numpy as np
import pytest
import torch

from opfoundry_amd import abi, dsa

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
NULL, SHAPE, UNSUPPORTED, FORMAT, WORKSPACE, SPLITS, STRIDE = -1, -2, -3, -4, -5, -6, -7


# ------------------------------------------------------------------ the rules

@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("seq") / "libseq_check.so")
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-Wall", "-Werror",
                    os.path.join(HERE, "native", "seq_check.cpp"), "-o", so], check=True)
    L = ctypes.CDLL(so)
    i32, i64, vp = ctypes.c_int32, ctypes.c_int64, ctypes.c_void_p
    for name, args, res in [("seq_row", [vp, i64, i32, i32, i64, i32, i64, i64], i64),
                            ("seq_position", [vp, vp, i32, i32], i64), ("seq_common", [i32, i32], i32),
                            ("seq_block_start", [i64, i32, i32, i32], i64),
                            ("seq_parts", [i32, i32, ctypes.c_float], i32)]:
        f = getattr(L, name)
        f.argtypes, f.restype = args, res
    return L


BAD_PAGES = [-(2 ** 31), -1, 2 ** 31 - 1]


@pytest.mark.parametrize("bs,blocks", [(1, 9), (16, 5), (48, 3), (64, 4), (1000, 1)])
def test_rows_of_paged_positions(rules, bs, blocks):
    """Every position: the row of its page if that lies in the cache, else none; never a row outside."""
    rng = np.random.default_rng(bs)
    rows = 7 * bs + 3                                   # the last page is cut short
    table = rng.integers(0, 8, (3, blocks + 2), dtype=np.int32)
    table[1, 0], table[2, blocks - 1] = BAD_PAGES[0], BAD_PAGES[1]
    table[0, blocks - 1] = BAD_PAGES[2]
    none = 0
    for b in range(3):
        for p in [-(2 ** 62), -1, *range(blocks * bs + 3), 2 ** 31, 2 ** 40]:
            got = rules.seq_row(table.ctypes.data, blocks + 2, blocks, bs, 0, b, p, rows)
            want = -1
            if 0 <= p < blocks * bs:
                r = int(table[b, p // bs]) * bs + p % bs
                want = r if 0 <= r < rows else -1
            assert got == want, (b, p)
            none += got < 0
    assert none > 3 * bs


def test_rows_of_flat_positions(rules):
    """A sequence's rows end where the next one's begin; the largest offsets pass 32 bits and stay in the cache."""
    big = 2 ** 31 - 1
    assert rules.seq_row(None, 0, 0, 0, 100, 2, 99, 300) == 299
    assert rules.seq_row(None, 0, 0, 0, 100, 2, 100, 10 ** 6) == -1
    assert rules.seq_row(None, 0, 0, 0, 100, 2, 99, 299) == -1
    assert rules.seq_row(None, 0, 0, 0, 0, 5, 41, 42) == 41
    assert rules.seq_row(None, 0, 0, 0, 2 ** 20, 2047, 2 ** 20 - 1, big) == -1
    assert rules.seq_row(None, 0, 0, 0, 2 ** 20, 2047, 2 ** 20 - 2, big) == big - 1
    assert rules.seq_row(None, 0, 0, 0, 2 ** 40, big, 1, big) == -1


def test_positions(rules):
    indptr = np.array([2, 5, 5, 9], np.int32)
    lens = np.array([3, 7, 2 ** 31 - 1], np.int32)
    at = lambda b, t: rules.seq_position(indptr.ctypes.data, lens.ctypes.data, b, t)
    assert [at(0, t) for t in (2, 3, 4)] == [0, 1, 2]
    assert [at(2, t) for t in (5, 8)] == [2 ** 31 - 5, 2 ** 31 - 2]
    lens[2] = 1                                         # fewer positions than tokens: the first have none
    assert [at(2, t) for t in range(5, 9)] == [-3, -2, -1, 0]


@pytest.mark.parametrize("m", [32, 128])
@pytest.mark.parametrize("H", [1, 3, 8, 16, 17, 24, 40, 64, 96, 100, 128, 200])
def test_blocks_hold_every_row(rules, H, m):
    """Each sequence's blocks suffice for its rows, and at most one block a sequence stays empty."""
    assert rules.seq_common(H, m) == math.gcd(H, m)
    rng = np.random.default_rng(H * m)
    for _ in range(30):
        B = int(rng.integers(1, 40))
        new = rng.integers(0, 6, B) * rng.integers(0, 2, B)
        ends = np.concatenate([[0], np.cumsum(new)]) + int(rng.integers(0, 4))
        start = [rules.seq_block_start(int(ends[b]), b, H, m) for b in range(B + 1)]
        for b in range(B):
            need = -(-int(new[b]) * H // m)
            assert start[b + 1] - start[b] >= need, (H, m, b)
            assert start[b + 1] - start[b] <= need + 1
    # rows of one token that fill their blocks leave none empty
    if H % m == 0:
        assert [rules.seq_block_start(b, b, H, m) for b in range(9)] == [b * H // m for b in range(9)]


def test_block_start_of_the_largest_calls(rules):
    T, H, m = (2 ** 31 - 1) // 200 - 1000, 200, 32
    assert rules.seq_block_start(T, 1000, H, m) == (T * H + 1000 * (m - math.gcd(H, m))) // m


def test_parts(rules):
    """Exact below 2^20, never too few, whatever way the reciprocal is off by one step."""
    rng = np.random.default_rng(1)
    cases = [(a, b) for a in range(0, 700) for b in (1, 2, 3, 7, 24, 31, 64)]
    for _ in range(20000):
        a, b = min(int(2 ** rng.uniform(0, 31)), 2 ** 31 - 1), int(2 ** rng.uniform(0, 26))
        cases += [(a, b)] + [(min(2 ** 31 - 1, max(0, a // b * b + d)), b) for d in (-1, 0, 1)]
    for a, b in cases:
        r = np.float32(1) / np.float32(b)
        want = -(-a // b)
        for x in (r, np.nextafter(r, np.float32(0)), np.nextafter(r, np.float32(2))):
            got = rules.seq_parts(a, b, float(x))
            assert got == want if want < 2 ** 20 else want <= got <= want * (1 + 2.0 ** -19), (a, b, got, want)


# ------------------------------------------------------------------ layouts

def _c_layout(name, fields, tmp_path):
    src = tmp_path / "layout.c"
    body = "".join(f'printf("%zu\\n", offsetof({name}, {f}));\n' for f in fields)
    src.write_text(f'#include <stddef.h>\n#include <stdio.h>\n#include "dsa_chunk.h"\n'
                   f'int main(void){{\nprintf("%zu\\n", sizeof({name}));\n{body}return 0;}}\n')
    exe = str(tmp_path / "layout")
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(ROOT, "include"), str(src), "-o", exe], check=True)
    v = [int(x) for x in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split()]
    return v[0], v[1:]


STRUCTS = [(abi.NormRopeRows, "dsa_norm_rope_rows", None),
           (abi.QkNormRopeArgs, "dsa_qk_norm_rope_args", abi.pack_norm_rope),
           (abi.KvAppendArgs, "dsa_kv_append_args", abi.pack_append),
           (abi.ChunkArgs, "dsa_mla_chunk_args", abi.pack_chunk)]


@pytest.mark.parametrize("cls,name,pack", STRUCTS, ids=[s[1] for s in STRUCTS])
def test_layouts(cls, name, pack, tmp_path):
    fields = [f for f, _ in cls._fields_]
    size, offsets = _c_layout(name, fields, tmp_path)
    assert ctypes.sizeof(cls) == size and [getattr(cls, f).offset for f in fields] == offsets
    if pack is None:
        return
    # the packed bytes are the struct's, field by field
    leaves = []

    def walk(c, path):
        for f, t in c._fields_:
            if hasattr(t, "_fields_"):
                walk(t, path + [f])
            else:
                leaves.append((path + [f], t))

    walk(cls, [])
    values = [float(i) + 0.5 if t is ctypes.c_float else 16 * (i + 1) for i, (_, t) in enumerate(leaves)]
    data = pack(*values)
    assert len(data) == size
    s = cls.from_buffer_copy(data)
    for (path, t), v in zip(leaves, values):
        x = s
        for f in path:
            x = getattr(x, f)
        assert x == v, path


def test_enums_match_the_header(tmp_path):
    src = tmp_path / "e.c"
    src.write_text('#include <stdio.h>\n#include "dsa_chunk.h"\nint main(void){printf("%d %d %d %d %d %d\\n", DSA_NORM_NONE, '
                   'DSA_NORM_RMS, DSA_NORM_LAYER, DSA_ROPE_NONE, DSA_ROPE_INTERLEAVED, DSA_ROPE_HALVES);return 0;}\n')
    exe = str(tmp_path / "e")
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(ROOT, "include"), str(src), "-o", exe], check=True)
    v = [int(x) for x in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split()]
    assert [abi.NORMS[k] for k in ("none", "rms", "layer")] == v[:3]
    assert [abi.ROPES[k] for k in (None, "interleaved", "halves")] == v[3:]


# ------------------------------------------------------------------ refusals of the C entries

@pytest.fixture(scope="module")
def lib():
    return abi.load_library()


def _set(a, kw):
    for k, v in kw.items():
        x, f = a, k
        if "." in k:
            head, f = k.split(".")
            x = getattr(a, head)
        setattr(x, f, v)
    return a


def _prep(**kw):
    a = abi.QkNormRopeArgs()
    base = {"q.x": 0x1000, "q.stride_t": 16 * 576, "q.stride_h": 576, "q.out": 0x2000, "q.out_stride_t": 16 * 576,
            "q.out_stride_h": 576, "q.weight": 0x3000, "q.H": 16, "q.norm": 1, "cos_sin": 0x4000, "n_pos": 10,
            "positions": 0x5004, "T": 3, "D": 576, "norm_dim": 512, "rot_off": 512, "rope": 1, "eps": 1e-6}
    return _set(a, {**base, **kw})


PREP_BAD = [
    (dict(T=-1), SHAPE), (dict(B=-1), SHAPE), (dict(n_pos=-1), SHAPE), (dict(D=64), UNSUPPORTED), (dict(D=577), UNSUPPORTED),
    (dict(rope=3), UNSUPPORTED), (dict(rope=-1), UNSUPPORTED), (dict(norm_dim=520), SHAPE), (dict(norm_dim=0), SHAPE),
    (dict(norm_dim=12), SHAPE), (dict(D=128, norm_dim=136), SHAPE), (dict(rot_off=513), SHAPE), (dict(rot_off=576), SHAPE),
    (dict(rot_off=-64), SHAPE), (dict(rot_off=32), SHAPE), (dict(eps=-1.0), SHAPE), (dict(eps=math.nan), SHAPE),
    ({"q.H": -1}, SHAPE), ({"q.norm": 3}, UNSUPPORTED), ({"q.norm": 0}, UNSUPPORTED),
    ({"q.norm": 0, "q.weight": 0, "q.bias": 0x10}, UNSUPPORTED), ({"q.x": 0}, NULL), ({"q.out": 0}, NULL),
    ({"q.stride_t": 12}, STRIDE), ({"q.stride_h": 580}, STRIDE), ({"q.stride_t": -8}, STRIDE), ({"q.out_stride_h": 568}, STRIDE),
    ({"q.out_stride_t": 568}, STRIDE), ({"q.out_stride_t": 0}, STRIDE), ({"q.out": 0x1000, "q.stride_h": 584}, STRIDE),
    ({"q.x": 0x1008}, STRIDE), ({"q.out": 0x2008}, STRIDE), ({"q.weight": 0x3004}, STRIDE), ({"q.bias": 0x3004}, STRIDE),
    ({"k.H": 1}, NULL), ({"k.H": 1, "k.norm": 7}, UNSUPPORTED), ({"cos_sin": 0}, NULL), ({"cos_sin": 0x4008}, STRIDE),
    ({"positions": 0, "B": 1}, NULL), ({"positions": 0, "B": 1, "q_indptr": 0x6000}, NULL),
    ({"positions": 0, "B": 1, "seq_lens": 0x6000}, NULL), ({"T": 2 ** 31 - 1, "q.H": 2 ** 20}, SHAPE),
    ({"T": 2 ** 25 + 1, "q.H": 16}, SHAPE),
]


@pytest.mark.parametrize("kw,code", PREP_BAD, ids=[f"{i}" for i in range(len(PREP_BAD))])
def test_norm_rope_refuses(lib, kw, code):
    assert lib.dsa_qk_norm_rope(ctypes.byref(_prep(**kw)), None) == code


def test_norm_rope_of_nothing(lib):
    assert lib.dsa_qk_norm_rope(None, None) == NULL
    for kw in (dict(T=0), {"q.H": 0}, {"T": 0, "q.x": 0, "q.out": 0}, {"positions": 0, "B": 0}):
        assert lib.dsa_qk_norm_rope(ctypes.byref(_prep(**kw)), None) == 0, kw


def _append(**kw):
    a = abi.KvAppendArgs()
    base = dict(kv=0x1000, kv_stride_t=576, weight=0x2000, cache=0x10000, cache_rows=640, kv_format=abi.KV_FP8_656, norm=1,
                rope=1, cos_sin=0x3000, n_pos=100, q_indptr=0x4004, seq_lens=0x5004, block_table=0x6004,
                block_table_stride=10, table_blocks=10, block_size=64, T=3, B=1, eps=1e-6, index_eps=1e-6)
    return _set(a, {**base, **kw})


INDEX = dict(index_k=0x7000, index_stride_t=128, index_cache=0x8000, index_rows=640)
MX = dict(kv_format=abi.KV_MXFP8, cache_scale=0x9000, cache_rope=0xa000)
APPEND_BAD = [
    (dict(T=-1), SHAPE), (dict(B=-1), SHAPE), (dict(n_pos=-1), SHAPE), (dict(cache_rows=-1), SHAPE), (dict(index_rows=-1), SHAPE),
    (dict(rope=3), UNSUPPORTED), (dict(index_rope=-1), UNSUPPORTED), (dict(index_norm=3), UNSUPPORTED), (dict(norm=2), UNSUPPORTED),
    (dict(norm=-1), UNSUPPORTED), (dict(norm=0), UNSUPPORTED), (dict(index_weight=0x10), UNSUPPORTED),
    (dict(index_bias=0x10), UNSUPPORTED), (dict(kv_format=-1), FORMAT), (dict(kv_format=99), FORMAT), (dict(eps=-1e-9), SHAPE),
    (dict(eps=math.nan), SHAPE), (dict(index_eps=math.nan), SHAPE), (dict(block_size=0), SHAPE), (dict(table_blocks=-1), SHAPE),
    (dict(block_size=2 ** 20, table_blocks=2 ** 12), SHAPE), (dict(block_table_stride=-1), STRIDE),
    (dict(block_table=0, kv_batch_stride=-1), STRIDE), (dict(block_table=0, B=2), STRIDE), (dict(q_indptr=0), NULL),
    (dict(seq_lens=0), NULL), (dict(cos_sin=0), NULL), (dict(cos_sin=0x3008), STRIDE), (dict(cache=0), NULL),
    ({**MX, "cache_scale": 0}, NULL), ({**MX, "cache_rope": 0}, NULL), (dict(stride_row=640), STRIDE), (dict(stride_row=660), STRIDE),
    (dict(kv_format=abi.KV_BF16, stride_row=580), STRIDE), (dict(kv_format=abi.KV_BF16, stride_row=568), STRIDE),
    ({**MX, "rope_stride_row": 60}, STRIDE), ({**MX, "rope_stride_row": 68}, STRIDE), ({**MX, "scale_stride_row": 24}, STRIDE),
    ({**MX, "scale_stride_row": 8}, STRIDE), (dict(kv_stride_t=-8), STRIDE), (dict(kv_stride_t=580), STRIDE), (dict(kv=0x1002), STRIDE),
    (dict(weight=0x2004), STRIDE), (dict(cache=0x10008), STRIDE), ({**MX, "cache_scale": 0x9004}, STRIDE),
    ({**MX, "cache_rope": 0xa008}, STRIDE), ({**INDEX, "index_cache": 0}, NULL), ({**INDEX, "index_stride_row": 120}, STRIDE),
    ({**INDEX, "index_stride_row": 132}, STRIDE), ({**INDEX, "index_stride_t": -8}, STRIDE), ({**INDEX, "index_stride_t": 4}, STRIDE),
    ({**INDEX, "index_k": 0x7008}, STRIDE), ({**INDEX, "index_cache": 0x8008}, STRIDE),
    (dict(T=2 ** 26), SHAPE), ({**INDEX, "T": 2 ** 26 - 2 ** 20}, SHAPE),
    ({**INDEX, "index_norm": 2, "index_weight": 0x14}, STRIDE), ({**INDEX, "index_norm": 2, "index_bias": 0x14}, STRIDE),
]


@pytest.mark.parametrize("kw,code", APPEND_BAD, ids=[f"{i}" for i in range(len(APPEND_BAD))])
def test_append_refuses(lib, kw, code):
    assert lib.dsa_kv_append(ctypes.byref(_append(**kw)), None) == code


def test_append_of_nothing(lib):
    assert lib.dsa_kv_append(None, None) == NULL
    for kw in (dict(T=0), dict(B=0), dict(kv=0), dict(T=0, q_indptr=0, seq_lens=0, cache=0)):
        assert lib.dsa_kv_append(ctypes.byref(_append(**kw)), None) == 0, kw


def _chunk(**kw):
    a = abi.ChunkArgs()
    base = dict(q=0x1000, q_stride_t=16 * 576, q_stride_h=576, q_indptr=0x2004, seq_lens=0x3004, kv_cache=0x10000,
                kv_total_rows=6400, kv_format=abi.KV_BF16, block_size=64, block_table=0x4004, block_table_stride=100,
                out=0x5008, o_stride_t=16 * 512, o_stride_h=512, lse=0x6004, table_blocks=100, T=2, B=1, H=16, causal=1,
                max_kv_len=6000, num_splits=4, sm_scale=0.07)
    return _set(a, {**base, **kw})


CHUNK_BAD = [
    (dict(kv_format=abi.KV_BF16_D512), FORMAT), (dict(kv_format=abi.KV_MXFP8), FORMAT), (dict(kv_format=-1), FORMAT),
    (dict(T=-1), SHAPE), (dict(B=-1), SHAPE), (dict(H=0), SHAPE), (dict(max_kv_len=-1), SHAPE), (dict(max_kv_len=2 ** 31 - 1), SHAPE),
    (dict(kv_total_rows=-1), SHAPE), (dict(kv_total_rows=2 ** 31), SHAPE), (dict(num_splits=-1), SPLITS), (dict(num_splits=65), SPLITS),
    (dict(T=2 ** 27), SHAPE), (dict(B=2 ** 24), SHAPE), (dict(T=2 ** 25, num_splits=1), SHAPE), (dict(T=2 ** 25), SHAPE),
    (dict(T=2 ** 22, num_splits=2), SHAPE), (dict(kv_stride_row=568), STRIDE), (dict(kv_stride_row=580), STRIDE),
    (dict(kv_stride_row=2 ** 31), STRIDE), (dict(kv_format=abi.KV_FP8_656, kv_stride_row=664), STRIDE), (dict(block_size=0), SHAPE),
    (dict(table_blocks=-1), SHAPE), (dict(block_size=2 ** 20, table_blocks=2 ** 12), SHAPE), (dict(block_table_stride=-1), STRIDE),
    (dict(block_table=0, kv_batch_stride=-1), STRIDE), (dict(sm_scale=0.0), UNSUPPORTED), (dict(sm_scale=-1.0), UNSUPPORTED),
    (dict(sm_scale=math.nan), UNSUPPORTED), (dict(sm_scale=math.inf), UNSUPPORTED), (dict(q=0), NULL), (dict(out=0), NULL),
    (dict(q_indptr=0), NULL), (dict(seq_lens=0), NULL), (dict(kv_cache=0), NULL), (dict(q_stride_t=-8), STRIDE),
    (dict(q_stride_h=580), STRIDE), (dict(o_stride_t=514), STRIDE), (dict(o_stride_h=-4), STRIDE), (dict(o_stride_h=0), STRIDE),
    (dict(o_stride_h=508), STRIDE), (dict(o_stride_t=0), STRIDE), (dict(q=0x1008), STRIDE), (dict(kv_cache=0x10008), STRIDE),
    (dict(out=0x5004), STRIDE),
]


@pytest.mark.parametrize("kw,code", CHUNK_BAD, ids=[f"{i}" for i in range(len(CHUNK_BAD))])
def test_chunk_refuses(lib, kw, code):
    """All three entries, before they look at a workspace."""
    a = ctypes.byref(_chunk(**kw))
    n, size = ctypes.c_int32(-5), ctypes.c_size_t(7)
    assert lib.dsa_mla_chunk(a, 0x100000, 1 << 40, None) == code
    assert lib.dsa_mla_chunk_num_splits(a, ctypes.byref(n)) == code and n.value == -5
    assert lib.dsa_mla_chunk_workspace_size(a, ctypes.byref(size)) == code and size.value == 7


def test_chunk_of_nothing_and_null(lib):
    assert lib.dsa_mla_chunk(None, None, 0, None) == NULL
    assert lib.dsa_mla_chunk_num_splits(None, None) == NULL
    assert lib.dsa_mla_chunk_workspace_size(ctypes.byref(_chunk()), None) == NULL
    size = ctypes.c_size_t(7)
    for kw in (dict(T=0), dict(B=0), dict(T=0, q=0, out=0)):
        a = ctypes.byref(_chunk(**kw))
        assert lib.dsa_mla_chunk(a, None, 0, None) == 0, kw
        assert lib.dsa_mla_chunk_workspace_size(a, ctypes.byref(size)) == 0 and size.value == 0


def test_chunk_workspace(lib):
    """A split call's partials and the 16 bytes behind them; too small, misaligned or missing is refused."""
    a = _chunk()
    at = ctypes.byref(a)
    size = ctypes.c_size_t(0)
    assert lib.dsa_mla_chunk_workspace_size(at, ctypes.byref(size)) == 0
    need = 4 * 2 * 16 * 513 * 4 + 16
    assert size.value == need
    for ws, n in ((None, need), (0x100000, need - 1), (0x100008, need), (0x100000, 0)):
        assert lib.dsa_mla_chunk(at, ws, n, None) == WORKSPACE
    a.num_splits = 1
    assert lib.dsa_mla_chunk_workspace_size(at, ctypes.byref(size)) == 0 and size.value == 0


@pytest.mark.parametrize("fmt", [abi.KV_BF16, abi.KV_FP8_656])
@pytest.mark.parametrize("T,B,H,longest", [(1, 1, 1, 0), (1, 1, 128, 1), (1, 1, 128, 33), (1, 1, 128, 100000), (64, 64, 16, 9000),
                                           (65, 65, 16, 9000), (4096, 2, 128, 4096), (2 ** 20, 1, 16, 2 ** 20),
                                           (1, 1, 1, 2147481599), (2 ** 22, 1, 127, 64), (0, 0, 1, 0)])
def test_chunk_automatic_splits(lib, fmt, T, B, H, longest):
    """From 1 to 64, no more than there are tiles of 32 positions (twice the planned ones, where the device
    deals them), with a workspace that goes by them; an unsplit call needs none."""
    a = _chunk(T=T, B=B, H=H, max_kv_len=longest, num_splits=0, q_stride_t=H * 576, o_stride_t=H * 512, kv_format=fmt)
    n, size = ctypes.c_int32(0), ctypes.c_size_t(0)
    assert lib.dsa_mla_chunk_num_splits(ctypes.byref(a), ctypes.byref(n)) == 0
    assert lib.dsa_mla_chunk_workspace_size(ctypes.byref(a), ctypes.byref(size)) == 0
    assert 1 <= n.value <= 64 and n.value <= max(1, 2 * (longest // 32))
    assert size.value == (n.value * T * H * 513 * 4 + 16 if n.value > 1 and T else 0)


# ------------------------------------------------------------------ refusals of the Python entries

def test_host_tensors_are_refused():
    """No fallback: tensors on the host are an error that names the argument."""
    q, kv = torch.zeros(2, 16, 576, dtype=torch.bfloat16), torch.zeros(4, 64, 576, dtype=torch.bfloat16)
    indptr, lens = torch.tensor([0, 2], dtype=torch.int32), torch.tensor([5], dtype=torch.int32)
    table = torch.zeros(1, 4, dtype=torch.int32)
    with pytest.raises(ValueError, match="q must"):
        dsa.mla_chunk(q, kv, indptr, lens, 0.07, block_table=table)
    with pytest.raises(ValueError, match="q must"):
        dsa.qk_norm_rope(q, torch.zeros(9, 64), torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="q_indptr must be a device tensor"):
        dsa.kv_append(q[:, 0], kv, indptr, lens, torch.zeros(9, 64), block_table=table)


def test_rows_of_caches():
    """(rows, stride; 0 = dense) of a cache; rows that lie on one another or unevenly are refused, not taken
    for dense ones (whose memory would end past the tensor's)."""
    t = torch.zeros(6, 4, 576)
    assert dsa._rows(t, 576, "cache") == (24, 0)
    assert dsa._rows(torch.zeros(6, 4, 640)[..., :576], 576, "cache") == (24, 640)
    assert dsa._rows(torch.zeros(6, 2, 1, 576)[:, 0], 576, "cache") == (6, 1152)
    assert dsa._rows(torch.zeros(1, 576).expand(1, 576), 576, "cache") == (1, 0)
    for bad in (torch.zeros(1, 576).expand(100, 576), torch.zeros(1, 1, 576).expand(100, 1, 576),
                torch.zeros(1, 4, 576).expand(6, 4, 576), torch.zeros(6, 1, 576).expand(6, 4, 576),
                t[:, :3], t.transpose(0, 1), torch.zeros(6 * 576).as_strided((6, 576), (64, 1)),
                torch.zeros(576, 6).t()):
        with pytest.raises(ValueError, match="cache must"):
            dsa._rows(bad, 576, "cache")


def test_shapes_are_refused_before_the_device():
    with pytest.raises(ValueError, match="q must"):
        dsa.mla_chunk(torch.zeros(2, 576, dtype=torch.bfloat16), None, None, None, 0.07)
    with pytest.raises(ValueError, match="q must"):
        dsa.qk_norm_rope(torch.zeros(2, 128, dtype=torch.bfloat16))
