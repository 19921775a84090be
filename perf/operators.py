"""The operators in front of and beside sparse attention, as measurable cases.

Three kinds, all over the same ragged chunk of new tokens (``indptr``: where each sequence's
tokens start, ``lens``: each sequence's length with them, ``table``: its cache pages):

* ``prep``    norms of queries and keys for each head with the position rotation in the same pass
* ``append``  latent rows (and index keys) normed, rotated and written into the paged cache
* ``chunk``   dense attention of the chunk's tokens over the paged latent cache

With ``own`` false, ``run`` computes them from elementary torch operations in 32 bits; with
``own`` true through ``opfoundry_amd.dsa``.  ``exact`` restates them in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

D_QK, D_VO, D_ROPE, D_INDEX = 576, 512, 64, 128
SM_SCALE = 1.0 / math.sqrt(192.0)
EPS = 1e-6
PAGE = 64
GOLDEN = 0.6180339887498949
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu

# width, first rotated column, values under the norm, of each kind of row
SHAPES = {"mla": (576, 512, 512), "v4": (512, 448, 512), "index": (128, 0, 128)}
# bytes of one cache row
ROW_BYTES = {"bf16": 1152, "fp8": 656, "v4": 1024, "mx": 656, "v4fp8": 448 + 14 + 128}


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # One session's decode step: its token's latent row and index key go into the caches.  Latency.
        dict(name="append_fp8_b1", kind="append", rows="fp8", B=1, lo=1, hi=1, ctx=1500, index=True, norm=True),
        # A full decode batch with one speculative token each.
        dict(name="append_bf16_b64", kind="append", rows="bf16", B=64, lo=2, hi=2, ctx=1000, index=True, norm=True),
        # Three prompts of one prefill step, uneven lengths.
        dict(name="append_fp8_prompts", kind="append", rows="fp8", B=3, lo=1200, hi=4500, ctx=777, index=True, norm=True),
        # A V4 chunk into its fp8 pool (two streams, power-of-two scales).
        dict(name="append_v4fp8_4099", kind="append", rows="v4fp8", B=1, lo=4099, hi=4099, ctx=640, index=False, norm=True),
        # A decode step of two tokens: absorbed queries rotated, the latent key normed and rotated.
        dict(name="prep_mla_t2", kind="prep", shape="mla", T=2, H=128, Hk=1, ctx=4000, qn="none", kn="rms",
             style="interleaved", inverse=False),
        # A V4 prefill's queries (norm for each head) and its key rows.
        dict(name="prep_v4_4096", kind="prep", shape="v4", T=4096, H=128, Hk=1, ctx=0, qn="rms", kn="rms",
             style="interleaved", inverse=False),
        # The index queries and keys of a ragged chunk.
        dict(name="prep_index_1531", kind="prep", shape="index", T=1531, H=64, Hk=1, ctx=20011, qn="none", kn="layer",
             style="halves", inverse=False),
        # One session's decode step with a context shorter than any top-k: every row is attended.  Latency.
        dict(name="chunk_fp8_b1", kind="chunk", rows="fp8", B=1, lo=1, hi=1, H=128, ctx=1500, ragged=False),
        # One rank of an 8-way head shard decoding long ragged contexts with up to 3 speculative tokens.
        dict(name="chunk_bf16_b16_h16", kind="chunk", rows="bf16", B=16, lo=1, hi=4, H=16, ctx=20011, ragged=True),
        # A prefill chunk of 1024 tokens over a long context.
        dict(name="chunk_bf16_1024", kind="chunk", rows="bf16", B=1, lo=1024, hi=1024, H=128, ctx=8192, ragged=False),
        # Two whole prompts on the fp8 cache.
        dict(name="chunk_fp8_prompts", kind="chunk", rows="fp8", B=2, lo=1700, hi=2048, H=128, ctx=0, ragged=False),
        # A mixed step on an odd head shard: single tokens beside chunks.
        dict(name="chunk_bf16_mixed_h40", kind="chunk", rows="bf16", B=7, lo=1, hi=301, H=40, ctx=5000, ragged=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    kind = rng.choice(["append", "prep", "chunk", "chunk"])
    if kind == "append":
        rows = rng.choice(["fp8", "fp8", "bf16", "v4", "mx", "v4fp8"])
        B = _log(rng, 1, 128)
        hi = _log(rng, 1, 9000 // B)
        return dict(kind=kind, rows=rows, B=B, lo=rng.randint(1, hi), hi=hi, ctx=_log(rng, 1, 40000 // B),
                    index=rng.random() < 0.6, norm=rng.random() < 0.8)
    if kind == "prep":
        shape = rng.choice(["mla", "v4", "v4", "index"])
        H = rng.choice([16, 40, 64, 128]) if shape != "index" else rng.choice([32, 64])
        T = _log(rng, 1, 4096 * 128 * 512 // (H * SHAPES[shape][0]) // 2)
        inverse = shape == "v4" and rng.random() < 0.3      # an output's rotation taken back: no norm, no key
        return dict(kind=kind, shape=shape, T=T, H=H, Hk=0 if inverse else 1, ctx=_log(rng, 1, 100000),
                    qn="rms" if shape == "v4" and not inverse else "none", kn="layer" if shape == "index" else "rms",
                    style="halves" if shape == "index" else rng.choice(["interleaved", "interleaved", "halves"]),
                    inverse=inverse)
    rows, H = rng.choice(["bf16", "fp8"]), rng.choice([16, 16, 32, 40, 64, 96, 128, 128])
    B = _log(rng, 1, 64)
    if rng.random() < 0.5:                                  # decode: a few tokens each over long contexts
        hi, ctx = rng.randint(1, 4), _log(rng, 200, 1_000_000 // B)
    else:                                                   # chunks
        B = min(B, 8)
        hi, ctx = _log(rng, 5, 2048), _log(rng, 1, 16000)
    c = dict(kind=kind, rows=rows, B=B, lo=rng.randint(1, hi), hi=hi, H=H, ctx=ctx, ragged=rng.random() < 0.7)
    while work(c)["flops"] > 2.4e12 or B * c["hi"] * H * (ctx + c["hi"]) > 1.2e9:
        c["hi"] = max(1, c["hi"] * 2 // 3)
        c["ctx"] = ctx = max(1, ctx * 4 // 5)
        c["lo"] = min(c["lo"], c["hi"])
    return c


# ------------------------------------------------------------------ sizes that follow from a case

def _spread(count, lo, hi):
    """`count` whole numbers spread unevenly over [lo, hi]: the same ones for every seed."""
    return [lo + int((hi - lo + 1) * (((i + 1) * GOLDEN) % 1.0)) for i in range(count)]


def _chunk_of(c):
    """New tokens of each sequence, and its length with them."""
    new = _spread(c["B"], c["lo"], c["hi"])
    ctx = _spread(c["B"], c["ctx"] // 3, c["ctx"]) if c.get("ragged", True) else [c["ctx"]] * c["B"]
    return new, [n + x for n, x in zip(new, ctx)]


def work(case):
    c = case
    if c["kind"] == "prep":
        D = SHAPES[c["shape"]][0]
        values = c["T"] * (c["H"] + c["Hk"]) * D
        return {"bytes": 4 * values + c["T"] * (4 * D_ROPE + 4), "flops": 6 * values}
    new, lens = _chunk_of(c)
    T = sum(new)
    if c["kind"] == "append":
        width = 2 * (D_QK if c["rows"] in ("bf16", "fp8", "mx") else 512)
        per = width + ROW_BYTES[c["rows"]] + 4 * D_ROPE + (4 * D_INDEX if c["index"] else 0)
        return {"bytes": T * per + 8 * c["B"], "flops": 10 * T * (width // 2)}
    pairs = sum(n * s - n * (n - 1) // 2 for n, s in zip(new, lens))
    return {"bytes": sum(lens) * ROW_BYTES[c["rows"]] + T * c["H"] * (2 * D_QK + 2 * D_VO + 4),
            "flops": 2 * c["H"] * (D_QK + D_VO) * pairs}


# ------------------------------------------------------------------ inputs

def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _bf16(g, *shape):
    return _randn(g, *shape).to(torch.bfloat16)


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _angles(n):
    """cos (first 32 columns) and sin of the rotation at positions 0..n-1, as fp32: computed in 64
    bits, as far positions need."""
    at = torch.arange(n, device="cuda", dtype=torch.float64)
    freq = 10000.0 ** (-torch.arange(0, D_ROPE, 2, device="cuda", dtype=torch.float64) / D_ROPE)
    a = at[:, None] * freq[None, :]
    return torch.cat([torch.cos(a), torch.sin(a)], 1).float()


def _codes(g, n, width):
    return _randn(g, n, width).to(E4M3).view(torch.uint8)


def _cache(g, rows, n):
    """n cache rows in use: the tensors of the format."""
    if rows in ("bf16", "v4"):
        return (_bf16(g, n, D_QK if rows == "bf16" else 512),)
    if rows == "fp8":
        out = torch.empty((n, 656), dtype=torch.uint8, device="cuda")
        out[:, :512] = (_randn(g, n, 512) * 100).clamp(-448, 448).to(E4M3).view(torch.uint8)
        out[:, 512:528] = (0.008 + 0.004 * torch.rand((n, 4), generator=g, device="cuda")).view(torch.uint8)
        out[:, 528:] = _bf16(g, n, D_ROPE).view(torch.uint8)
        return (out,)
    if rows == "mx":
        scale = torch.randint(119, 122, (n, 16), generator=g, device="cuda").to(torch.uint8)
        return _codes(g, n, 512), scale, _bf16(g, n, D_ROPE)
    nope = torch.zeros((n, 512), dtype=torch.uint8, device="cuda")
    nope[:, :448] = _codes(g, n, 448)
    nope[:, 448:462] = torch.randint(119, 122, (n, 14), generator=g, device="cuda").to(torch.uint8)
    return nope, _bf16(g, n, D_ROPE)


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    if c["kind"] == "prep":
        D, off, norm = SHAPES[c["shape"]]
        s = dict(c=c, q=_bf16(g, c["T"], c["H"], D), pos=_int32(range(c["ctx"], c["ctx"] + c["T"])),
                 cs=_angles(c["ctx"] + c["T"]))
        if c["Hk"]:
            s["k"] = _bf16(g, c["T"], c["Hk"], D)
            s["w"] = 1.0 + 0.1 * _randn(g, norm)
            s["b"] = 0.1 * _randn(g, norm) if c["kn"] == "layer" else None
        return s
    new, lens = _chunk_of(c)
    blocks = -(-max(lens) // PAGE)
    s = dict(c=c, new=_int32(new), lens=_int32(lens), longest=max(lens), widest=max(new),
             indptr=_int32([0] + torch.tensor(new).cumsum(0).tolist()),
             table=torch.randperm(c["B"] * blocks, generator=g, device="cuda").to(torch.int32).view(c["B"], blocks))
    T, n = sum(new), c["B"] * blocks * PAGE
    s["cache"] = _cache(g, c["rows"], n)
    if c["kind"] == "chunk":
        s["q"] = _bf16(g, T, c["H"], D_QK)
        return s
    s["x"] = _bf16(g, T, D_QK if c["rows"] in ("bf16", "fp8", "mx") else 512)
    s["w"] = 1.0 + 0.1 * _randn(g, 512) if c["norm"] else None
    s["cs"] = _angles(max(lens))
    if c["index"]:
        s["ix"], s["icache"] = _bf16(g, T, D_INDEX), _bf16(g, n, D_INDEX)
        s["iw"], s["ib"] = 1.0 + 0.1 * _randn(g, D_INDEX), 0.1 * _randn(g, D_INDEX)
    return s


# ------------------------------------------------------------------ the plain forms (32 bits)

def _normed(x, kind, n, w, b):
    """The first n columns of x under a norm, the others as they are."""
    if kind == "none":
        return x
    y = x[..., :n]
    if kind == "layer":
        y = y - y.mean(-1, keepdim=True)
    y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS)
    if w is not None:
        y = y * w
    if b is not None:
        y = y + b
    return torch.cat([y, x[..., n:]], -1)


def _rotated(x, off, cs, style, inverse=False):
    """Columns off..off+63 of x turned by the angles cs [..., 64], which broadcast over x's rows."""
    r = x[..., off:off + D_ROPE]
    cos, sin = cs[..., :32], cs[..., 32:]
    if inverse:
        sin = -sin
    if style == "interleaved":
        u, v = r[..., 0::2], r[..., 1::2]
        t = torch.stack([u * cos - v * sin, v * cos + u * sin], -1).flatten(-2)
    else:
        u, v = r[..., :32], r[..., 32:]
        t = torch.cat([u * cos - v * sin, v * cos + u * sin], -1)
    return torch.cat([x[..., :off], t, x[..., off + D_ROPE:]], -1)


def _places(s):
    """Position and cache row of every token of the chunk."""
    t = torch.arange(s["q" if "q" in s else "x"].shape[0], device="cuda")
    b = (t[:, None] >= s["indptr"][None, 1:]).sum(1)
    pos = (s["lens"] - s["new"])[b] + t - s["indptr"][b]
    return b, pos, s["table"][b, pos // PAGE].long() * PAGE + pos % PAGE


def _plain_prep(s):
    c = s["c"]
    _, off, n = SHAPES[c["shape"]]
    cs = s["cs"][s["pos"].long()][:, None]
    got = [_rotated(_normed(s["q"].float(), c["qn"], n, None, None), off, cs, c["style"], c["inverse"])]
    if c["Hk"]:
        got.append(_rotated(_normed(s["k"].float(), c["kn"], n, s["w"], s["b"]), off, cs, c["style"]))
    return [x.to(torch.bfloat16) for x in got]


def _power_scaled(y, group):
    """y [n, m] in groups as e4m3 codes and the exponent bytes of their scales: the least power of two
    with every |value| / 2^e at most 448."""
    v = y.view(y.shape[0], -1, group)
    top = v.abs().amax(-1)
    m, e = torch.frexp(top / 448.0)
    e = torch.where(m == 0.5, e - 1, e).clamp(min=-126)
    e = torch.where(top > 0, e, torch.zeros_like(e))
    codes = torch.ldexp(v, -e[..., None]).clamp(-448, 448).to(E4M3)
    return codes.view(y.shape).view(torch.uint8), (e + 127).to(torch.uint8)


def _plain_append(s):
    c, cache = s["c"], s["cache"]
    _, pos, row = _places(s)
    cs = s["cs"][pos]
    off = 512 if c["rows"] in ("bf16", "fp8", "mx") else 448
    x = _normed(s["x"].float(), "rms" if c["norm"] else "none", 512, s["w"], None)
    x = _rotated(x, off, cs, "interleaved")
    rope = x[:, off:].to(torch.bfloat16)
    if c["rows"] in ("bf16", "v4"):
        cache[0][row] = x.to(torch.bfloat16)
    elif c["rows"] == "fp8":
        v = x[:, :512].view(-1, 4, 128)
        scale = v.abs().amax(-1) / 448.0
        codes = (v / torch.where(scale > 0, scale, torch.ones_like(scale))[..., None]).clamp(-448, 448).to(E4M3)
        cache[0][row] = torch.cat([codes.view(-1, 512).view(torch.uint8), scale.contiguous().view(torch.uint8),
                                   rope.contiguous().view(torch.uint8)], 1)
    elif c["rows"] == "mx":
        cache[0][row], cache[1][row] = _power_scaled(x[:, :512].contiguous(), 32)
        cache[2][row] = rope
    else:
        codes, scale = _power_scaled(x[:, :448].contiguous(), 32)
        cache[0][row] = torch.cat([codes, scale, cache[0][row][:, 462:]], 1)
        cache[1][row] = rope
    if c["index"]:
        k = _rotated(_normed(s["ix"].float(), "layer", D_INDEX, s["iw"], s["ib"]), 0, cs, "halves")
        s["icache"][row] = k.to(torch.bfloat16)


def _latent(cache, rows):
    """Cache rows as 32-bit values [..., 576]."""
    if rows == "bf16":
        return cache.float()
    codes = cache[..., :512].contiguous().view(E4M3).float().unflatten(-1, (4, 128))
    scale = cache[..., 512:528].contiguous().view(torch.float32)
    return torch.cat([(codes * scale[..., None]).flatten(-2),
                      cache[..., 528:].contiguous().view(torch.bfloat16).float()], -1)


def _plain_chunk(s):
    """Every sequence padded to the longest, in one batch."""
    c, B, L, W = s["c"], s["c"]["B"], s["longest"], s["widest"]
    j = torch.arange(L, device="cuda")
    k = _latent(s["cache"][0][s["table"][:, j // PAGE].long() * PAGE + j % PAGE], c["rows"])
    i = torch.arange(W, device="cuda")
    token = (s["indptr"][:-1, None] + torch.minimum(i[None, :], s["new"][:, None] - 1)).long()
    q = s["q"][token].float().view(B, W * c["H"], D_QK)
    p = torch.matmul(q, k.transpose(1, 2).contiguous()).mul_(SM_SCALE).view(B, W, c["H"], L)
    last = (s["lens"] - s["new"])[:, None] + torch.minimum(i[None, :], s["new"][:, None] - 1)
    p.masked_fill_((j[None, None, :] > last[:, :, None])[:, :, None, :], -math.inf)
    top = p.amax(-1, keepdim=True)
    p = p.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, W * c["H"], L), k[..., :D_VO].contiguous()).view(B, W, c["H"], D_VO) / total
    b, pos, _ = _places(s)
    at = (pos - (s["lens"] - s["new"])[b]).long()
    return o[b, at].to(torch.bfloat16), (top + total.log())[b, at].squeeze(-1)


# ------------------------------------------------------------------ one pass

def _views(rows, cache):
    """A cache's tensors by what its bytes stand for."""
    if rows in ("bf16", "v4"):
        return list(cache)
    if rows == "fp8":
        x = cache[0]
        return [x[:, :512].view(E4M3), x[:, 512:528].view(torch.float32), x[:, 528:].view(torch.bfloat16)]
    if rows == "mx":
        return [cache[0].view(E4M3), cache[1].view(E8M0), cache[2]]
    return [cache[0][:, :448].view(E4M3), cache[0][:, 448:462].view(E8M0), cache[1]]


def _own(s):
    from opfoundry_amd import dsa
    c = s["c"]
    if c["kind"] == "prep":
        _, off, n = SHAPES[c["shape"]]
        key = dict(k=s["k"], k_norm=c["kn"], k_weight=s["w"], k_bias=s["b"]) if c["Hk"] else {}
        q, k = dsa.qk_norm_rope(s["q"], s["cs"], s["pos"], q_norm=c["qn"], norm_dim=n, eps=EPS, rot_off=off,
                                style=c["style"], inverse=c["inverse"], **key)
        return [q, k] if c["Hk"] else [q]
    if c["kind"] == "append":
        index = dict(index_k=s["ix"], index_cache=s["icache"], index_norm="layer", index_weight=s["iw"],
                     index_bias=s["ib"], index_style="halves") if c["index"] else {}
        dsa.kv_append(s["x"], s["cache"] if len(s["cache"]) > 1 else s["cache"][0], s["indptr"], s["lens"],
                      s["cs"], block_table=s["table"], block_size=PAGE, weight=s["w"], eps=EPS,
                      style="interleaved", **index)
        return None
    return dsa.mla_chunk(s["q"], s["cache"][0], s["indptr"], s["lens"], SM_SCALE, block_table=s["table"],
                         block_size=PAGE, causal=True, max_kv_len=s["longest"])


def run(state):
    s = state
    if own:
        got = _own(s)
    else:
        got = {"prep": _plain_prep, "append": _plain_append, "chunk": _plain_chunk}[s["c"]["kind"]](s)
    if s["c"]["kind"] == "append":
        return _views(s["c"]["rows"], s["cache"]) + ([s["icache"]] if s["c"]["index"] else [])
    return list(got)


# ------------------------------------------------------------------ the same in 64 bits

def _turn64(x, first, cs, style, sign=1.0):
    """x [n, D] (or [n, H, D]) with its 64 rotated columns as complex numbers times e^(i angle)."""
    z = torch.complex(cs[:, :32], sign * cs[:, 32:])
    if x.dim() == 3:
        z = z[:, None, :]
    r = x[..., first:first + 64]
    pair = r.unflatten(-1, (32, 2)) if style == "interleaved" else torch.stack([r[..., :32], r[..., 32:]], -1)
    t = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * z)
    x = x.clone()
    x[..., first:first + 64] = t.flatten(-2) if style == "interleaved" else torch.cat([t[..., 0], t[..., 1]], -1)
    return x


def _norm64(x, kind, n, w, b):
    if kind == "none":
        return x
    x = x.clone()
    y = x[..., :n]
    mean = y.sum(-1, keepdim=True) / n if kind == "layer" else torch.zeros_like(y[..., :1])
    y = (y - mean) / torch.sqrt(((y - mean) ** 2).sum(-1, keepdim=True) / n + EPS)
    if w is not None:
        y = y * w.double()
    x[..., :n] = y if b is None else y + b.double()
    return x


def _exact_prep(s):
    c = s["c"]
    _, first, n = SHAPES[c["shape"]]
    cs = s["cs"].double()[s["pos"].long()]
    q = _turn64(_norm64(s["q"].double(), c["qn"], n, None, None), first, cs, c["style"], -1.0 if c["inverse"] else 1.0)
    if not c["Hk"]:
        return [q]
    return [q, _turn64(_norm64(s["k"].double(), c["kn"], n, s["w"], s["b"]), first, cs, c["style"])]


def _exact_append(s):
    """The values written, before their rounding to the row's type (codes: value / scale)."""
    c = s["c"]
    new, lens = _chunk_of(c)
    at, pos = [], []
    for b in range(c["B"]):
        p = torch.arange(lens[b] - new[b], lens[b], device="cuda")
        pos.append(p)
        at.append(s["table"][b].long()[p // PAGE] * PAGE + p % PAGE)
    at, cs = torch.cat(at), s["cs"].double()[torch.cat(pos)]
    wide = c["rows"] in ("bf16", "fp8", "mx")
    split = 512 if wide else 448
    x = _turn64(_norm64(s["x"].double(), "rms" if c["norm"] else "none", 512, s["w"], None), split, cs, "interleaved")
    outs = [v.double() for v in _views(c["rows"], s["cache"])]
    if c["rows"] in ("bf16", "v4"):
        outs[0][at] = x
    else:
        v = x[:, :split].reshape(x.shape[0], -1, 128 if c["rows"] == "fp8" else 32)
        scale = v.abs().amax(-1) / 448.0
        if c["rows"] != "fp8":
            scale = torch.exp2(torch.ceil(torch.log2(scale)))
        outs[0][at], outs[1][at], outs[2][at] = (v / scale[..., None]).reshape(-1, split), scale, x[:, split:]
    if c["index"]:
        k = s["icache"].double()
        k[at] = _turn64(_norm64(s["ix"].double(), "layer", D_INDEX, s["iw"], s["ib"]), 0, cs, "halves")
        outs.append(k)
    return outs


def _exact_chunk(s):
    c = s["c"]
    new, lens = _chunk_of(c)
    o = torch.empty((sum(new), c["H"], D_VO), dtype=torch.float64, device="cuda")
    lse = torch.empty((sum(new), c["H"]), dtype=torch.float64, device="cuda")
    first = 0
    for b in range(c["B"]):
        j = torch.arange(lens[b], device="cuda")
        rows = s["cache"][0][s["table"][b].long()[j // PAGE] * PAGE + j % PAGE]
        if c["rows"] == "bf16":
            k = rows.double()
        else:
            scale = rows[:, 512:528].contiguous().view(torch.float32).double().repeat_interleave(128, 1)
            k = torch.cat([rows[:, :512].contiguous().view(E4M3).double() * scale,
                           rows[:, 528:].contiguous().view(torch.bfloat16).double()], 1)
        kt, v = k.t().contiguous(), k[:, :D_VO].contiguous()
        step = max(1, 100_000_000 // (c["H"] * lens[b]))
        for t in range(0, new[b], step):
            m = min(step, new[b] - t)
            x = (s["q"][first + t:first + t + m].double().reshape(m * c["H"], D_QK) @ kt) * SM_SCALE
            limit = lens[b] - new[b] + t + torch.arange(m, device="cuda")
            x = x.view(m, c["H"], lens[b]).masked_fill(j[None, None, :] > limit[:, None, None], -math.inf)
            z = torch.logsumexp(x, 2)
            o[first + t:first + t + m] = (torch.exp(x - z[..., None]).view(m * c["H"], lens[b]) @ v).view(m, c["H"], D_VO)
            lse[first + t:first + t + m] = z
        first += new[b]
    return [o, lse]


def exact(case, seed):
    s = prepare(case, seed)
    return {"prep": _exact_prep, "append": _exact_append, "chunk": _exact_chunk}[s["c"]["kind"]](s)
