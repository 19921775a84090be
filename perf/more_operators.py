"""A latent cache held in 4 bits, and what writes and reads it, as measurable cases.

A row is 400 bytes: 512 e2m1 codes (two a byte, the even value in the low half), 16 power-of-two
scales (one byte each, 2^(byte - 127), for 32 values) and 64 bf16 RoPE values.  Four kinds:

* ``append``  a ragged chunk's latent rows (and index keys) normed, rotated and written into the paged
              cache, then its rows read back: what they hold now
* ``read``    rows of ragged contexts read back as bf16, from the 4-bit cache or one of 656-byte rows
* ``chunk``   dense attention of a chunk's tokens over the paged 4-bit cache
* ``sparse``  attention of every query token over its own list of positions of the 4-bit cache: decode
              (paged, several tokens of a sequence) or prefill (one flat prompt)

With ``own`` false, ``run`` computes them from elementary torch operations in 32 bits; with
``own`` true through ``opfoundry_amd.dsa``.  ``exact`` restates them in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

D_QK, D_VO, D_ROPE, D_INDEX = 576, 512, 64, 128
ROW, ROW8 = 400, 656
SM_SCALE = 1.0 / math.sqrt(192.0)
EPS = 1e-6
PAGE = 64
GOLDEN = 0.6180339887498949
E4M3 = torch.float8_e4m3fn
# e2m1's values in the order of their codes, and what lies half way between two of them
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
POOL = 65536


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # One session's decode step: its token's latent row and index key go into the caches.  Latency.
        dict(name="append_b1", kind="append", B=1, lo=1, hi=1, ctx=1500, index=True, norm=True),
        # Three prompts of one prefill step, uneven lengths.
        dict(name="append_prompts", kind="append", B=3, lo=1200, hi=4500, ctx=777, index=True, norm=True),
        # A short shared prefix read back for one new request.  Latency.
        dict(name="read_b1", kind="read", rows="fp4", B=1, lo=333, hi=333, ctx=0),
        # Ragged contexts read back beside a step of prompt chunks.
        dict(name="read_b9", kind="read", rows="fp4", B=9, lo=1000, hi=20011, ctx=500),
        # The same of a cache of 656-byte rows.
        dict(name="read_fp8_b4", kind="read", rows="fp8", B=4, lo=777, hi=9000, ctx=64),
        # One session's decode step with a context shorter than any top-k: every row is attended.  Latency.
        dict(name="chunk_b1", kind="chunk", B=1, lo=1, hi=1, H=128, ctx=1500, ragged=False),
        # One rank of an 8-way head shard decoding long ragged contexts with up to 3 speculative tokens.
        dict(name="chunk_b16_h16", kind="chunk", B=16, lo=1, hi=4, H=16, ctx=20011, ragged=True),
        # A prefill chunk of 1024 tokens over a long context.
        dict(name="chunk_1024", kind="chunk", B=1, lo=1024, hi=1024, H=128, ctx=8192, ragged=False),
        # A mixed step on an odd head shard: single tokens beside chunks.
        dict(name="chunk_mixed_h40", kind="chunk", B=7, lo=1, hi=301, H=40, ctx=5000, ragged=True),
        # Two sessions' decode step over their selected positions.  Latency.
        dict(name="sparse_b2", kind="sparse", form="decode", T=2, s_q=1, H=128, topk=2048, ctx=8192, ragged=False),
        # A full decode batch with one speculative token each, all heads.
        dict(name="sparse_b128_s2", kind="sparse", form="decode", T=256, s_q=2, H=128, topk=2048, ctx=32768, ragged=True),
        # A prompt's tokens on one rank of an 8-way head shard.
        dict(name="sparse_prefill_h16", kind="sparse", form="prefill", T=1531, s_q=1, H=16, topk=2048, ctx=3000, ragged=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    kind = rng.choice(["append", "read", "chunk", "chunk", "sparse", "sparse"])
    if kind == "append":
        B = _log(rng, 1, 128)
        hi = _log(rng, 1, 9000 // B)
        return dict(kind=kind, B=B, lo=rng.randint(1, hi), hi=hi, ctx=_log(rng, 1, 40000 // B),
                    index=rng.random() < 0.6, norm=rng.random() < 0.8)
    if kind == "read":
        B = _log(rng, 1, 64)
        hi = _log(rng, 1, 90000 // B)
        return dict(kind=kind, rows=rng.choice(["fp4", "fp4", "fp8"]), B=B, lo=rng.randint(1, hi), hi=hi,
                    ctx=rng.choice([0, _log(rng, 1, 4000)]))
    H = rng.choice([16, 16, 32, 40, 64, 96, 128, 128])
    if kind == "chunk":
        B = _log(rng, 1, 64)
        if rng.random() < 0.5:                                  # decode: a few tokens each over long contexts
            hi, ctx = rng.randint(1, 4), _log(rng, 200, 1_000_000 // B)
        else:                                                   # chunks
            B = min(B, 8)
            hi, ctx = _log(rng, 5, 2048), _log(rng, 1, 16000)
        c = dict(kind=kind, B=B, lo=rng.randint(1, hi), hi=hi, H=H, ctx=ctx, ragged=rng.random() < 0.7)
        while work(c)["flops"] > 2.4e12 or B * c["hi"] * H * (ctx + c["hi"]) > 1.2e9:
            c["hi"] = max(1, c["hi"] * 2 // 3)
            c["ctx"] = ctx = max(1, ctx * 4 // 5)
            c["lo"] = min(c["lo"], c["hi"])
        return c
    form, s_q = rng.choice(["decode", "decode", "prefill"]), rng.randint(1, 4)
    topk = rng.choice([512, 1024, 2048, 2048, _log(rng, 1, 2500)])
    T = max(s_q, _log(rng, 1, min(2048, 640000 * 128 // (H * topk), 1_100_000 // topk)) // s_q * s_q)
    return dict(kind=kind, form=form, T=T, s_q=s_q if form == "decode" else 1, H=H, topk=topk,
                ctx=_log(rng, 300, 40000 if form == "decode" else 20000), ragged=form == "decode" and rng.random() < 0.7)


# ------------------------------------------------------------------ sizes that follow from a case

def _spread(count, lo, hi):
    """`count` whole numbers spread unevenly over [lo, hi]: the same ones for every seed."""
    return [lo + int((hi - lo + 1) * (((i + 1) * GOLDEN) % 1.0)) for i in range(count)]


def _chunk_of(c):
    """New tokens (or rows to read) of each sequence, and its length with them."""
    new = _spread(c["B"], c["lo"], c["hi"])
    ctx = _spread(c["B"], c["ctx"] // 3, c["ctx"]) if c.get("ragged", True) else [c["ctx"]] * c["B"]
    return new, [n + x for n, x in zip(new, ctx)]


def _lists_of(c):
    """A decode's sequence lengths (their tokens included); how many positions each query token attends."""
    if c["form"] == "prefill":
        lens = [c["ctx"] + c["T"]]
        sees = [c["ctx"] + i + 1 for i in range(c["T"])]
    else:
        n = c["T"] // c["s_q"]
        ctx = _spread(n, c["ctx"] // 3, c["ctx"]) if c["ragged"] else [c["ctx"]] * n
        lens = [x + c["s_q"] for x in ctx]
        sees = [x + t + 1 for x in ctx for t in range(c["s_q"])]
    return lens, sees


def work(case):
    c = case
    if c["kind"] == "sparse":
        lens, sees = _lists_of(c)
        pairs = sum(min(c["topk"], n) for n in sees)
        # a row that several tokens of a prompt or a sequence attend counts once
        rows = min(pairs, sum(lens))
        return {"bytes": rows * ROW + c["T"] * (4 * c["topk"] + c["H"] * (2 * D_QK + 2 * D_VO + 4)),
                "flops": 2 * c["H"] * (D_QK + D_VO) * pairs}
    new, lens = _chunk_of(c)
    T = sum(new)
    if c["kind"] == "append":
        per = 2 * D_QK + ROW + 4 * D_ROPE + (4 * D_INDEX if c["index"] else 0) + ROW + 2 * D_QK
        return {"bytes": T * per + 8 * c["B"], "flops": 10 * T * D_QK}
    if c["kind"] == "read":
        return {"bytes": T * ((ROW if c["rows"] == "fp4" else ROW8) + 2 * D_QK) + 8 * c["B"], "flops": T * D_VO}
    pairs = sum(n * s - n * (n - 1) // 2 for n, s in zip(new, lens))
    return {"bytes": sum(lens) * ROW + T * c["H"] * (2 * D_QK + 2 * D_VO + 4),
            "flops": 2 * c["H"] * (D_QK + D_VO) * pairs}


# ------------------------------------------------------------------ the 4-bit format

def _e2m1(v):
    """The codes (0 .. 15) of v: nearest value, ties to the even code, at most 6."""
    a = v.abs()
    n = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    return n + 8 * (v < 0).to(torch.uint8)


def _pack(x):
    """x [n, 512] (32 bits) as codes [n, 256] and scale bytes [n, 16]: of 32 values the least power of two
    with every |value| / 2^e at most 6."""
    v = x.view(x.shape[0], 16, 32)
    top = v.abs().amax(-1)
    m, e = torch.frexp(top / 6.0)
    e = torch.where(m == 0.5, e - 1, e).clamp(min=-125)
    e = torch.where(top > 0, e, torch.zeros_like(e))
    code = _e2m1(torch.ldexp(v, -e[..., None])).view(x.shape[0], 256, 2)
    return code[..., 0] | (code[..., 1] << 4), (e + 127).to(torch.uint8)


def _grid(dtype):
    return torch.tensor(GRID + tuple(-x for x in GRID), dtype=dtype, device="cuda")


def _unpack(rows, dtype=torch.float32):
    """4-bit rows [..., 400] as values [..., 576]."""
    b = rows[..., :256]
    code = torch.stack([b & 15, b >> 4], -1).unflatten(-2, (16, 16)).flatten(-2)          # [..., 16, 32]
    scale = torch.ldexp(torch.ones((), dtype=dtype, device="cuda"), rows[..., 256:272].int() - 127)
    nope = (_grid(dtype)[code.int()] * scale[..., None]).flatten(-2)
    return torch.cat([nope, rows[..., 272:].contiguous().view(torch.bfloat16).to(dtype)], -1)


def _unpack8(rows, dtype=torch.float32):
    """656-byte rows [..., 656] as values [..., 576]."""
    codes = rows[..., :512].contiguous().view(E4M3).to(dtype).unflatten(-1, (4, 128))
    scale = rows[..., 512:528].contiguous().view(torch.float32).to(dtype)
    return torch.cat([(codes * scale[..., None]).flatten(-2), rows[..., 528:].contiguous().view(torch.bfloat16).to(dtype)], -1)


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


def _cache(g, rows, n):
    """n cache rows in use (of a large cache, rows drawn from as many as POOL)."""
    m = min(n, POOL)
    if rows == "fp8":
        out = torch.empty((m, ROW8), dtype=torch.uint8, device="cuda")
        out[:, :512] = (_randn(g, m, 512) * 100).clamp(-448, 448).to(E4M3).view(torch.uint8)
        out[:, 512:528] = (0.008 + 0.004 * torch.rand((m, 4), generator=g, device="cuda")).view(torch.uint8)
        out[:, 528:] = _bf16(g, m, D_ROPE).view(torch.uint8)
    else:
        out = torch.cat([*_pack(_randn(g, m, 512)), _bf16(g, m, D_ROPE).view(torch.uint8)], 1)
    return out if n <= m else out[torch.randint(0, m, (n,), generator=g, device="cuda")]


def _pages(g, s, sequences, longest):
    blocks = -(-longest // PAGE)
    s["table"] = torch.randperm(sequences * blocks, generator=g, device="cuda").to(torch.int32).view(sequences, blocks)
    return sequences * blocks * PAGE


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    if c["kind"] == "sparse":
        lens, sees = _lists_of(c)
        s = dict(c=c, lens=_int32(lens))
        n = lens[0] if c["form"] == "prefill" else _pages(g, s, len(lens), max(lens))
        s["cache"] = _cache(g, "fp4", n)
        s["q"] = _bf16(g, c["T"], c["H"], D_QK)
        # topk different positions of those that a token sees, ascending; all of them and -1 where it sees fewer
        k, see = torch.arange(c["topk"], device="cuda"), torch.tensor(sees, device="cuda", dtype=torch.float64)[:, None]
        u = torch.rand((c["T"], c["topk"]), generator=g, device="cuda", dtype=torch.float64)
        spread = torch.minimum(((k + u) * (see / c["topk"])).floor(), see - 1)
        s["indices"] = torch.where(see > c["topk"], spread, torch.where(k < see, k.double(), -1.0)).to(torch.int32)
        return s
    new, lens = _chunk_of(c)
    s = dict(c=c, new=_int32(new), lens=_int32(lens), longest=max(lens), widest=max(new), T=sum(new),
             indptr=_int32([0] + torch.tensor(new).cumsum(0).tolist()))
    n = _pages(g, s, c["B"], max(lens))
    s["cache"] = _cache(g, c.get("rows", "fp4"), n)
    if c["kind"] == "chunk":
        s["q"] = _bf16(g, s["T"], c["H"], D_QK)
    if c["kind"] == "append":
        s["x"] = _bf16(g, s["T"], D_QK)
        s["w"] = 1.0 + 0.1 * _randn(g, 512) if c["norm"] else None
        s["cs"] = _angles(max(lens))
        if c["index"]:
            s["ix"], s["icache"] = _bf16(g, s["T"], D_INDEX), _bf16(g, n, D_INDEX)
            s["iw"], s["ib"] = 1.0 + 0.1 * _randn(g, D_INDEX), 0.1 * _randn(g, D_INDEX)
    return s


# ------------------------------------------------------------------ the plain forms (32 bits)

def _normed(x, kind, w, b):
    y = x
    if kind == "layer":
        y = y - y.mean(-1, keepdim=True)
    if kind != "none":
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS)
    if w is not None:
        y = y * w
    return y if b is None else y + b


def _rotated(r, cs, style):
    """The 64 columns r turned by the angles cs [n, 64]."""
    cos, sin = cs[:, :32], cs[:, 32:]
    if style == "interleaved":
        u, v = r[:, 0::2], r[:, 1::2]
        return torch.stack([u * cos - v * sin, v * cos + u * sin], -1).flatten(-2)
    u, v = r[:, :32], r[:, 32:]
    return torch.cat([u * cos - v * sin, v * cos + u * sin], -1)


def _places(s):
    """Sequence, position and cache row of every token of the chunk."""
    t = torch.arange(s["T"], device="cuda")
    b = (t[:, None] >= s["indptr"][None, 1:]).sum(1)
    pos = (s["lens"] - s["new"])[b] + t - s["indptr"][b]
    return b, pos, s["table"][b, pos // PAGE].long() * PAGE + pos % PAGE


def _plain_append(s):
    c = s["c"]
    _, pos, row = _places(s)
    cs = s["cs"][pos]
    x = s["x"].float()
    codes, scale = _pack(_normed(x[:, :512], "rms" if c["norm"] else "none", s["w"], None).contiguous())
    rope = _rotated(x[:, 512:], cs, "interleaved").to(torch.bfloat16)
    s["cache"][row] = torch.cat([codes, scale, rope.contiguous().view(torch.uint8)], 1)
    out = [_unpack(s["cache"][row]).to(torch.bfloat16)]
    if c["index"]:
        k = _normed(s["ix"].float(), "layer", s["iw"], s["ib"])
        k = torch.cat([_rotated(k[:, :64], cs, "halves"), k[:, 64:]], 1)
        s["icache"][row] = k.to(torch.bfloat16)
        out.append(s["icache"])
    return out


def _plain_read(s):
    rows = s["cache"][_places(s)[2]]
    return [(_unpack(rows) if s["c"]["rows"] == "fp4" else _unpack8(rows)).to(torch.bfloat16)]


def _attend(q, k, on):
    """q [n, m, 576] over k [n, L, 576] where on [n, m or 1, L]: outputs and log-sum-exps."""
    p = torch.matmul(q, k.transpose(1, 2).contiguous()).mul_(SM_SCALE)
    p.masked_fill_(~on, -math.inf)
    top = p.amax(-1, keepdim=True)
    p = p.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p, k[..., :D_VO].contiguous()) / total, top + total.log()


def _plain_chunk(s):
    """Every sequence padded to the longest, in one batch."""
    c, B, L, W = s["c"], s["c"]["B"], s["longest"], s["widest"]
    j = torch.arange(L, device="cuda")
    k = _unpack(s["cache"][s["table"][:, j // PAGE].long() * PAGE + j % PAGE])
    i = torch.minimum(torch.arange(W, device="cuda")[None, :], s["new"][:, None] - 1)
    q = s["q"][(s["indptr"][:-1, None] + i).long()].float().view(B, W * c["H"], D_QK)
    last = ((s["lens"] - s["new"])[:, None] + i).repeat_interleave(c["H"], 1)
    o, z = _attend(q, k, j[None, None, :] <= last[:, :, None])
    b, pos, _ = _places(s)
    at = (pos - (s["lens"] - s["new"])[b]).long()
    return [o.view(B, W, c["H"], D_VO)[b, at].to(torch.bfloat16), z.view(B, W, c["H"])[b, at]]


def _plain_sparse(s):
    c, T, H = s["c"], s["c"]["T"], s["c"]["H"]
    on, j = s["indices"] >= 0, s["indices"].clamp(min=0).long()
    if c["form"] == "decode":
        b = torch.arange(T, device="cuda")[:, None] // c["s_q"]
        j = s["table"][b, j // PAGE].long() * PAGE + j % PAGE
    o, z = _attend(s["q"].float(), _unpack(s["cache"][j]), on[:, None, :])
    lead = (T // c["s_q"], c["s_q"]) if c["form"] == "decode" else (T,)
    return [o.to(torch.bfloat16).view(*lead, H, D_VO), z.view(*lead, H)]


# ------------------------------------------------------------------ one pass

def _own(s):
    from opfoundry_amd import dsa
    c = s["c"]
    if c["kind"] == "sparse":
        if c["form"] == "prefill":
            return dsa.mla_prefill(s["q"], s["cache"], s["indices"], SM_SCALE, causal=True, causal_offset=c["ctx"])
        lead = (c["T"] // c["s_q"], c["s_q"])
        return dsa.mla_decode(s["q"].view(*lead, c["H"], D_QK), s["cache"], s["indices"].view(*lead, -1), SM_SCALE,
                              seq_lens=s["lens"], block_table=s["table"], block_size=PAGE, causal=True)
    paged = dict(block_table=s["table"], block_size=PAGE)
    if c["kind"] == "chunk":
        return dsa.mla_chunk(s["q"], s["cache"], s["indptr"], s["lens"], SM_SCALE, causal=True, max_kv_len=s["longest"], **paged)
    if c["kind"] == "append":
        index = dict(index_k=s["ix"], index_cache=s["icache"], index_norm="layer", index_weight=s["iw"],
                     index_bias=s["ib"], index_style="halves") if c["index"] else {}
        dsa.kv_append(s["x"], s["cache"], s["indptr"], s["lens"], s["cs"], weight=s["w"], eps=EPS, style="interleaved",
                      **paged, **index)
    rows = dsa.kv_read(s["cache"], s["indptr"], s["lens"], s["T"], **paged)
    return [rows, s["icache"]] if c.get("index") else [rows]


def run(state):
    if own:
        return list(_own(state))
    return {"append": _plain_append, "read": _plain_read, "chunk": _plain_chunk,
            "sparse": _plain_sparse}[state["c"]["kind"]](state)


# ------------------------------------------------------------------ the same in 64 bits

def _turn64(r, cs, style):
    """The 64 columns r as 32 complex numbers times e^(i angle)."""
    pair = r.unflatten(-1, (32, 2)) if style == "interleaved" else torch.stack([r[:, :32], r[:, 32:]], -1)
    t = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * torch.complex(cs[:, :32], cs[:, 32:]))
    return t.flatten(-2) if style == "interleaved" else torch.cat([t[..., 0], t[..., 1]], -1)


def _norm64(x, centred, w, b):
    y = x - x.sum(-1, keepdim=True) / x.shape[-1] if centred else x
    y = y / torch.sqrt((y ** 2).sum(-1, keepdim=True) / x.shape[-1] + EPS)
    if w is not None:
        y = y * w.double()
    return y if b is None else y + b.double()


def _values64(rows):
    """4-bit rows' values: sign, exponent and mantissa of each code, and its scale."""
    code = torch.stack([rows[:, :256] & 15, rows[:, :256] >> 4], -1).view(-1, 512).long()
    e, m = (code >> 1) & 3, (code & 1).double()
    size = torch.where(e > 0, torch.exp2(e.double() - 1) * (1 + m / 2), m / 2)
    scale = torch.exp2(rows[:, 256:272].double() - 127).repeat_interleave(32, 1)
    rope = rows[:, 272:].contiguous().view(torch.bfloat16).double()
    return torch.cat([torch.where(code >= 8, -size, size) * scale, rope], 1)


def _rows_of(c, s):
    """The cache row and position of every token of the chunk."""
    new, lens = _chunk_of(c)
    at, pos = [], []
    for b in range(c["B"]):
        p = torch.arange(lens[b] - new[b], lens[b], device="cuda")
        pos.append(p)
        at.append(s["table"][b].long()[p // PAGE] * PAGE + p % PAGE)
    return torch.cat(at), torch.cat(pos)


def _held64(x):
    """What a 4-bit row holds for x [n, 512]: steps of 1/2 below 2, of 1 below 4 and of 2 up to 6, times
    the group's power of two."""
    v = x.view(-1, 16, 32)
    top = v.abs().amax(-1, keepdim=True)
    scale = torch.exp2(torch.ceil(torch.log2(torch.where(top > 0, top, 1.0) / 6)).clamp(min=-125))
    a = v.abs() / scale
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    return (torch.copysign((torch.round(a / step) * step).clamp(max=6), v) * scale).view(-1, 512)


def _exact_append(s):
    """The values written: NoPE as the row's codes hold them, the others before their rounding."""
    c = s["c"]
    at, pos = _rows_of(c, s)
    cs, x = s["cs"].double()[pos], s["x"].double()
    nope = _norm64(x[:, :512], False, s["w"], None) if c["norm"] else x[:, :512]
    out = [torch.cat([_held64(nope.contiguous()), _turn64(x[:, 512:], cs, "interleaved")], 1)]
    if c["index"]:
        k = _norm64(s["ix"].double(), True, s["iw"], s["ib"])
        whole = s["icache"].double()
        whole[at] = torch.cat([_turn64(k[:, :64], cs, "halves"), k[:, 64:]], 1)
        out.append(whole)
    return out


def _exact_read(s):
    rows = s["cache"][_rows_of(s["c"], s)[0]]
    return [_values64(rows) if s["c"]["rows"] == "fp4" else _unpack8(rows, torch.float64)]


def _one64(q, k, on):
    """q [m, 576] over k [L, 576] where on [m, L]."""
    x = ((q @ k.t().contiguous()) * SM_SCALE).masked_fill(~on, -math.inf)
    z = torch.logsumexp(x, 1)
    return torch.exp(x - z[:, None]) @ k[:, :D_VO].contiguous(), z


def _exact_chunk(s):
    c = s["c"]
    new, lens = _chunk_of(c)
    o = torch.empty((sum(new), c["H"], D_VO), dtype=torch.float64, device="cuda")
    lse = torch.empty((sum(new), c["H"]), dtype=torch.float64, device="cuda")
    first = 0
    for b in range(c["B"]):
        j = torch.arange(lens[b], device="cuda")
        k = _values64(s["cache"][s["table"][b].long()[j // PAGE] * PAGE + j % PAGE])
        step = max(1, 100_000_000 // (c["H"] * lens[b]))
        for t in range(0, new[b], step):
            m = min(step, new[b] - t)
            last = (lens[b] - new[b] + t + torch.arange(m, device="cuda")).repeat_interleave(c["H"])
            x, z = _one64(s["q"][first + t:first + t + m].double().view(m * c["H"], D_QK), k, j[None, :] <= last[:, None])
            o[first + t:first + t + m], lse[first + t:first + t + m] = x.view(m, c["H"], D_VO), z.view(m, c["H"])
        first += new[b]
    return [o, lse]


def _exact_sparse(s):
    c = s["c"]
    o = torch.empty((c["T"], c["H"], D_VO), dtype=torch.float64, device="cuda")
    lse = torch.empty((c["T"], c["H"]), dtype=torch.float64, device="cuda")
    for t in range(c["T"]):
        j = s["indices"][t]
        j = j[j >= 0].long()
        if c["form"] == "decode":
            j = s["table"][t // c["s_q"]].long()[j // PAGE] * PAGE + j % PAGE
        k = _values64(s["cache"][j])
        o[t], lse[t] = _one64(s["q"][t].double(), k, torch.ones((1, len(j)), dtype=torch.bool, device="cuda"))
    lead = (c["T"] // c["s_q"], c["s_q"]) if c["form"] == "decode" else (c["T"],)
    return [o.view(*lead, c["H"], D_VO), lse.view(*lead, c["H"])]


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "read": _exact_read, "chunk": _exact_chunk,
            "sparse": _exact_sparse}[s["c"]["kind"]](s)
