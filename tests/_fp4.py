"""Inputs and 64-bit references of the tests of 400-byte rows (DSA_KV_MXFP4, include/dsa_mla.h).

A row's values are exact in bf16, so the bf16 rows of the same values are what tests/_chunk.py's references
take.  Nothing here is of the library's: codes are chosen from the table of values by distance."""
from __future__ import annotations

import math
from types import SimpleNamespace

import torch

from _chunk import SM_SCALE, bf16, check_chunk

GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def nearest(a):
    """Codes 0 .. 7 of a >= 0 (float64): the nearest value, of two equally near the even code."""
    d = (a[..., None] - torch.tensor(GRID, dtype=torch.float64, device=a.device)).abs()
    best = d.amin(-1, keepdim=True)
    code = torch.arange(8, device=a.device).expand(d.shape)
    # (an odd code only where it alone is nearest)
    return torch.where(d == best, code + 8 * (code % 2), 99).amin(-1) % 8


def exponent(amax):
    """e of the least power of two 2^e >= amax / 6 (float64), at least -125; 0 for 0."""
    e = torch.full(amax.shape, -125, dtype=torch.int64, device=amax.device)
    for k in range(-125, 128):
        e = torch.where(6.0 * 2.0 ** k < amax, k + 1, e)
    return torch.where(amax == 0, 0, e)


def pack(x):
    """x float64 [n, 512] as code bytes [n, 256] and scale bytes [n, 16]."""
    v = x.view(-1, 16, 32)
    bad = ~torch.isfinite(v).all(-1)
    v = torch.where(bad[..., None], 0.0, v)
    e = exponent(v.abs().amax(-1))
    scaled = v / torch.exp2(e.double())[..., None]
    limit = torch.where(e >= 126, 5, 7)[..., None]
    code = torch.minimum(nearest(scaled.abs()), limit) + 8 * torch.signbit(v).long()
    code = torch.where(bad[..., None], 0, code).view(-1, 256, 2)
    return (code[..., 0] + 16 * code[..., 1]).to(torch.uint8), torch.where(bad, 255, e + 127).to(torch.uint8)


def rows(g, n, spread=True):
    """Rows of N(0, 1) values, groups spread over 2^-2 .. 2^2 of that."""
    x = torch.randn((n, 16, 32), generator=g, device=g.device)
    if spread:
        x = x * torch.exp2(torch.randint(-2, 3, (n, 16, 1), generator=g, device=g.device).float())
    # (any values: the codes need not be the nearest ones)
    e = torch.ceil(torch.log2(x.abs().amax(-1) / 6))
    a = (x / torch.exp2(e)[..., None]).abs()
    code = torch.bucketize(a, torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=g.device))
    code = (code + 8 * (x < 0)).view(n, 256, 2)
    return torch.cat([(code[..., 0] + 16 * code[..., 1]).to(torch.uint8), (e + 127).to(torch.uint8),
                      bf16(g, n, 64).view(torch.uint8)], 1)


def values(r):
    """Rows [..., 400] as float64 [..., 576]."""
    b = r[..., :256].long()
    grid = torch.tensor(GRID + tuple(-x for x in GRID), dtype=torch.float64, device=r.device)
    nope = grid[torch.stack([b % 16, b // 16], -1).flatten(-2)]
    s = r[..., 256:272].long()
    scale = torch.where(s == 255, math.nan, torch.exp2(s.double() - 127)).repeat_interleave(32, -1)
    return torch.cat([nope * scale, r[..., 272:].contiguous().view(torch.bfloat16).double()], -1)


def as_bf16(r):
    return values(r).to(torch.bfloat16)


def attend_lists64(q, kv, lists, H, sm_scale=SM_SCALE):
    """(c, reference) for _chunk.check_chunk of tokens q [T, H, 576] that attend cache rows lists[t] (ints) of bf16
    rows kv; duplicates count each time."""
    T = q.shape[0]
    dev = q.device
    z = dict(dtype=torch.float64, device=dev)
    o, A, N = torch.zeros((T, H, 512), **z), torch.zeros((T, H, 512), **z), torch.zeros((T, H, 512), **z)
    lse, E = torch.full((T, H), math.inf, **z), torch.zeros((T, H), **z)
    for t in range(T):
        at = torch.as_tensor(lists[t], dtype=torch.long, device=dev)
        if not len(at):
            continue
        k = kv[at].double()
        x = q[t].double()
        s = (x @ k.t().contiguous()) * sm_scale
        lse[t] = torch.logsumexp(s, 1)
        p = torch.exp(s - lse[t][:, None])
        v = k[:, :512].contiguous()
        o[t], A[t], N[t] = p @ v, p @ v.abs(), v.abs().sum(0)
        E[t] = 2 * 64 * 2.0 ** -24 * (x.abs() @ k.abs().t().contiguous()).amax(1) * abs(sm_scale)
    return SimpleNamespace(T=T, first=0, new=[T]), (o, lse, A, E, N)


def check(c, out, lse, ref, what=""):
    """_chunk.check_chunk with the probabilities that P cannot hold.  P is bf16, whose values end at 2^-126, and
    stands for 2^-15 (or, of n positions that start again, 2^(-1 - ceil(log2 n))) where a row's probability is
    largest: a probability below 2^-126 / 2^-25 = 2^-101 of the largest, n up to 2^24, may count as 0.  O is then off by
    at most 2^-101 of the sum N of |V|, which is far below 2^-8 of A = sum p |V| wherever the likely rows' V is not 0;
    here it is 0 for one code in eight.  (A + 2^-90 N, of which the bound takes over 2^-8: 2^-98 N.)"""
    o, l, A, E, N = ref
    check_chunk(c, out, lse, (o, l, A + 2.0 ** -90 * N, E, N), False, what)
