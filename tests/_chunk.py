"""Inputs and 64-bit references of the chunk operators' tests (include/dsa_chunk.h).

Everything here is float64 torch from the operators' definitions; where a bound is
given, it counts the roundings that the definition allows:
  a value rounded to bf16 is off by at most 2^-8 of itself (half a step), to fp16 2^-11,
  to e4m3 2^-4 (2^-10 absolute below 2^-6), in fp32 2^-24 a step.
"""
from __future__ import annotations

import math

import torch

SM_SCALE = 1.0 / math.sqrt(192.0)
E4M3 = torch.float8_e4m3fn


def gen(seed, dev):
    return torch.Generator(device=dev).manual_seed(seed)


def bf16(g, *shape, scale=1.0):
    return (torch.randn(shape, generator=g, device=g.device) * scale).to(torch.bfloat16)


def i32(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def cos_sin(n, dev):
    at = torch.arange(n, device=dev, dtype=torch.float64)
    f = 10000.0 ** (-torch.arange(32, device=dev, dtype=torch.float64) / 32)
    a = at[:, None] * f
    return torch.cat([a.cos(), a.sin()], 1).float()


class Chunk:
    """new[b] tokens of sequence b, lens[b] long with them, over shuffled pages (block_size None: flat
    caches of `flat` rows a sequence).  first: rows before the first sequence's tokens; pad: behind the last's."""

    def __init__(self, g, new, lens, block_size=64, flat=0, first=0, pad=0, spare=0):
        dev = g.device
        self.new, self.lens, self.bs, self.flat = new, lens, block_size, flat
        self.B, self.first = len(new), first
        ends = [first]
        for n in new:
            ends.append(ends[-1] + n)
        self.T = ends[-1] + pad
        self.indptr, self.seq_lens = i32(ends, dev), i32(lens, dev)
        if block_size:
            self.blocks = max(1, -(-max(list(lens) + [1]) // block_size))
            self.rows = (self.B * self.blocks + spare) * block_size
            perm = torch.randperm(self.B * self.blocks + spare, generator=g, device=dev)[:self.B * self.blocks]
            self.table = perm.to(torch.int32).view(self.B, self.blocks)
            self.kw = dict(block_table=self.table, block_size=block_size)
        else:
            self.rows, self.table = self.B * flat, None
            self.kw = dict(kv_batch_stride=flat)

    def tokens(self):
        """(token, sequence, position) of every token that has one."""
        t = self.first
        for b, n in enumerate(self.new):
            for i in range(n):
                yield t, b, self.lens[b] - n + i
                t += 1

    def row(self, b, p):
        """Cache row of position p of sequence b, or -1."""
        if p < 0:
            return -1
        if self.table is None:
            r = b * self.flat + p if not self.flat or p < self.flat else -1
        else:
            if p >= self.blocks * self.bs:
                return -1
            r = int(self.table_cpu()[b, p // self.bs]) * self.bs + p % self.bs
        return r if 0 <= r < self.rows else -1

    def table_cpu(self):
        if not hasattr(self, "_t"):
            self._t = self.table.cpu()
        return self._t


def norm64(x, kind, n, eps, w=None, b=None):
    x = x.double().clone()
    if kind == "none":
        return x
    y = x[..., :n]
    if kind == "layer":
        y = y - y.mean(-1, keepdim=True)
    y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps)
    if w is not None:
        y = y * w.double()
    if b is not None:
        y = y + b.double()
    x[..., :n] = y
    return x


def rope64(x, off, cs, style, inverse=False):
    """cs [..., 64] broadcasts over x's rows."""
    x = x.clone()
    if style is None:
        return x
    r = x[..., off:off + 64].clone()
    c, s = cs[..., :32].double(), cs[..., 32:].double()
    s = -s if inverse else s
    ia = torch.arange(0, 64, 2) if style == "interleaved" else torch.arange(32)
    ib = ia + 1 if style == "interleaved" else ia + 32
    a, b = r[..., ia], r[..., ib]
    x[..., off + ia] = a * c - b * s
    x[..., off + ib] = b * c + a * s
    return x


def near_bf16(got, want, slack):
    """got (bf16) is want rounded once, after fp32 work whose own error is at most `slack` (absolute)."""
    got, want = got.double(), want.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    fin = ~torch.isnan(want)
    over = (got - want).abs()[fin] - (2.0 ** -8 * want.abs()[fin] + slack)
    assert over.numel() == 0 or float(over.max()) <= 0, float(over.max())


def fp8_rows(g, n, spread=True):
    """656-byte rows: codes of N(0, 100^2), scales around 0.01 (spread over 2^-6 .. 2^6 of it)."""
    dev = g.device
    out = torch.empty((n, 656), dtype=torch.uint8, device=dev)
    out[:, :512] = (torch.randn((n, 512), generator=g, device=dev) * 100).clamp(-448, 448).to(E4M3).view(torch.uint8)
    sc = 0.005 + 0.01 * torch.rand((n, 4), generator=g, device=dev)
    if spread:
        sc = sc * torch.exp2(torch.randint(-2, 3, (n, 4), generator=g, device=dev).float())
    out[:, 512:528] = sc.contiguous().view(torch.uint8)
    out[:, 528:] = bf16(g, n, 64).view(torch.uint8)
    return out


def latent64(rows):
    if rows.dtype == torch.bfloat16:
        return rows.double()
    sc = rows[:, 512:528].contiguous().view(torch.float32).double().repeat_interleave(128, 1)
    return torch.cat([rows[:, :512].contiguous().view(E4M3).double() * sc,
                      rows[:, 528:].contiguous().view(torch.bfloat16).double()], 1)


def attend64(c: Chunk, q, kv, causal, sm_scale=SM_SCALE, max_len=None):
    """(O, LSE, A, E, N) in float64: A = sum p |v| / sum p, E the bound of a score's fp32 error times 2
    (relative error of a probability): 64 additions of 2^-24 of sum |q k|, each row's largest; N = sum |v|."""
    T, H, _ = q.shape
    dev = q.device
    o = torch.full((T, H, 512), float("nan"), dtype=torch.float64, device=dev)
    N = torch.zeros_like(o)
    A, lse, E = torch.zeros_like(o), torch.full((T, H), float("nan"), dtype=torch.float64, device=dev), \
        torch.zeros((T, H), dtype=torch.float64, device=dev)
    first = c.first
    for b, n in enumerate(c.new):
        L = c.lens[b]
        rows = torch.tensor([c.row(b, j) for j in range(L)], dtype=torch.long, device=dev)
        keep = torch.nonzero(rows >= 0).flatten()
        k = latent64(kv[rows[keep]]) if len(keep) else torch.zeros((0, 576), dtype=torch.float64, device=dev)
        kt, v, va = k.t().contiguous(), k[:, :512].contiguous(), k[:, :512].abs().contiguous()
        step = max(1, 60_000_000 // max(1, H * L))
        for i in range(0, n, step):
            m = min(step, n - i)
            at = slice(first + i, first + i + m)
            if max_len is not None and L > max_len:
                continue
            x = q[at].double().reshape(m * H, 576)
            limit = (L - n + i + torch.arange(m, device=dev)) if causal else torch.full((m,), L - 1, device=dev)
            on = (keep[None, :] <= limit[:, None])[:, None, :]
            s = ((x @ kt) * sm_scale).view(m, H, -1)
            # (what a row that is not attended holds counts for nothing)
            s = torch.where(on, s, -math.inf)
            none = ~on.any(2).expand(m, H)
            z = torch.where(none, math.inf, torch.logsumexp(s, 2)) if len(keep) else torch.full_like(E[at], math.inf)
            p = torch.where(on, torch.exp(s - torch.where(none, 0.0, z)[..., None]), 0.0).view(m * H, -1)
            fv = torch.where(torch.isfinite(v), v, 0.0)      # (NaN reaches O by p, which then is NaN)
            o[at], A[at] = (p @ fv).view(m, H, 512), (p @ torch.where(torch.isfinite(va), va, 0.0)).view(m, H, 512)
            lse[at] = z
            N[at] = torch.where(torch.isfinite(va), va, 0.0).sum(0)
            if len(keep):
                big = ((x.abs() @ torch.where(torch.isfinite(kt), kt.abs(), 0.0)).view(m, H, -1) * on).amax(2)
                E[at] = 2 * 64 * 2.0 ** -24 * big * abs(sm_scale)
        first += n
    return o, lse, A, E, N


def check_chunk(c: Chunk, out, lse, ref, fp8, what=""):
    """Bound of O: P rounded (2^-8; fp16 2^-11), V rounded to fp16 (656-byte rows: the scale's mantissa and
    its product with the code, 2^-11 each, and 2^-25 below fp16's normal range), the output rounded
    (2^-8 |O|), fp32 sums of up to 2^6 partial sums a split, the scores' error E.  LSE: E and 2^-20 of itself and 1."""
    o, l, A, E, N = ref
    own = torch.zeros(c.T, dtype=torch.bool, device=out.device)
    own[c.first:c.first + sum(c.new)] = True
    g, gl = out.double(), lse.double()
    g, gl, o, l, A, E, N = g[own], gl[own], o[own], l[own], A[own], E[own], N[own]
    assert torch.equal(torch.isnan(g), torch.isnan(o)), f"{what}: NaN where none is due, or none where one is"
    assert torch.equal(torch.isnan(gl), torch.isnan(l)) and torch.equal(torch.isinf(gl), torch.isinf(l)), what
    rel = (3 * 2.0 ** -11 if fp8 else 2.0 ** -8) + 2.0 ** -17
    bound = (rel + E[..., None]) * A + 2.0 ** -8 * o.abs() + (2.0 ** -24 * (1 + N) if fp8 else 0.0)
    fin = torch.isfinite(o)
    over = ((g - o).abs() / bound.clamp(min=1e-300))[fin & (bound > 0)]
    assert over.numel() == 0 or float(over.max()) <= 1, f"{what}: O off by {float(over.max())} of its bound"
    zero = fin & (bound == 0)
    assert bool((g[zero] == 0).all()), what
    fl = torch.isfinite(l)
    lb = E + 2.0 ** -20 * (1 + l.abs())
    worst = ((gl - l).abs() / lb)[fl]
    assert worst.numel() == 0 or float(worst.max()) <= 1, f"{what}: LSE off by {float(worst.max())} of its bound"
