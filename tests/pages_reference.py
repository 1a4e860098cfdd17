"""A key/value cache in pages in 64 bits on the host, from its definitions: what the tests of the ops over one are held to."""
from __future__ import annotations

import random
from dataclasses import dataclass
from typing import List, Optional, Tuple

import torch

import svod_amd

E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
F64 = torch.float64


def half_step(dtype) -> float:
    """The most a value is off, relative to itself, when it is rounded to `dtype`."""
    return torch.finfo(dtype).eps / 2


def exponents(x: torch.Tensor) -> torch.Tensor:
    """The scales' exponents of rows [..., D]: the least e >= -117 with max|x| <= 448 * 2^e over the finite values."""
    amax = torch.where(torch.isfinite(x), x.to(F64).abs(), 0.0).amax(-1)
    e = torch.full(amax.shape, -117, dtype=torch.int64)
    for at in range(-117, 121):
        e = torch.where(amax > 448.0 * 2.0 ** at, at + 1, e)
    return e


def quantised(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """(values, exponents) of rows [..., D] stored in 8 bits, the values as the codes stand for them."""
    e = exponents(x)
    y = x.to(F64) * torch.pow(2.0, -e.to(F64))[..., None]
    top = 8 if x.dtype == torch.float16 else 120
    most = torch.where(e >= top, 240.0, 448.0).to(F64)[..., None]
    # Four significant bits, steps of 2^-9 at least, ties to the even one.
    _, power = torch.frexp(y.abs().clamp(min=2.0 ** -20))
    step = torch.pow(2.0, (power - 4).clamp(min=-9).to(F64))
    y = torch.where(torch.isfinite(y), torch.maximum(torch.minimum(torch.round(y / step) * step, most), -most), float("nan"))
    return y * torch.pow(2.0, e.to(F64))[..., None], e


@dataclass
class Case:
    """A cache and a step's place in it, on the host; `pages` holds the device's copies."""

    lens: List[int]
    starts: List[int]
    table: torch.Tensor
    k: torch.Tensor  # pools in 64 bits, as they stand
    v: torch.Tensor
    rows: int  # of the packed operands
    dtype: torch.dtype
    pages: "svod_amd.Pages"

    def tokens(self, which: str, b: int, n: Optional[int] = None) -> torch.Tensor:
        """Sequence b's first n tokens [n, kv_heads, D]."""
        pool = getattr(self, which)
        page = pool.shape[2]
        n = self.lens[b] if n is None else n
        ids = self.table[b][:-(-n // page)].long()
        return pool[ids].transpose(1, 2).reshape(-1, pool.shape[1], pool.shape[3])[:n]

    def places(self):
        """(packed row, sequence, position) of every new token that has a position."""
        for b, n in enumerate(self.lens):
            fresh = self.starts[b + 1] - self.starts[b]
            for i in range(fresh):
                if n - fresh + i >= 0:
                    yield self.starts[b] + i, b, n - fresh + i


def make(device, context, fresh, *, kv_heads=2, d=64, page=16, dtype=torch.bfloat16, coded=False, seed=0, rows_before=0,
         rows_after=0, lens=None, wide=(torch.int32, torch.int32), spare=2, columns=None, fill=float("nan")) -> Case:
    """Sequences of `context[b]` earlier and `fresh[b]` new tokens (`lens`: other lengths than their sums), with the pages of
    the pool in any order; rows and pages of no token hold `fill`, the table past a sequence's pages a page that is none."""
    g = torch.Generator().manual_seed(seed)
    lens = [c + t for c, t in zip(context, fresh)] if lens is None else lens
    counts = [-(-n // page) for n in lens]
    count = sum(counts) + spare
    order = torch.randperm(count, generator=g).tolist()
    width = columns or max([1, *counts])
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    table[:, 1::2] = 0x7fffffff
    at = 0
    used = torch.zeros(count, page, dtype=torch.bool)
    for b, c in enumerate(counts):
        ids = order[at:at + c]
        table[b, :c] = torch.tensor(ids, dtype=torch.int32)
        for j, i in enumerate(ids):
            used[i, :max(0, min(page, lens[b] - j * page))] = True
        at += c
    starts = [rows_before]
    for t in fresh:
        starts.append(starts[-1] + t)

    def pool():
        x = (torch.randn(count, kv_heads, page, d, generator=g) * (0.5 + torch.rand(d, generator=g) * 2)).to(dtype)
        return torch.where(used[:, None, :, None], x, torch.tensor(fill, dtype=dtype))

    pools = [pool(), pool()]
    if coded:
        stood, scales, codes = [], [], []
        for x in pools:
            y, e = quantised(x)
            codes.append((y * torch.pow(2.0, -e.to(F64))[..., None]).float().to(E4M3))
            scales.append((e + 127).to(torch.uint8))
            stood.append(y)
        sent = [c.view(torch.uint8).to(device).view(E4M3) for c in codes]
        scales = tuple(s.to(device).view(E8M0) for s in scales)
    else:
        stood, sent, scales = [x.to(F64) for x in pools], [x.to(device) for x in pools], None
    pages = svod_amd.Pages(sent[0], sent[1], table.to(device), torch.tensor(lens, dtype=wide[0], device=device),
                           torch.tensor(starts, dtype=wide[1], device=device), scales=scales)
    return Case(lens, starts, table, stood[0], stood[1], starts[-1] + rows_after, dtype, pages)


def attention(case: Case, q: torch.Tensor, causal=False, window=None, scale=None):
    """(out, allowed) [rows, H, D]: the result in 64 bits, NaN in rows of no sequence, and how far a kernel's may be from it.

    Allowed, with u the half step of the 16-bit type: a probability rounded to it is off by u of itself, so the sum of p v by
    u * A, A the probabilities' mean of |v|; the result's own rounding is u * |o|.  A score is a sum of D products in 32 bits, off by
    (D + 4) 2^-24 of the sum of their magnitudes S (log2 e and the exponent's own rounding among the 4, and 2^-20 for the
    hardware's exponential); that much of itself a probability moves, in the sum above and the sum below: 2 A times it.  The sums over n keys in
    32 bits add n 2^-24 A each.  In f16 a probability below 2^-14 is off by up to 2^-25, beside a largest one of 1 or more."""
    rows, heads, d = q.shape
    hkv = case.k.shape[1]
    scale = d ** -0.5 if scale is None else scale
    out = torch.full((rows, heads, d), float("nan"), dtype=F64)
    allowed = torch.zeros((rows, heads, d), dtype=F64)
    u = half_step(q.dtype)
    q = q.to(F64).cpu()
    for b, n in enumerate(case.lens):
        s, e = case.starts[b], case.starts[b + 1]
        if e == s:
            continue
        k, v = (case.tokens(x, b).repeat_interleave(heads // hkv, 1).transpose(0, 1) for x in ("k", "v"))  # [H, n, D]
        at = torch.arange(n - (e - s), n)[:, None]
        key = torch.arange(n)[None]
        seen = (torch.ones((e - s, n), dtype=torch.bool) & (at >= 0)) if causal else torch.ones((e - s, n), dtype=torch.bool)
        if causal:
            seen &= key <= at
        if window is not None:
            seen &= (key >= at - window[0]) & (key <= at + window[1])
        z = (q[s:e].transpose(0, 1) @ k.transpose(1, 2)) * scale
        size = (q[s:e].transpose(0, 1).abs() @ k.transpose(1, 2).abs()) * abs(scale)
        z = z.masked_fill(~seen, -float("inf"))
        some = seen.any(-1)[None, :, None]
        top = z.amax(-1, keepdim=True) if n else torch.zeros(heads, e - s, 1, dtype=F64)
        p = torch.where(seen, torch.exp(z - torch.where(some, top, 0.0)), 0.0)
        total = p.sum(-1, keepdim=True).clamp(min=1e-300)
        o = torch.where(some, p @ v / total, 0.0)
        mean = torch.where(some, p @ v.abs() / total, 0.0)
        worst = torch.where(seen, size, 0.0).amax(-1, keepdim=True) if n else torch.zeros_like(total)
        off = mean * (u + 2 * ((d + 4) * 2.0 ** -24 * worst + 2.0 ** -20) + 2 * n * 2.0 ** -24) + o.abs() * u
        if q.dtype is not None and case.dtype == torch.float16:
            off = off + n * 2.0 ** -25 * (v.abs().amax() if n else 0.0)
        out[s:e] = o.transpose(0, 1)
        allowed[s:e] = off.transpose(0, 1) * (1 + 2.0 ** -6)
    return out, allowed


def draw_lengths(seed: int, count: int, context: int, fresh: int):
    r = random.Random(seed)
    return [r.randint(0, context) for _ in range(count)], [r.randint(0, fresh) for _ in range(count)]
