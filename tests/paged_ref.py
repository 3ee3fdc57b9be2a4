"""Plain implementations of the paged 4-bit latent cache: the allocator as Python lists, the block
format and the attention in 64 bits."""

from __future__ import annotations

import torch

LAT, ROPE, ROW, TOKEN = 512, 64, 576, 400
VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


class Allocator:
    """paged_cache_step, request by request."""

    def __init__(self, lens, table, ring, head, count, page_size):
        self.lens, self.ps = list(lens), page_size
        self.table = [list(r) for r in table]
        self.ring, self.head, self.count = list(ring), head, count

    def pages(self, n):
        return -(-n // self.ps)

    def step(self, delta, max_tokens):
        """(slots, positions, rows) of the new tokens; changes lens, table, ring, head and count."""
        P, width = len(self.ring), len(self.table[0])
        out = [(-1, -1, -1)] * max_tokens
        tokens = pages = used = back = 0
        errors = 0
        after = list(self.lens)
        for b, d in enumerate(delta):
            have = self.pages(self.lens[b])
            if d < 0:
                after[b] = max(self.lens[b] + d, 0)
                for k in range(self.pages(after[b]), have):
                    self.ring[(self.head + self.count + back) % P] = self.table[b][k]
                    back += 1
            if d <= 0:
                continue
            fits = self.lens[b] + d <= width * self.ps
            need = self.pages(self.lens[b] + d) - have if fits else 0
            first, first_page = tokens, pages
            tokens += d
            pages += need
            if not fits:
                errors |= 1
            elif tokens > max_tokens:
                errors |= 8
            elif need and pages > self.count:
                errors |= 2
            else:
                for k in range(need):
                    self.table[b][have + k] = self.ring[(self.head + first_page + k) % P]
                used += need
                after[b] = self.lens[b] + d
                for j in range(d):
                    t = self.lens[b] + j
                    out[first + j] = (self.table[b][t // self.ps] * self.ps + t % self.ps, t, b)
        self.lens = after
        self.head = (self.head + used) % P
        self.count += back - used
        return [list(x) for x in zip(*out)] if out else [[], [], []], errors


def pow2(e):
    """2^e in 64 bits, exactly (torch.pow on the GPU is an ulp off for some)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def held(rows: torch.Tensor) -> torch.Tensor:
    """The values, in 64 bits, that the cache holds of bf16 rows [n, 576]."""
    x = rows[:, :LAT].double().unflatten(1, (16, 32))
    bad = ~torch.isfinite(x).all(-1, keepdim=True)
    x = torch.where(bad, 0.0, x)
    most = x.abs().amax(-1, keepdim=True)
    m, e = torch.frexp(most)  # most = m 2^e with m in [1/2, 1): within 6 * 2^(e - 3) up to m = 3/4
    scale = pow2((e - 3 + (m > 0.75)).clamp(-124, 125))
    scale = torch.where(most == 0, 1.0, scale)
    y = (x.abs() / scale).clamp(max=6.0)
    value = torch.tensor(VALUES, dtype=torch.float64, device=rows.device)
    away = (y[..., None] - value).abs()
    away[..., 1::2] += 1e-12  # a tie goes to the even code; differing distances differ by far more
    got = value[away.argmin(-1)] * torch.sign(x) * scale
    got = torch.where(bad, torch.nan, got)
    return torch.cat([got.flatten(1), rows[:, LAT:].double()], 1)


def stored(pages: torch.Tensor, slots: torch.Tensor, page_size: int) -> torch.Tensor:
    """The 64-bit rows that the bytes of a pool's slots stand for."""
    slots = slots.long()
    pg, i = slots // page_size, slots % page_size

    def take(start, n):
        cols = start + i * n
        return pages[pg[:, None], cols[:, None] + torch.arange(n, device=pages.device)]

    code, rope = take(0, 256).long(), take(256 * page_size, 128)
    scale = take(384 * page_size, 16)
    value = torch.tensor(VALUES + tuple(-v for v in VALUES), dtype=torch.float64, device=pages.device)
    x = torch.stack([value[code % 16], value[code // 16]], -1).flatten(1).unflatten(1, (16, 32))
    s = torch.where(scale == 255, torch.nan, pow2(scale.long() - 127))
    return torch.cat([(x * s[..., None]).flatten(1), rope.contiguous().view(torch.bfloat16).double()], 1)


def attention(q, keys, seen, scale):
    """One query token's heads q [H, 576] over the rows keys [n, 576] (64 bits), the first `seen` of
    them: (outputs [H, 512], how far a kernel that multiplies bf16 may be off each of them)."""
    h = q.shape[0]
    if seen <= 0:
        z = torch.zeros(h, LAT, dtype=torch.float64, device=q.device)
        return z, z
    q, k = q.double(), keys[:seen]
    p = torch.softmax(q @ k.T * scale, -1)
    v = k[:, :LAT]
    o, mass = p @ v, p @ v.abs()
    # scores: fp32 sums of 576 exact products, scaled (2^-24 a step); exp2 and its argument 2^-20;
    # p in bf16 (2^-8) against fp32 sums; the division and the joining of parts 2^-20; out in bf16
    size = (q.abs() @ k.abs().T).amax(-1, keepdim=True) * scale
    tol = 2.0 ** -8 * o.abs() + mass * (2.0 ** -8 * 1.01 + 2 * 580 * 2.0 ** -24 * size + 2.0 ** -18)
    return o, tol * 1.01 + 1e-30
