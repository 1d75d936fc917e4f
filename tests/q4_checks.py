"""Checks of the attention over the 4-bit cache by rows and by single keys (torch, CPU),
for what the value-wise bounds of q4_oracle.py leave open: those add up every rounding at
its worst and pass the size of the outputs where keys are many.

near_rows: a row's error relative to the row.  Its output is rounded once, half a step
h of its type.  16-bit queries: a weight (times a scale) is rounded to fp16, and where
tiles are shared each key and value too, twice: five times 2^-11 at most, less than h of
bf16; that is relative to the weighted values that are summed, and so to the row where
they add up at random, as the row itself does.  fp16 has one such rounding and h =
2^-11.  What fp32 sums add is far below.  Less than 3 h; the bound is 4.  fp32: a score
is off by hd sums at random, a weight by 2^-22, a sum of n keys, 32 at a time, by n / 64
half steps: 64 + n / 64 half steps.

planted: queries that score two keys alike and 60 above the mean, one of them at a
border, so that a row is about the mean of two values.  A score is a sum of |q| |k| of
about 1.3 times 60, off by 2^-10 of that at the very most (keys made into fp16 numbers by
two roundings), 0.08; so a weight by 0.04, and a row by less than a sixteenth of the
distance of both values, beside its rounding.  A key that is lost moves it by a half, one
that counts twice by a sixth.
"""
import torch

import q4_oracle as qo
from serve_oracle import half_step


def joint(batch, b):
    """Keys and values [2][n_kv, keys, hd] of sequence b in 64 bits (0 where a page is not
    there) and which are there."""
    codes, pairs, there = batch.rows(b)
    x = qo.values(codes, pairs)
    return [torch.where(there[None, :, None], x[:, i].transpose(0, 1), 0.0) for i in range(2)], there


def exact(batch, q, tokens, scale, count=None):
    """Outputs [N, n_q, hd] in 64 bits; count: how often key j of a joint axis counts (a
    mistake, planted)."""
    out = torch.zeros(q.shape, dtype=torch.float64)
    for b in range(len(batch.lens)):
        (k, v), there = joint(batch, b)
        n = len(there)
        times = there.double() if count is None else there * count[:n].double()
        ends = batch.prefix + (n - batch.prefix - tokens + 1 + torch.arange(tokens)).clamp(min=0)
        w = times * (torch.arange(n)[None] < ends[:, None])             # [tokens, keys]
        for h in range(batch.n_kv):
            at = slice(b * tokens, (b + 1) * tokens), slice(h * batch.rep, (h + 1) * batch.rep)
            s = q[at].double() @ k[h].T * scale                         # [tokens, rep, keys]
            s = s.masked_fill((w == 0)[:, None], -float("inf"))
            if n and bool((w > 0).any()):
                p = (s - s.amax(-1, keepdim=True).clamp(min=-1e300)).exp() * w[:, None]
                total = p.sum(-1, keepdim=True)
                out[at] = p @ v[h] / torch.where(total > 0, total, 1.0)
    return out


def bound(batch):
    n = batch.prefix + max(batch.lens, default=0)
    return half_step(batch.dtype) * (64 + n / 64 if batch.dtype == torch.float32 else 4)


def near_rows(got, want, bar, what):
    got = got.double().cpu()
    off, size = (got - want).norm(dim=-1), want.norm(dim=-1)
    bad = ~(off <= bar * size)
    worst = float((off / size.clamp(min=1e-300))[size > 0].max()) if bool((size > 0).any()) else 0.0
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} rows off, by {worst:.2e} at most, bound {bar:.2e}"
    return worst


def borders(n):
    """The first and last of n keys and those beside every tile's border."""
    near = {0, n - 1} | {32 * t + d for t in range(n // 32 + 1) for d in (-1, 0, 1)}
    return [j for j in near if 0 <= j < n]


def planted(batch, tokens, scale, top=60.0):
    """Queries, and each row's two keys' values."""
    N, g = tokens * len(batch.lens), batch.g
    q = torch.zeros(N, batch.n_q, batch.hd, dtype=torch.float64)
    two = torch.zeros(2, N, batch.n_q, batch.hd, dtype=torch.float64)
    turn = {}                                           # the next border of each stretch of keys
    for b in range(len(batch.lens)):
        (k, v), there = joint(batch, b)
        for t in range(tokens):
            own = max(len(there) - batch.prefix - (tokens - 1 - t), 0)
            stretches = [(0, batch.prefix)] * (batch.prefix > 0) + [(batch.prefix, own)] * (own > 0)
            n = batch.prefix + own
            if n < 2:
                continue
            for i in range(batch.n_q):
                first, size = stretches[(i + t) % len(stretches)]
                key = b if first else -1, size
                if not turn.get(key):
                    at = borders(size)
                    turn[key] = [at[x] for x in torch.randperm(len(at), generator=g).tolist()]
                j = first + turn[key].pop()
                other = (j + 1 + int(torch.randint(0, n - 1, (1,), generator=g))) % n
                h = i // batch.rep
                pair = torch.stack([k[h, j], k[h, other]])
                want = torch.full((2, 1), top / scale, dtype=torch.float64)
                q[b * tokens + t, i] = (pair.T @ torch.linalg.solve(pair @ pair.T, want))[:, 0]
                two[:, b * tokens + t, i] = torch.stack([v[h, j], v[h, other]])
    return q.to(batch.dtype), two


def near_planted(got, want, two, batch, what):
    got = got.double().cpu()
    apart = (two[0] - two[1]).norm(dim=-1)
    off = (got - want).norm(dim=-1)
    bad = ~(off <= apart / 16 + 2 * half_step(batch.dtype) * want.norm(dim=-1))
    worst = float((off / apart.clamp(min=1e-300))[apart > 0].max())
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} rows off, by {worst:.3f} of their two values' distance"
    return worst
