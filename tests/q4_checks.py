"""Checks of the attention over the 4-bit cache by rows (torch, CPU), for what the
value-wise bounds of q4_oracle.py leave open: those add up every rounding at its worst and
pass the size of the outputs where keys are many.

near_rows: a row's error relative to the row.  Its output is rounded once, half a step
h of its type.  16-bit queries: a weight (times a scale) is rounded to fp16, and where
tiles are shared each key and value too, twice: five times 2^-11 at most, less than h of
bf16; that is relative to the weighted values that are summed, and so to the row where
they add up at random, as the row itself does.  fp16 has one such rounding and h =
2^-11.  What fp32 sums add is far below.  Less than 3 h; the bound is 4.  fp32: a score
is off by hd sums at random, a weight by 2^-22, a sum of n keys, 32 at a time, by n / 64
half steps: 64 + n / 64 half steps.
"""
import torch

import q4_oracle as qo


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


def near_rows(got, want, bar, what):
    got = got.double().cpu()
    off, size = (got - want).norm(dim=-1), want.norm(dim=-1)
    bad = ~(off <= bar * size)
    worst = float((off / size.clamp(min=1e-300))[size > 0].max()) if bool((size > 0).any()) else 0.0
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} rows off, by {worst:.2e} at most, bound {bar:.2e}"
    return worst
