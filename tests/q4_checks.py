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


def near_rows(got, want, bar, what):
    got = got.double().cpu()
    off, size = (got - want).norm(dim=-1), want.norm(dim=-1)
    bad = ~(off <= bar * size)
    worst = float((off / size.clamp(min=1e-300))[size > 0].max()) if bool((size > 0).any()) else 0.0
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} rows off, by {worst:.2e} at most, bound {bar:.2e}"
    return worst
