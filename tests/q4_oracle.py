"""Plain float64 forms of the operators over the 4-bit paged cache and of the
verification of drafts (torch, CPU), and the batches that the tests run them on.

Tolerances of the attention.  With HALF half a step of fp32, a row's weights p_j,
and of each key's group g scale s, mid m:
  - a score is summed from q (c + z) s, (z + 7.5) q s and q m, z at most 16 (of 16-bit
    queries 256 for half the codes): hd products and sums and eight roundings more (the
    factors, the maximum, exp2's argument), each off by HALF of S = |scale| max_j sum_d
    |q_d| (54.5 s + |m|), 280 s more for 16 bits.  That is a relative error of its weight,
    and twice that of the quotient, of sum p |v| / sum p;
  - the weighted sums add p s (c + z), (z + 7.5) p s and p m, z at most 16 (bf16: 64 for
    half of them): n terms, 32 at a time and joined over waves and parts: fewer than n /
    16 + 64 half steps of sum p (54.5 s + |m|) / sum p, bf16 151 s;
  - p s is cut to fp16 numbers, one for 16-bit queries (half a step, 2^-11 of it), two for
    fp32 (2^-22), times |c - 7.5| <= 7.5, and below 2^-14 of their range to a whole
    step of 2^-25: n 2^-25 max s / sum p times 7.5;
  - a prefix that more than 16 rows of bf16 queries share may be made into fp16 numbers
    first: 2^-11 of each key and value, |m| + 7.5 s of it at most, and 2^-11 of p: a
    score is off by 2^-11 |scale| max_j sum_d |q_d| (7.5 s + |m|), and the sums by 2^-10
    of sum p (7.5 s + |m|) / sum p;
  - the output is rounded once, half a step of its type (fp16: 2^-25 at least).
"""
import random

import torch

from serve_oracle import HALF, TYPES, half_step

GROUP = 64
CUT = {torch.float32: 2.0 ** -22, torch.bfloat16: 2.0 ** -11, torch.float16: 2.0 ** -11}


def order(hd):
    """Places of a row's values among its codes."""
    d = torch.arange(hd)
    g, e = d // GROUP, d % GROUP
    return e // 4 * (hd // 16) + 4 * g + e % 4


def quantise(x):
    """[..., hd] in 64 bits -> codes [..., hd / 2] uint8, pairs [..., hd / 64, 2] bf16."""
    hd = x.shape[-1]
    y = x.double().unflatten(-1, (-1, GROUP))
    top, low = y.amax(-1), y.amin(-1)
    mid = ((top + low) / 2).float().bfloat16()
    m = mid.double()
    scale = (torch.maximum(top - m, m - low) / 7.5).float().bfloat16()
    s = scale.double()
    bad = ~y.isfinite().all(-1) | ~mid.isfinite() | ~scale.isfinite()
    c = (torch.floor((y - m[..., None]) / s[..., None]) + 8).clamp(0, 15)
    c = torch.where(((s > 0) & ~bad)[..., None], c, 8.0).to(torch.uint8).flatten(-2)
    row = torch.empty_like(c)
    row[..., order(hd)] = c
    mid = torch.where(bad, torch.tensor(float("nan"), dtype=torch.bfloat16), mid)
    scale = torch.where(bad, torch.tensor(0.0, dtype=torch.bfloat16), scale)
    return row[..., 0::2] | row[..., 1::2] << 4, torch.stack([scale, mid], -1)


def parts(codes, pairs):
    """(c - 7.5, scale, mid), each [..., hd] in 64 bits."""
    hd = 2 * codes.shape[-1]
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)[..., order(hd)].double()
    p = pairs.double().repeat_interleave(GROUP, -2)
    return c - 7.5, p[..., 0], p[..., 1]


def values(codes, pairs):
    c, s, m = parts(codes, pairs)
    return m + s * c


class Batch:
    """Sequences over a 4-bit pool: own lengths, a shared prefix, tables with room to
    grow, pages scattered.  Rows that no sequence has hold random codes and NaN."""

    def __init__(self, lens, prefix=0, n_kv=2, rep=3, hd=64, page=16, dtype="bf16", rows_first=False,
                 room=1, seed=0, offset=0.0):
        rng, g = random.Random(seed), torch.Generator().manual_seed(seed)
        self.lens, self.prefix, self.n_kv, self.rep, self.hd, self.page = (list(lens), prefix, n_kv,
                                                                           rep, hd, page)
        self.n_q, self.dtype, self.g = n_kv * rep, TYPES[dtype], g
        counts = [-(-n // page) for n in lens]
        shared = -(-prefix // page)
        n_pages = sum(counts) + shared + 2
        pool = list(range(n_pages))
        rng.shuffle(pool)
        width = max(counts, default=0) + room
        self.prefix_table = torch.tensor([pool.pop() for _ in range(shared)], dtype=torch.int32)
        rows = [[pool.pop() for _ in range(c)] + [-1] * (width - c) for c in counts]
        self.tables = torch.tensor(rows, dtype=torch.int32).reshape(len(rows), width)
        self.lengths = torch.tensor(lens, dtype=torch.int32)
        lead = (n_pages, 2, page, n_kv) if rows_first else (n_pages, 2, n_kv, page)
        codes = torch.randint(0, 256, (*lead, hd // 2), generator=g, dtype=torch.uint8)
        pairs = torch.full((*lead, hd // GROUP, 2), float("nan"), dtype=torch.bfloat16)
        if rows_first:
            codes, pairs = codes.transpose(2, 3), pairs.transpose(2, 3)
        self.codes, self.pairs = codes, pairs
        for table, n in [(self.prefix_table, prefix)] + list(zip(self.tables, lens)):
            j = torch.arange(n)
            p, r = table[j // page].long(), j % page
            for i in range(2):
                x = torch.randn(n, n_kv, hd, generator=g) + offset
                codes[p, i, :, r], pairs[p, i, :, r] = quantise(x)

    def queries(self, tokens, factor=1.0):
        n = tokens * len(self.lens)
        return (factor * torch.randn(n, self.n_q, self.hd, generator=self.g)).to(self.dtype)

    def rows(self, b):
        """Codes and pairs [keys, 2, n_kv, ..] of sequence b's joint axis, and which
        of them are there (the others' are page 0's first)."""
        n_pages = self.codes.shape[0]
        at, row, there = [], [], []
        capacity = self.tables.shape[1] * self.page
        for table, n in ((self.prefix_table, self.prefix),
                         (self.tables[b], min(max(int(self.lengths[b]), 0), capacity))):
            j = torch.arange(n)
            p = table[j // self.page].long() if n else j
            ok = (p >= 0) & (p < n_pages)
            at.append(torch.where(ok, p, 0))
            row.append(torch.where(ok, j % self.page, 0))
            there.append(ok)
        at, row, there = (torch.cat(x) for x in (at, row, there))
        return self.codes[at, :, :, row], self.pairs[at, :, :, row], there

    def cuda(self):
        """The device's copies, laid out as here: (k_codes, k_scales, v_codes, v_scales)
        and (prefix_table, tables, lengths)."""
        c, p = (torch.empty_strided(x.shape, x.stride(), dtype=x.dtype, device="cuda").copy_(x)
                for x in (self.codes, self.pairs))
        return ((c[:, 0], p[:, 0], c[:, 1], p[:, 1]),
                (self.prefix_table.cuda(), self.tables.cuda(), self.lengths.cuda()))


def attend(batch, q, tokens, scale):
    """Outputs [N, n_q, hd] in 64 bits and the tolerance of each."""
    out = torch.zeros(q.shape, dtype=torch.float64)
    tol = torch.zeros(q.shape, dtype=torch.float64)
    half, cut = half_step(batch.dtype), CUT[batch.dtype]
    for b in range(len(batch.lens)):
        codes, pairs, there = batch.rows(b)
        length = len(there) - batch.prefix
        for h in range(batch.n_kv):
            (kc, ks, km), (vc, vs, vm) = (parts(codes[:, i, h], pairs[:, i, h]) for i in range(2))
            k, v = km + ks * kc, vm + vs * vc
            k_big = (54.5 if batch.dtype == torch.float32 else 334.5) * ks + km.abs()
            v_big = (151 if batch.dtype == torch.bfloat16 else 54.5) * vs + vm.abs()
            for t in range(tokens):
                see = there.clone()
                see[batch.prefix + max(length - (tokens - 1 - t), 0):] = False
                if not see.any():
                    continue
                n = int(see.sum())
                for i in range(h * batch.rep, (h + 1) * batch.rep):
                    at = (b * tokens + t, i)
                    x = q[at].double()
                    s = k[see] @ x * scale
                    p = torch.exp(s - s.max())
                    p = p / p.sum()
                    out[at] = p @ v[see]
                    big = abs(scale) * float((k_big[see] @ x.abs()).max())
                    tol[at] = (half * out[at].abs() + 2 * (batch.hd + 8) * big * HALF * (p @ v[see].abs())
                               + (n / 16 + 64) * HALF * (p @ v_big[see]) + cut * 7.5 * (p @ vs[see])
                               + 7.5 * n * 2.0 ** -25 * vs[see].amax(0) * p.max())
                    if (batch.prefix and tokens * batch.rep * len(batch.lens) > 16
                            and batch.dtype == torch.bfloat16):
                        made = vm[see].abs() + 7.5 * vs[see]
                        big = abs(scale) * float(((km[see].abs() + 7.5 * ks[see]) @ x.abs()).max())
                        tol[at] += 2.0 ** -10 * ((p @ made) + big * (p @ v[see].abs()))
                    if batch.dtype == torch.float16:
                        tol[at] += 2.0 ** -25
    return out, tol


def verify(probs, drafts, draft_probs, n_drafts, uniforms):
    """(tokens, counts) by the rule as it is told, in 64 bits."""
    B, K = drafts.shape
    V = probs.shape[2]
    tokens, counts = torch.full((B, K + 1), -1, dtype=torch.int64), torch.zeros(B, dtype=torch.int32)
    for b in range(B):
        n = K if n_drafts is None else min(max(int(n_drafts[b]), 0), K)
        u = uniforms[b].double()
        a = 0
        while a < n:
            d = int(drafts[b, a])
            inside = 0 <= d < V
            p = float(probs[b, a, d]) if inside else 0.0
            q = 1.0 if draft_probs is None else float(draft_probs[b, a, d]) if inside else 0.0
            if not float(u[a]) * q < p:
                break
            a += 1
        p = probs[b, a].double()
        w = p.clone()
        if a < n and draft_probs is not None:
            w = w - draft_probs[b, a].double()
        elif a < n and 0 <= int(drafts[b, a]) < V:
            w[int(drafts[b, a])] = 0
        w, p = (torch.where(x > 0, x, 0.0) for x in (w, p))
        w = w if bool((w > 0).any()) else p
        tokens[b, :a] = drafts[b, :a]
        if bool((w > 0).any()):
            c = w.cumsum(0)
            over = (c > float(u[K]) * float(c[-1])).nonzero()
            tokens[b, a] = int(over[0]) if len(over) else int((w > 0).nonzero()[-1])
        counts[b] = a + 1
    return tokens, counts
