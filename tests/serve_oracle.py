"""Plain float64 forms of the batched serving operators (torch, CPU) and the
batches that the tests run them on.

Tolerances.  An output of type t is rounded once: half a step, eps_t / 2 of its
value.  Append adds fp32 arithmetic: at most 16 squares a thread, 4 levels of
shuffles, a mean, a root, a quotient, two products for the norm (half of the
sum's error goes through the root), then two products and a sum a pair: below
32 half steps of the pair's magnitude.  Attention, with A = sum p |v| / sum p
and S = scale * max_j sum |q_i k_ij|:
  - a score is off by (hd + 4) half steps of S (hd products and sums, the
    factor, exp2's argument), which is a relative error of its weight, and
    twice that of the quotient;
  - sums of n weights, 16 or 64 at a time and joined over waves and parts, are
    off by fewer than n / 16 + 64 half steps of A;
  - 16-bit weights are rounded to the type: half a step of A, and for fp16,
    whose smallest step is 2^-24, 2^-25 a weight: n 2^-25 max|v| / sum p, the
    maximum over the keys.
"""
import random

import torch

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
HALF = 2.0 ** -24                       # half a step of fp32


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


class Batch:
    """Sequences over a pool of pages: own lengths, a shared prefix, tables with
    room to grow, pages scattered; unused rows of the pool hold `fill`."""

    def __init__(self, lens, prefix=0, n_kv=2, rep=3, hd=64, page=16, dtype="bf16", rows_first=False,
                 room=1, seed=0, fill=float("nan"), scale_k=1.0):
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
        shape = (n_pages, 2, page, n_kv, hd) if rows_first else (n_pages, 2, n_kv, page, hd)
        pages = torch.full(shape, fill, dtype=self.dtype)
        if rows_first:
            pages = pages.transpose(2, 3)
        self.k, self.v = pages[:, 0], pages[:, 1]
        for table, n in [(self.prefix_table, prefix)] + list(zip(self.tables, lens)):
            for j in range(n):
                p, r = int(table[j // page]), j % page
                self.k[p, :, r] = scale_k * torch.randn(n_kv, hd, generator=g)
                self.v[p, :, r] = torch.randn(n_kv, hd, generator=g)

    def queries(self, n, factor=1.0):
        return (factor * torch.randn(n, self.n_q, self.hd, generator=self.g)).to(self.dtype)

    def dense(self, b):
        """Keys and values [keys, n_kv, hd] of sequence b's joint axis in 64
        bits, and which of them are there."""
        n_pages = self.k.shape[0]
        k, v, there = [], [], []
        for table, n in ((self.prefix_table, self.prefix), (self.tables[b], int(self.lengths[b]))):
            for j in range(n):
                p, r = int(table[j // self.page]), j % self.page
                ok = 0 <= p < n_pages
                there.append(ok)
                k.append(self.k[p, :, r].double() if ok else torch.zeros(self.n_kv, self.hd).double())
                v.append(self.v[p, :, r].double() if ok else torch.zeros(self.n_kv, self.hd).double())
        e = torch.zeros(0, self.n_kv, self.hd, dtype=torch.float64)
        return (torch.stack(k) if k else e, torch.stack(v) if v else e,
                torch.tensor(there, dtype=torch.bool))

    def cuda(self):
        """The device's copies: (k_pages, v_pages, prefix_table, tables, lengths)."""
        both = torch.empty_strided((self.k.shape[0],) + (2,) + tuple(self.k.shape[1:]),
                                   (self.k.stride(0), self.v.storage_offset()) + self.k.stride()[1:],
                                   dtype=self.dtype, device="cuda")
        both[:, 0].copy_(self.k)
        both[:, 1].copy_(self.v)
        return (both[:, 0], both[:, 1], self.prefix_table.cuda(), self.tables.cuda(),
                self.lengths.cuda())


def attend(batch, q, q_start, scale):
    """Outputs [N, n_q, hd] in 64 bits and the tolerance of each."""
    out = torch.zeros(q.shape, dtype=torch.float64)
    tol = torch.zeros(q.shape, dtype=torch.float64)
    half = half_step(batch.dtype)
    for b in range(len(batch.lens)):
        k, v, there = batch.dense(b)
        lo, hi = int(q_start[b]), int(q_start[b + 1])
        for t in range(lo, hi):
            own = max(int(batch.lengths[b]) - (hi - 1 - t), 0)
            see = there.clone()
            see[batch.prefix + own:] = False
            if not see.any():
                continue
            for h in range(batch.n_q):
                ks, vs = k[see, h // batch.rep], v[see, h // batch.rep]
                x = q[t, h].double()
                s = ks @ x * scale
                p = torch.exp(s - s.max())
                total = p.sum()
                out[t, h] = (p / total) @ vs
                mass = (p / total) @ vs.abs()
                big = abs(scale) * float((ks.abs() @ x.abs()).max())
                n = len(s)
                part = (2 * (batch.hd + 4) * big + n / 16 + 64) * HALF
                tol[t, h] = half * out[t, h].abs() + part * mass
                if batch.dtype != torch.float32:
                    tol[t, h] += half * mass
                if batch.dtype == torch.float16:
                    tol[t, h] += n * 2.0 ** -25 * vs.abs().amax(0) / total + 2.0 ** -25
    return out, tol


def attend_prompt(batch, q, q_start, scale):
    """attend() by matrix products, for larger prompts whose values are finite."""
    out, tol = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    half = half_step(batch.dtype)
    for b in range(len(batch.lens)):
        k, v, there = batch.dense(b)
        lo, hi = int(q_start[b]), int(q_start[b + 1])
        if lo == hi:
            continue
        ends = batch.prefix + (int(batch.lengths[b]) - hi + 1 + torch.arange(lo, hi)).clamp(min=0)
        see = there[None] & (torch.arange(len(k))[None] < ends[:, None])
        assert see.any(-1).all(), "a row without keys"
        for h in range(batch.n_q):
            ks, vs, x = k[:, h // batch.rep], v[:, h // batch.rep], q[lo:hi, h].double()
            s = (x @ ks.T * scale).masked_fill(~see, float("-inf"))
            p = torch.exp(s - s.amax(-1, keepdim=True))
            total = p.sum(-1, keepdim=True)
            big = abs(scale) * (x.abs() @ ks.abs().T).masked_fill(~see, 0).amax(-1, keepdim=True)
            n = see.sum(-1, keepdim=True)
            out[lo:hi, h], mass = p / total @ vs, p / total @ vs.abs()
            tol[lo:hi, h] = half * out[lo:hi, h].abs() + (2 * (batch.hd + 4) * big + n / 16 + 64) * HALF * mass
            if batch.dtype != torch.float32:
                tol[lo:hi, h] += half * mass
            if batch.dtype == torch.float16:
                top = (vs.abs() * there[:, None]).cummax(0).values[ends - 1]
                tol[lo:hi, h] += n * 2.0 ** -25 * top / total + 2.0 ** -25
    return out, tol


def append_rows(x, weight, cos, sin, positions, norm, eps):
    """Normed and rotated heads [N, heads, hd] in 64 bits and the magnitude of
    each value's pair."""
    x = x.double()
    if norm:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
        if weight is not None:
            x = x * weight.double()
    half = cos.shape[1] // 2
    at = torch.where((positions >= 0) & (positions < cos.shape[0]), positions, 0)
    c, s = (t.double()[at, None, :half] for t in (cos, sin))
    a, b, rest = x[..., :half], x[..., half:2 * half], x[..., 2 * half:]
    mag = a.abs() + b.abs()
    return (torch.cat([a * c - b * s, b * c + a * s, rest], -1),
            torch.cat([mag, mag, rest.abs()], -1))


def near(got, want, tol, what):
    """Every value within its tolerance; NaN nowhere."""
    got = got.double().cpu()
    assert got.shape == want.shape
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} values off, first at "
                           f"{bad.nonzero()[0].tolist()}: {got[bad][0]} for {want[bad][0]} +- "
                           f"{tol[bad][0]}")
