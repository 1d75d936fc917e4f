"""Greedy decoding of a batch of prompts behind one shared prefix, over the
compressed linears of a decoder.Qwen3Decoder and a paged key/value cache.

The prefix (a system prompt, a document) is run once; its pages are read by
every sequence and by the attention once for all of them.  Each prompt's and
each new token's keys and values are appended to the sequence's own pages.
Per layer: torch.ops.cbq.paged_append (head norm, rotation, pages), then
prefix_attention_prompt for the ragged prompts or prefix_attention_decode for
one token a sequence; the linears take the batch's tokens together (2..63 on
the few-token GEMM, more on the prompt GEMM).

    batch = BatchDecoder(decoder.from_synthetic(cfg, tensors), n_pages=512)
    batch.set_prefix(system_ids)
    tokens = batch.generate([question_ids, other_ids, ...], n_new=64)

Activations are fp32; the cache is fp32 or one of the 16-bit types, to which
queries, keys and values are rounded, and in the attention the softmax weights
(whose sum is not) and the outputs.  Tokens stay on the device between
steps; the host only counts positions and hands out pages.
"""
from __future__ import annotations

from typing import List, Optional, Sequence

import torch

import cbq_ops


class PagePool:
    """Pages of every layer, [layers, n_pages, 2, n_kv, page, head_dim] (keys,
    values), and which of them are free."""

    def __init__(self, cfg, n_pages: int, page: int, dtype: torch.dtype, device):
        if page < 1:
            raise ValueError(f"pages of {page} rows")
        self.page = page
        self.pages = torch.zeros(cfg.layers, n_pages, 2, cfg.n_kv, page, cfg.head_dim, dtype=dtype,
                                 device=device)
        self._free = list(range(n_pages - 1, -1, -1))

    def take(self, tokens: int) -> List[int]:
        """Pages for `tokens` rows."""
        n = -(-tokens // self.page)
        if n > len(self._free):
            raise RuntimeError(f"{n} pages of {self.page} rows needed, {len(self._free)} are free")
        return [self._free.pop() for _ in range(n)]

    def give(self, pages: Sequence[int]) -> None:
        self._free.extend(pages)


class BatchDecoder:
    """See the module's text.  model: any Qwen3Decoder (its own one-sequence
    cache is not used); positions stay below model.max_len."""

    def __init__(self, model, n_pages: int, page: int = 64, dtype: torch.dtype = torch.float32):
        self.model, self.cfg, self.device = model, model.cfg, model.device
        self.ops = cbq_ops.load()
        self.pool = PagePool(model.cfg, n_pages, page, dtype, model.device)
        self.prefix = 0
        self._prefix_pages: List[int] = []
        self._prefix_table = self._ints([])
        self._own: List[List[int]] = []         # pages of each sequence
        self._lens: List[int] = []              # own tokens of each sequence
        self._tables: Optional[torch.Tensor] = None

    def _ints(self, values, dtype=torch.int32) -> torch.Tensor:
        return torch.tensor(values, dtype=dtype, device=self.device)

    # ---- layers over stacked tokens -------------------------------------------
    def _layers(self, ids: torch.Tensor, positions, slots, attend) -> torch.Tensor:
        """The final norm's output [N, hidden] of N stacked tokens; attend(q,
        k_pages, v_pages) is the layer's attention."""
        c, m, g = self.cfg, self.model, self.model.glue
        nq, nk = c.n_q * c.head_dim, c.n_kv * c.head_dim
        N = ids.numel()
        h = m.embed(ids).reshape(N, c.hidden).to(torch.float32)
        x = g.add_rms(h, None)
        for i in range(c.layers):
            p = f"model.layers.{i}."
            qkv = m.linears.get(p + "self_attn.qkv_proj")
            if qkv is not None:                  # row-stacked q/k/v: read in place
                q, k, v = qkv(x).split([nq, nk, nk], 1)
            else:
                q, k, v = (m.linears[p + f"self_attn.{n}_proj"](x) for n in "qkv")
            kp, vp = self.pool.pages[i, :, 0], self.pool.pages[i, :, 1]
            q = self.ops.paged_append(q.unflatten(1, (c.n_q, c.head_dim)),
                                      k.unflatten(1, (c.n_kv, c.head_dim)),
                                      v.unflatten(1, (c.n_kv, c.head_dim)), m.cos, m.sin, positions,
                                      slots, kp, vp, True, None, None, c.eps)
            att = attend(q, kp, vp).flatten(1).to(torch.float32)
            x = g.add_rms(h, m.linears[p + "self_attn.o_proj"](att))
            gu = m.linears.get(p + "mlp.gate_up_proj")
            if gu is not None:
                y = gu(x)
                a = g.silu_mul(y[:, :c.inter].contiguous(), y[:, c.inter:].contiguous())
            else:
                a = g.silu_mul(m.linears[p + "mlp.gate_proj"](x), m.linears[p + "mlp.up_proj"](x))
            x = g.add_rms(h, m.linears[p + "mlp.down_proj"](a))
        return x

    def _prompts(self, runs: Sequence[Sequence[int]], tables: torch.Tensor, pages, prefix: int,
                 prefix_table: torch.Tensor) -> torch.Tensor:
        """Runs of new tokens from own position 0 on: the final norm's output of
        each run's last token, [len(runs), hidden]."""
        lens = [len(r) for r in runs]
        ends = [0]
        for n in lens:
            ends.append(ends[-1] + n)
        positions = self._ints([prefix + j for n in lens for j in range(n)], torch.int64)
        slots = self._ints([row[j // self.pool.page] * self.pool.page + j % self.pool.page
                            for row, n in zip(pages, lens) for j in range(n)], torch.int64)
        q_start, lengths = self._ints(ends), self._ints(lens)
        scale = self.cfg.head_dim ** -0.5

        def attend(q, kp, vp):
            return self.ops.prefix_attention_prompt(q, q_start, kp, vp, prefix_table, prefix, tables,
                                                    lengths, scale)
        ids = self._ints([t for r in runs for t in r], torch.int64)
        x = self._layers(ids, positions, slots, attend)
        return x[self._ints([e - 1 for e in ends[1:]], torch.int64)]

    # ---- public API --------------------------------------------------------------
    def release(self) -> None:
        """Gives the sequences' pages back; the prefix stays."""
        for pages in self._own:
            self.pool.give(pages)
        self._own, self._lens, self._tables = [], [], None

    @torch.no_grad()
    def set_prefix(self, ids: Sequence[int]) -> None:
        """Runs `ids` as the shared prefix of what follows (none when empty); the
        sequences of the prefix before are released."""
        if len(ids) > self.model.max_len:
            raise ValueError(f"a prefix of {len(ids)} tokens exceeds max_len {self.model.max_len}")
        self.release()
        self.pool.give(self._prefix_pages)
        self._prefix_pages, self.prefix, self._prefix_table = [], 0, self._ints([])
        if not len(ids):
            return
        pages = self.pool.take(len(ids))
        try:
            table = self._ints(pages)
            self._prompts([ids], table[None], [pages], 0, self._ints([]))
        except BaseException:
            self.pool.give(pages)
            raise
        self._prefix_pages, self.prefix, self._prefix_table = pages, len(ids), table

    @torch.no_grad()
    def start(self, prompts: Sequence[Sequence[int]], room: int) -> torch.Tensor:
        """Runs a batch of prompts behind the prefix, with pages for `room` more
        tokens each: logits [batch, vocab] of their last tokens."""
        if not prompts or not all(len(p) for p in prompts):
            raise ValueError("every prompt needs a token")
        if room < 0:
            raise ValueError(f"room for {room} more tokens")
        longest = self.prefix + max(len(p) for p in prompts) + room
        if longest > self.model.max_len:
            raise ValueError(f"sequences of {longest} exceed max_len {self.model.max_len}")
        self.release()
        try:
            for p in prompts:
                self._own.append(self.pool.take(len(p) + room))
            width = max(len(r) for r in self._own)
            self._tables = self._ints([r + [-1] * (width - len(r)) for r in self._own])
            x = self._prompts(prompts, self._tables, self._own, self.prefix, self._prefix_table)
        except BaseException:
            self.release()
            raise
        self._lens = [len(p) for p in prompts]
        return self.model.linears["lm_head"](x)

    @torch.no_grad()
    def step(self, tokens: torch.Tensor) -> torch.Tensor:
        """One token of each sequence (device int64 [batch]): logits [batch, vocab]."""
        page, scale = self.pool.page, self.cfg.head_dim ** -0.5
        if not self._lens:
            raise ValueError("no sequences: start() first")
        if tokens.numel() != len(self._lens):
            raise ValueError(f"{tokens.numel()} tokens for {len(self._lens)} sequences")
        if any(n >= len(row) * page for n, row in zip(self._lens, self._own)):
            raise RuntimeError("no room for another token: start() with more")
        if self.prefix + max(self._lens) >= self.model.max_len:
            raise ValueError(f"sequences exceed max_len {self.model.max_len}")
        positions = self._ints([self.prefix + n for n in self._lens], torch.int64)
        slots = self._ints([row[n // page] * page + n % page for n, row in zip(self._lens, self._own)],
                           torch.int64)
        lens = [n + 1 for n in self._lens]
        lengths = self._ints(lens)

        def attend(q, kp, vp):
            return self.ops.prefix_attention_decode(q, kp, vp, self._prefix_table, self.prefix,
                                                    self._tables, lengths, scale)
        x = self._layers(tokens, positions, slots, attend)
        self._lens = lens
        return self.model.linears["lm_head"](x)

    @torch.no_grad()
    def generate(self, prompts: Sequence[Sequence[int]], n_new: int) -> List[List[int]]:
        """Greedy: n_new tokens of each prompt behind the prefix (EOS ignored)."""
        if n_new < 1:
            return [[] for _ in prompts]
        tokens = [torch.argmax(self.start(prompts, n_new - 1), -1)]      # the last one is not run
        for _ in range(n_new - 1):
            tokens.append(torch.argmax(self.step(tokens[-1]), -1))
        self.release()
        return torch.stack(tokens, 1).tolist()


def main() -> None:
    """A synthetic model's batch: prompts of several lengths behind one prefix."""
    import argparse
    import random
    import time

    import decoder
    import synthetic
    ap = argparse.ArgumentParser(description=main.__doc__)
    ap.add_argument("--config", default="qwen3-1.7b", choices=sorted(synthetic.CONFIGS))
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--batch", type=int, default=8)
    ap.add_argument("--prefix", type=int, default=512)
    ap.add_argument("--new", type=int, default=32)
    ap.add_argument("--cache", default="float32", choices=["float32", "bfloat16", "float16"])
    a = ap.parse_args()
    syn = synthetic.SyntheticDecoder(a.config, layers=a.layers, log=lambda *x: None)
    c = syn.cfg
    cfg = decoder.DecoderConfig(layers=c["layers"], hidden=c["hidden"], inter=c["inter"], n_q=c["n_q"],
                                n_kv=c["n_kv"], head_dim=c["head_dim"], vocab=c["vocab"])
    tensors = syn.build_fixed(syn.all_linears() + [syn.embed])
    model = decoder.from_synthetic(cfg, tensors, max_len=a.prefix + 256 + a.new)
    rng = random.Random(0)
    prompts = [[rng.randrange(cfg.vocab) for _ in range(rng.randint(1, 256))] for _ in range(a.batch)]
    per = -(-(256 + a.new) // 64)
    batch = BatchDecoder(model, a.batch * per + -(-a.prefix // 64), dtype=getattr(torch, a.cache))
    batch.set_prefix([rng.randrange(cfg.vocab) for _ in range(a.prefix)])
    batch.generate(prompts, 2)                          # loads the kernels
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    tokens = batch.generate(prompts, a.new)
    s = time.perf_counter() - t0
    print(f"{a.batch} prompts of {sum(map(len, prompts))} tokens behind {a.prefix}: "
          f"{a.batch * a.new} tokens in {s:.3f} s ({a.batch * a.new / s:.0f} tokens/s, prompts included)")
    print("first tokens:", [t[:4] for t in tokens])


if __name__ == "__main__":
    main()
