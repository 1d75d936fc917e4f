"""Decoding of a batch of prompts behind one shared prefix, over the compressed
linears of a decoder.Qwen3Decoder and a paged key/value cache.

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
    tokens = batch.sample([question_ids, ...], n_new=64, temperature=0.8, drafts=4)

generate() is greedy.  sample() draws from the target's probabilities, and where
drafts are asked for, runs tokens that followed the newest ones earlier in the
text beside the newest: verify() keeps those that the probabilities and the
random numbers accept (torch.ops.cbq.verify_drafts), so the tokens are distributed
as without drafts.

Activations are fp32; the cache is fp32 or one of the 16-bit types, to which
queries, keys and values are rounded, and in the attention the softmax weights
(whose sum is not) and the outputs.  Or it is "q4": keys and values quantised to
4.5 bits as they are written (include/cbq_serve_q4.h; heads of 64, 128 or 256),
read in that form by prefix_attention_decode_q4 for the newest tokens, and read
back to fp32 values, a layer's at a time, for the prompts' attention; queries and
outputs stay fp32.  Tokens stay on the device between the steps of generate(); the
host only counts positions and hands out pages.
"""
from __future__ import annotations

from typing import List, Optional, Sequence, Tuple, Union

import torch

import cbq_ops


class PagePool:
    """Pages of every layer, [layers, n_pages, 2, n_kv, page, head_dim] (keys,
    values), and which of them are free.  dtype "q4": codes [.., head_dim / 2] and
    pairs [.., head_dim / 64, 2] instead."""

    def __init__(self, cfg, n_pages: int, page: int, dtype: Union[torch.dtype, str], device):
        if page < 1:
            raise ValueError(f"pages of {page} rows")
        self.page, self.scales = page, None
        lead = (cfg.layers, n_pages, 2, cfg.n_kv, page)
        if dtype == "q4":
            if cfg.head_dim not in (64, 128, 256):
                raise ValueError(f"a q4 cache of heads of {cfg.head_dim}: 64, 128 or 256")
            self.pages = torch.zeros(*lead, cfg.head_dim // 2, dtype=torch.uint8, device=device)
            self.scales = torch.zeros(*lead, cfg.head_dim // 64, 2, dtype=torch.bfloat16, device=device)
        elif isinstance(dtype, torch.dtype):
            self.pages = torch.zeros(*lead, cfg.head_dim, dtype=dtype, device=device)
        else:
            raise ValueError(f"a cache of {dtype!r}: a floating type or \"q4\"")
        self._free = list(range(n_pages - 1, -1, -1))

    def layer(self, i: int) -> Tuple[torch.Tensor, ...]:
        """Keys and values of layer i; of a q4 cache their codes and pairs."""
        if self.scales is None:
            return self.pages[i, :, 0], self.pages[i, :, 1]
        return self.pages[i, :, 0], self.scales[i, :, 0], self.pages[i, :, 1], self.scales[i, :, 1]

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

    def __init__(self, model, n_pages: int, page: int = 64,
                 dtype: Union[torch.dtype, str] = torch.float32):
        self.model, self.cfg, self.device = model, model.cfg, model.device
        self.ops = cbq_ops.load()
        self.pool = PagePool(model.cfg, n_pages, page, dtype, model.device)
        self.q4 = dtype == "q4"
        self.prefix = 0
        self._prefix_ids: List[int] = []
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
        *self.pool.layer(i)) is layer i's attention."""
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
            cache = self.pool.layer(i)
            append = self.ops.paged_append_q4 if self.q4 else self.ops.paged_append
            q = append(q.unflatten(1, (c.n_q, c.head_dim)), k.unflatten(1, (c.n_kv, c.head_dim)),
                       v.unflatten(1, (c.n_kv, c.head_dim)), m.cos, m.sin, positions, slots, *cache,
                       True, None, None, c.eps)
            att = attend(q, *cache).flatten(1).to(torch.float32)
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
        if self.q4:
            # a compact pool of values: the prefix's pages, then each run's, in order
            page = self.pool.page
            used = [row[:-(-n // page)] for row, n in zip(pages, lens)]
            shared = self._prefix_pages if prefix else []
            rows = (self._ints(shared + [p for row in used for p in row], torch.int64)[:, None] * page
                    + torch.arange(page, device=self.device)).flatten()
            prefix_table = self._ints(range(len(shared)))
            firsts = [len(shared)]
            for row in used:
                firsts.append(firsts[-1] + len(row))
            width = max(map(len, used))
            tables = self._ints([list(range(f, f + len(row))) + [-1] * (width - len(row))
                                 for f, row in zip(firsts, used)])

        def attend(q, *cache):
            if self.q4:
                cache = [x.unflatten(0, (-1, page)).transpose(1, 2)
                         for x in self.ops.paged_read_q4(*cache, rows, q.dtype)]
            return self.ops.prefix_attention_prompt(q, q_start, *cache, prefix_table, prefix, tables,
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
        self._prefix_ids = []
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
        self._prefix_ids = [int(t) for t in ids]

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
        """One token of each sequence (device int64 [batch]): logits [batch, vocab].  Or
        several, [batch, n] in order: logits [batch, n, vocab]."""
        page, scale, batch = self.pool.page, self.cfg.head_dim ** -0.5, len(self._lens)
        if not batch:
            raise ValueError("no sequences: start() first")
        several = tokens.dim() == 2 and tokens.shape[0] == batch and tokens.shape[1] > 1
        if tokens.numel() != batch and not several:
            raise ValueError(f"{tokens.numel()} tokens for {batch} sequences")
        T = tokens.shape[1] if several else 1
        if any(n + T > len(row) * page for n, row in zip(self._lens, self._own)):
            raise RuntimeError("no room for another token: start() with more")
        if self.prefix + max(self._lens) + T > self.model.max_len:
            raise ValueError(f"sequences exceed max_len {self.model.max_len}")
        positions = self._ints([self.prefix + n + t for n in self._lens for t in range(T)], torch.int64)
        slots = self._ints([row[j // page] * page + j % page for n, row in zip(self._lens, self._own)
                            for j in range(n, n + T)], torch.int64)
        lens = [n + T for n in self._lens]
        lengths = self._ints(lens)
        starts = self._ints(range(0, batch * T + 1, T)) if several and not self.q4 else None

        def attend(q, *cache):
            own = (*cache, self._prefix_table, self.prefix, self._tables, lengths, scale)
            if self.q4:
                return self.ops.prefix_attention_decode_q4(q, *own)
            if several:
                return self.ops.prefix_attention_prompt(q, starts, *own)
            return self.ops.prefix_attention_decode(q, *own)
        logits = self.model.linears["lm_head"](self._layers(tokens.reshape(-1), positions, slots, attend))
        self._lens = lens                       # nothing failed
        return logits.unflatten(0, (batch, T)) if several else logits

    @torch.no_grad()
    def verify(self, tokens: torch.Tensor, drafts: torch.Tensor, uniforms: torch.Tensor,
               draft_probs: Optional[torch.Tensor] = None, n_drafts: Optional[Sequence[int]] = None,
               temperature: float = 1.0) -> Tuple[torch.Tensor, List[int]]:
        """Runs each sequence's newest token (device int64 [batch]) and the drafts behind it
        ([batch, n], n_drafts of them where given) together, keeps the drafts that the
        probabilities softmax(logits / temperature) and the random numbers (uniforms, float32
        [batch, n + 1] of [0, 1)) accept, and draws the token behind them: (tokens [batch, n +
        1], the drafts that are kept, the drawn one (-1 of logits that are no numbers), then
        -1; their counts).  draft_probs [batch, n, vocab]: what the drafts were drawn from
        (None: they are certain).  The sequences end with the last draft that is kept; the
        drawn token is the newest then, and not run yet."""
        if not temperature > 0:
            raise ValueError(f"a temperature of {temperature}")
        batch, n = len(self._lens), drafts.shape[1] if drafts.dim() == 2 else -1
        if tokens.numel() != batch or drafts.shape[0] != batch or n < 0:
            raise ValueError(f"{tokens.numel()} tokens and drafts {tuple(drafts.shape)} for {batch} sequences")
        if n_drafts is not None and len(n_drafts) != batch:
            raise ValueError(f"{len(n_drafts)} counts of drafts for {batch} sequences")
        before = self._lens
        # a draft that is no token is run as some token; it is not kept
        logits = self.step(torch.cat([tokens.reshape(batch, 1), drafts.clamp(0, self.cfg.vocab - 1)], 1))
        try:
            probs = torch.softmax(logits.float() / temperature, -1).reshape(batch, n + 1, -1)
            out, counts = self.ops.verify_drafts(probs, drafts, draft_probs,
                                                 None if n_drafts is None else self._ints(n_drafts), uniforms)
            kept = counts.tolist()
        except BaseException:
            self._lens = before
            raise
        self._lens = [m + k for m, k in zip(before, kept)]
        return out, kept

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

    @torch.no_grad()
    def sample(self, prompts: Sequence[Sequence[int]], n_new: int, temperature: float = 1.0,
               drafts: int = 0, generator: Optional[torch.Generator] = None) -> List[List[int]]:
        """n_new tokens of each prompt behind the prefix, drawn from softmax(logits /
        temperature) (EOS ignored).  drafts: that many tokens a step at most, those that
        followed the sequence's two newest tokens where they stood last before, are run
        beside the newest one; pages and positions have to suffice for them too, n_new +
        drafts tokens behind each prompt.  generator: of the device's random numbers."""
        if not temperature > 0:
            raise ValueError(f"a temperature of {temperature}")
        if drafts < 0:
            raise ValueError(f"{drafts} drafts")
        if n_new < 1:
            return [[] for _ in prompts]
        # a sequence that is done waits for the others, whose drafts need rows of it too
        logits = self.start(prompts, n_new - 1 + (drafts + 1 if drafts else 0))
        try:
            return self._sample(prompts, logits, n_new, temperature, drafts, generator)
        finally:
            self.release()

    def _sample(self, prompts, logits, n_new, temperature, drafts, generator) -> List[List[int]]:
        batch = len(prompts)

        def uniforms(n):
            return torch.rand(batch, n, generator=generator, device=self.device)
        none = torch.empty(batch, 0, dtype=torch.int64, device=self.device)
        first, _ = self.ops.verify_drafts(torch.softmax(logits.float() / temperature, -1)[:, None], none,
                                          None, None, uniforms(1))
        said = [[t] for t in first[:, 0].tolist()]
        if min(min(new) for new in said) < 0:
            raise RuntimeError("logits that are no numbers")
        texts = [_Text(self._prefix_ids, p) for p in prompts]
        for text, new in zip(texts, said):
            text.add(new)
        while any(len(new) < n_new for new in said):
            guess = [text.guess(min(drafts, n_new - len(new) - 1)) for text, new in zip(texts, said)]
            width = max(map(len, guess))
            out, kept = self.verify(self._ints([new[-1] for new in said], torch.int64),
                                    self._ints([g + [0] * (width - len(g)) for g in guess],
                                               torch.int64).reshape(batch, width),
                                    uniforms(width + 1), None, [len(g) for g in guess], temperature)
            for b, row in enumerate(out.tolist()):
                if min(row[:kept[b]]) < 0:
                    raise RuntimeError("logits that are no numbers")
                if len(said[b]) < n_new:
                    said[b] += row[:kept[b]]
                    texts[b].add(row[:kept[b]])
                else:                                   # done: its token was run for the others' sake
                    self._lens[b] -= kept[b]
        return said


class _Text:
    """A sequence's tokens, and where each pair of neighbours stood last."""

    def __init__(self, *parts: Sequence[int]):
        self.tokens: List[int] = []
        self.after: dict = {}                           # pair -> place behind it
        for p in parts:
            self.add(p)

    def add(self, tokens: Sequence[int]) -> None:
        for t in map(int, tokens):
            n = len(self.tokens)
            if n > 1:                                   # the newest pair is not looked up as itself
                self.after[self.tokens[-2], self.tokens[-1]] = n
            self.tokens.append(t)

    def guess(self, n: int) -> List[int]:
        """At most n tokens that followed the two newest ones before."""
        at = self.after.get(tuple(self.tokens[-2:])) if n > 0 else None
        return self.tokens[at:at + n] if at is not None else []


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
    ap.add_argument("--cache", default="float32", choices=["float32", "bfloat16", "float16", "q4"])
    ap.add_argument("--drafts", type=int, default=0, help="sample with this many drafts a step")
    ap.add_argument("--temperature", type=float, default=0.0, help="above 0: sample")
    a = ap.parse_args()
    syn = synthetic.SyntheticDecoder(a.config, layers=a.layers, log=lambda *x: None)
    c = syn.cfg
    cfg = decoder.DecoderConfig(layers=c["layers"], hidden=c["hidden"], inter=c["inter"], n_q=c["n_q"],
                                n_kv=c["n_kv"], head_dim=c["head_dim"], vocab=c["vocab"])
    tensors = syn.build_fixed(syn.all_linears() + [syn.embed])
    model = decoder.from_synthetic(cfg, tensors, max_len=a.prefix + 256 + a.new + a.drafts + 1)
    rng = random.Random(0)
    prompts = [[rng.randrange(cfg.vocab) for _ in range(rng.randint(1, 256))] for _ in range(a.batch)]
    per = -(-(256 + a.new + a.drafts + 1) // 64)
    dtype = "q4" if a.cache == "q4" else getattr(torch, a.cache)
    batch = BatchDecoder(model, a.batch * per + -(-a.prefix // 64), dtype=dtype)
    batch.set_prefix([rng.randrange(cfg.vocab) for _ in range(a.prefix)])

    def run(n):
        if a.drafts or a.temperature > 0:
            return batch.sample(prompts, n, a.temperature or 1.0, a.drafts)
        return batch.generate(prompts, n)
    run(2)                                              # loads the kernels
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    tokens = run(a.new)
    s = time.perf_counter() - t0
    print(f"{a.batch} prompts of {sum(map(len, prompts))} tokens behind {a.prefix}: "
          f"{a.batch * a.new} tokens in {s:.3f} s ({a.batch * a.new / s:.0f} tokens/s, prompts included)")
    print("first tokens:", [t[:4] for t in tokens])


if __name__ == "__main__":
    main()
