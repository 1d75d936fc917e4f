"""BatchDecoder over the 4-bit cache, its steps of several tokens, its verification of
drafts and its sampling, on the compressed weights of a small model."""
import types

import numpy as np
import pytest
import torch

import decoder
import synthetic
from batch_decoder import BatchDecoder
from conftest import rel_l2

pytestmark = pytest.mark.gpu

CFG = decoder.DecoderConfig(layers=2, hidden=256, inter=512, n_q=4, n_kv=2, head_dim=64, vocab=1024)


def _ids(n, seed):
    return [int(t) for t in np.random.default_rng(seed).integers(0, CFG.vocab, n)]


@pytest.fixture(scope="module")
def model(cuda):
    comp = synthetic.compress_model_cpu(CFG, 11, "fixed")
    return decoder.from_compressed(CFG, comp, device=cuda, max_len=256)


def err(got, want):
    return rel_l2(got.float().cpu().numpy(), want.float().cpu().numpy())


def watched(batch):
    """batch, whose attention over the 4-bit cache is compared at every call with the one
    over the cache's values in fp32: the same sums in another order, rel-L2 <= 1e-5."""
    ops, pool, seen = batch.ops, batch.pool, []

    def attend(q, kc, kp, vc, vp, prefix_table, prefix, tables, lengths, scale):
        out = ops.prefix_attention_decode_q4(q, kc, kp, vc, vp, prefix_table, prefix, tables, lengths, scale)
        every = torch.arange(pool.pages.shape[1] * pool.page, device=q.device)
        k, v = (x.unflatten(0, (-1, pool.page)).transpose(1, 2)
                for x in ops.paged_read_q4(kc, kp, vc, vp, every, torch.float32))
        B = lengths.shape[0]
        starts = torch.arange(0, len(q) + 1, len(q) // B, dtype=torch.int32, device=q.device)
        want = ops.prefix_attention_prompt(q, starts, k, v, prefix_table, prefix, tables, lengths, scale)
        seen.append(err(out, want))
        assert seen[-1] <= 1e-5
        return out
    names = ("paged_append_q4", "paged_read_q4", "prefix_attention_prompt", "verify_drafts")
    batch.ops = types.SimpleNamespace(prefix_attention_decode_q4=attend, **{n: getattr(ops, n) for n in names})
    return seen


@pytest.mark.parametrize("prefix,lens,page", [(0, [9], 16), (0, [5, 40, 1], 16), (70, [33, 2, 8, 17], 64),
                                              (16, [1, 1], 3)])
def test_q4_cache(cuda, model, prefix, lens, page):
    """Every attention within the order of its sums.  Against the fp32 cache: a group's
    values lie 7.5 steps around its middle and are off by half a step at most, by the
    square root of a twelfth of one otherwise, a tenth of a key or value for normal ones:
    scores of about 1 by a tenth too, and two layers' outputs by less than 0.3."""
    shared, prompts = _ids(prefix, 1), [_ids(n, 2 + i) for i, n in enumerate(lens)]
    steps = [torch.tensor(_ids(len(lens), 50 + i), device=cuda) for i in range(2)]
    several = torch.tensor(_ids(3 * len(lens), 60), device=cuda).reshape(len(lens), 3)
    out = []
    for dtype in (torch.float32, "q4"):
        batch = BatchDecoder(model, n_pages=200, page=page, dtype=dtype)
        seen = watched(batch) if dtype == "q4" else []
        batch.set_prefix(shared)
        out.append([batch.start(prompts, 5)] + [batch.step(s) for s in steps] + [batch.step(several)])
    assert len(seen) == 3 * CFG.layers
    for i, (want, got) in enumerate(zip(*out)):
        assert got.shape == want.shape
        print(f"prefix {prefix}, {lens}, step {i}: rel-L2 {err(got, want):.1e} against fp32", flush=True)
        assert err(got, want) < 0.3


@pytest.mark.parametrize("dtype,bar", [(torch.float32, 1e-5), (torch.bfloat16, 3e-2)])
def test_several_tokens(cuda, model, dtype, bar):
    """Logits of four tokens at once and one by one: sums in another order, 16-bit
    roundings of the weights as they fall (ten half steps)."""
    prompts, steps = [_ids(20, 3), _ids(5, 4)], torch.tensor(_ids(8, 5), device=cuda).reshape(2, 4)
    batch = BatchDecoder(model, n_pages=40, page=16, dtype=dtype)
    batch.set_prefix(_ids(30, 1))
    batch.start(prompts, 4)
    want = torch.stack([batch.step(steps[:, t]) for t in range(4)], 1)
    batch.start(prompts, 4)
    got = batch.step(steps)
    print(f"{dtype}: rel-L2 {err(got, want):.1e}", flush=True)
    assert got.shape == (2, 4, CFG.vocab) and err(got, want) <= bar


def test_certain_tokens_are_greedy(cuda, model):
    """At a temperature where the likeliest token has all the probability, sampling is
    generate(), with drafts or without; pages come back."""
    batch = BatchDecoder(model, n_pages=40, page=16)
    prompts = [_ids(6, 7) * 3, _ids(11, 8)]
    batch.set_prefix(_ids(20, 9))
    want = batch.generate(prompts, 24)
    for drafts in (0, 3):
        assert batch.sample(prompts, 24, temperature=1e-5, drafts=drafts) == want
        assert len(batch.pool._free) == 38


@pytest.mark.parametrize("dtype", [torch.float32, "q4"], ids=str)
def test_verify(cuda, model, dtype):
    """Greedy tokens as drafts are kept, others end the run; the next step goes on from
    what was kept."""
    batch = BatchDecoder(model, n_pages=40, page=16, dtype=dtype)
    prompts = [_ids(9, 7), _ids(30, 8), _ids(3, 9)]
    batch.set_prefix(_ids(20, 9))
    first = batch.start(prompts, 12).argmax(-1)
    said = [first]
    for _ in range(6):
        said.append(batch.step(said[-1]).argmax(-1))
    said = torch.stack(said, 1)
    batch.start(prompts, 12)
    drafts = said[:, 1:5].clone()
    drafts[1, 2] = (drafts[1, 2] + 1) % CFG.vocab
    u = torch.full((3, 5), 0.5, device=cuda)
    out, kept = batch.verify(first, drafts, u, n_drafts=[4, 4, 1], temperature=1e-5)
    assert kept == [5, 3, 2] and batch._lens == [9 + 5, 30 + 3, 3 + 2]
    want = said[:, 1:6].clone()
    for b, n in enumerate(kept):
        want[b, n:] = -1
    assert torch.equal(out, want)
    newest = out.gather(1, torch.tensor(kept, device=cuda)[:, None] - 1)[:, 0]
    step = batch.step(newest).argmax(-1)
    assert step[1:].tolist() == [int(said[1, 4]), int(said[2, 3])] and int(step[0]) == int(said[0, 6])


def test_sample(cuda, model):
    """Reproduced by its generator's seed; every token is one of the vocabulary."""
    batch = BatchDecoder(model, n_pages=40, page=16, dtype="q4")
    prompts = [_ids(6, 7) * 3, _ids(11, 8)]
    runs = [batch.sample(prompts, 30, 0.9, 4, torch.Generator("cuda").manual_seed(s)) for s in (1, 1, 2)]
    assert runs[0] == runs[1] != runs[2]
    assert all(len(x) == 30 and 0 <= min(x) and max(x) < CFG.vocab for run in runs for x in run)
    assert len(batch.pool._free) == 40
