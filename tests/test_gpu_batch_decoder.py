"""BatchDecoder (batched greedy decoding over the paged cache) against the
one-sequence decoder on the same compressed weights: logits of the prompts and
of the steps, tokens, page accounting."""
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


@pytest.fixture(scope="module", params=["fixed", "huffman"])
def model(cuda, request):
    comp = synthetic.compress_model_cpu(CFG, 11, request.param)
    return decoder.from_compressed(CFG, comp, device=cuda, max_len=256)


@pytest.mark.parametrize("prefix,lens,page", [(0, [9], 16), (0, [5, 40, 1], 16), (70, [33, 2, 8, 17], 64),
                                              (16, [1, 1], 3)])
def test_logits_equal_one_by_one(cuda, model, prefix, lens, page):
    """Three steps behind each prompt, fp32 cache: rel-L2 <= 1e-5 against the
    one-sequence decoder, as its prompt against its single steps."""
    shared, prompts = _ids(prefix, 1), [_ids(n, 2 + i) for i, n in enumerate(lens)]
    steps = [_ids(len(lens), 50 + i) for i in range(3)]
    batch = BatchDecoder(model, n_pages=200, page=page)
    batch.set_prefix(shared)
    got = [batch.start(prompts, 3)] + [batch.step(torch.tensor(s, device=cuda)) for s in steps]
    for b, p in enumerate(prompts):
        model.reset()
        want = [model.forward(torch.tensor(shared + p))]
        want += [model.forward(torch.tensor([s[b]])) for s in steps]
        for i, (x, y) in enumerate(zip(got, want)):
            e = rel_l2(x[b].cpu().numpy(), y.cpu().numpy())
            print(f"prefix {prefix}, sequence {b} of {lens}, step {i}: rel-L2 {e:.1e}", flush=True)
            assert e <= 1e-5


@pytest.mark.parametrize("dtype,bar", [(torch.bfloat16, 3e-2), (torch.float16, 4e-3)])
def test_sixteen_bit_cache(cuda, model, dtype, bar):
    """Queries, keys, values, weights and outputs rounded to half a step each
    (2^-9 of the largest in bf16, 2^-12 in fp16) in two layers: within ten half
    steps of the fp32 cache."""
    shared, prompts = _ids(30, 1), [_ids(12, 2), _ids(41, 3)]
    out = []
    for t in (torch.float32, dtype):
        batch = BatchDecoder(model, n_pages=32, page=16, dtype=t)
        batch.set_prefix(shared)
        out.append(batch.start(prompts, 1).cpu().numpy())
    e = rel_l2(out[1], out[0])
    print(f"{dtype}: rel-L2 {e:.1e}", flush=True)
    assert e <= bar


def test_tokens_and_pages(cuda, model):
    """Greedy tokens as one by one, on a second batch and prefix too, and every
    page comes back."""
    batch = BatchDecoder(model, n_pages=24, page=16)
    for prefix, lens in ((40, [7, 30, 12]), (0, [20, 3]), (33, [5])):
        shared, prompts = _ids(prefix, prefix), [_ids(n, 9 + n) for n in lens]
        batch.set_prefix(shared)
        got = batch.generate(prompts, 10)
        assert got == [model.generate(shared + p, 10) for p in prompts]
        assert len(batch.pool._free) == 24 - -(-prefix // 16)


def test_refusals(cuda, model):
    batch = BatchDecoder(model, n_pages=6, page=16)
    batch.set_prefix(_ids(20, 1))
    with pytest.raises(RuntimeError, match="pages"):
        batch.start([_ids(30, 1), _ids(30, 2)], 16)             # 2 x 3 pages, 4 free
    assert len(batch.pool._free) == 4
    with pytest.raises(ValueError, match="token"):
        batch.start([_ids(3, 1), []], 1)
    with pytest.raises(ValueError, match="max_len"):
        batch.start([_ids(3, 1)], 250)
    with pytest.raises(ValueError, match="max_len"):
        batch.set_prefix(_ids(300, 1))
    batch.start([_ids(15, 1)], 1)
    batch.step(torch.tensor([3], device=cuda))
    with pytest.raises(RuntimeError, match="room"):
        batch.step(torch.tensor([3], device=cuda))
