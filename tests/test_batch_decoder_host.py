"""BatchDecoder's bookkeeping on the CPU: tokens, pages and refusals, with layers that
pass each token's id on and a head that picks the next one."""
import pytest
import torch

import decoder
from batch_decoder import BatchDecoder

CFG = decoder.DecoderConfig(layers=1, hidden=8, inter=8, n_q=2, n_kv=1, head_dim=4, vocab=50)


class Model:
    cfg, device, max_len = CFG, torch.device("cpu"), 40
    linears = {"lm_head": lambda x: torch.nn.functional.one_hot((x[:, 0].long() + 1) % CFG.vocab,
                                                                CFG.vocab).float()}


class Batch(BatchDecoder):
    fail = False

    def _layers(self, ids, positions, slots, attend):
        if self.fail:
            raise RuntimeError("no layers")
        assert positions.shape == slots.shape == ids.shape
        assert int(positions.max()) < self.model.max_len
        assert 0 <= int(slots.min()) and int(slots.max()) < self.pool.pages.shape[1] * self.pool.page
        self.written = slots.tolist()
        return ids[:, None].float()


@pytest.fixture
def batch():
    return Batch(Model(), n_pages=6, page=4)


def free(batch):
    return len(batch.pool._free)


def test_no_new_tokens(batch):
    """As the one-sequence decoder: none asked for, none given."""
    assert batch.generate([[1, 2], [3]], 0) == [[], []]
    assert batch.generate([[1, 2], [3]], 1) == [[3], [4]]
    assert batch.generate([[1, 2], [3]], 3) == [[3, 4, 5], [4, 5, 6]] and free(batch) == 6


def test_last_position(batch):
    """The last new token is not run: a prompt and its tokens may pass max_len and the
    pages by it, as one by one."""
    batch.set_prefix(list(range(20)))                           # 5 of 6 pages
    assert batch.generate([[7, 8]], 3) == [[9, 10, 11]]         # 2 + 2 rows: the last page
    assert max(batch.written) < 24
    with pytest.raises(RuntimeError, match="pages"):
        batch.generate([[7, 8]], 4)
    batch.set_prefix([])
    long = Batch(Model(), n_pages=10, page=4)
    assert long.generate([[1] * 30], 11) == [list(range(2, 13))]
    with pytest.raises(ValueError, match="max_len"):
        long.generate([[1] * 30], 12)


def test_failures_lose_no_pages(batch):
    batch.set_prefix([1, 2, 3, 4, 5])
    batch.fail = True
    with pytest.raises(RuntimeError, match="no layers"):
        batch.start([[1, 2, 3]], 4)
    assert free(batch) == 4                                     # the prefix stays
    with pytest.raises(RuntimeError, match="no layers"):
        batch.generate([[1, 2, 3]], 4)
    assert free(batch) == 4
    with pytest.raises(RuntimeError, match="no layers"):
        batch.set_prefix([1, 2, 3])
    assert free(batch) == 6 and batch.prefix == 0               # as without a prefix
    batch.fail = False
    with pytest.raises(RuntimeError, match="pages"):
        batch.set_prefix(list(range(30)))
    assert free(batch) == 6 and batch.generate([[1]], 2) == [[2, 3]]
    batch.set_prefix([1, 2, 3])
    batch.start([[1, 2, 3]], 4)
    batch.fail = True
    with pytest.raises(RuntimeError, match="no layers"):        # a step that failed is none
        batch.step(torch.tensor([7]))
    batch.fail = False
    batch.step(torch.tensor([7]))
    row = batch._own[0]
    assert batch.written == [row[0] * 4 + 3]
    batch.release()
    batch.set_prefix([])
    assert sorted(batch.pool._free) == list(range(6))


def test_refusals(batch):
    for call in (lambda: batch.step(torch.tensor([1])),         # nothing was started
                 lambda: batch.start([[1, 2]], -1), lambda: batch.start([], 1)):
        with pytest.raises(ValueError):
            call()
    batch.start([[1, 2], [3]], 2)
    with pytest.raises(ValueError, match="2 sequences"):
        batch.step(torch.tensor([1]))
    with pytest.raises(ValueError, match="2 sequences"):
        batch.step(torch.tensor([1, 2, 3]))
    assert batch._lens == [2, 1]
    batch.step(torch.tensor([1, 2]))
    batch.step(torch.tensor([1, 2]))
    assert batch._lens == [4, 3]
    with pytest.raises(RuntimeError, match="room"):
        batch.step(torch.tensor([1, 2]))
    batch.release()
    with pytest.raises(ValueError, match="start"):
        batch.step(torch.tensor([1, 2]))
    with pytest.raises(ValueError, match="page"):
        Batch(Model(), n_pages=4, page=0)
