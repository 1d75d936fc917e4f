"""BatchDecoder's steps of several tokens, its verification of drafts and its sampling on
the CPU: tokens, rows and refusals, with layers that pass each token's id on, a head that
makes the next one certain, and the plain form of the verification."""
import types

import pytest
import torch

import decoder
import q4_oracle as qo
from batch_decoder import BatchDecoder, _Text

VOCAB = 50


def cfg(head_dim):
    return decoder.DecoderConfig(layers=1, hidden=8, inter=8, n_q=2, n_kv=1, head_dim=head_dim, vocab=VOCAB)


class Model:
    device, max_len, period = torch.device("cpu"), 60, VOCAB

    def __init__(self, head_dim=4):
        self.cfg = cfg(head_dim)
        self.linears = {"lm_head": self.head}

    def head(self, x):
        """The next token is this one and one, the smallest behind the largest."""
        return torch.where(torch.arange(VOCAB) == (x[:, :1].long() + 1) % self.period, 0.0, -float("inf"))


class Batch(BatchDecoder):
    def __init__(self, *args, **kw):
        super().__init__(*args, **kw)
        self.ops = types.SimpleNamespace(verify_drafts=qo.verify)
        self.runs = []

    def _layers(self, ids, positions, slots, attend):
        assert ids.dim() == 1 and positions.shape == slots.shape == ids.shape
        assert int(ids.min()) >= 0 and int(ids.max()) < VOCAB
        assert int(positions.max()) < self.model.max_len
        assert len(set(slots.tolist())) == len(slots)               # a row of its own each
        rows = [r * self.pool.page + i for own in self._own for r in own for i in range(self.pool.page)]
        assert set(slots.tolist()) <= set(rows) or not rows          # (none: the prefix)
        self.runs.append((ids.tolist(), positions.tolist(), slots.tolist()))
        return ids[:, None].float()


@pytest.fixture(params=[torch.float32, "q4"], ids=str)
def batch(request):
    return Batch(Model(64 if request.param == "q4" else 4), n_pages=40, page=4, dtype=request.param)


def test_several_tokens(batch):
    """Logits, rows and positions of several tokens are those of one by one."""
    tokens = torch.tensor([[7, 9, 3], [1, 1, 4]])
    batch.start([[5, 6], [2, 3, 4, 8]], 4)
    one = torch.stack([batch.step(tokens[:, t]) for t in range(3)], 1)
    runs = batch.runs[1:]
    batch.release()
    batch.start([[5, 6], [2, 3, 4, 8]], 4)
    at, batch.runs = batch._own, []
    assert torch.equal(batch.step(tokens), one) and batch._lens == [5, 7]
    ids, positions, slots = batch.runs[0]
    assert ids == tokens.flatten().tolist()
    assert positions == [r[1][b] for b in range(2) for r in runs] == [2, 3, 4, 4, 5, 6]
    assert slots == [at[b][j // 4] * 4 + j % 4 for b, n in enumerate((2, 4)) for j in range(n, n + 3)]
    with pytest.raises(RuntimeError, match="room"):
        batch.step(tokens)
    assert batch._lens == [5, 7]
    batch.step(torch.tensor([[1], [2]]))                            # one a sequence, as a column
    assert batch._lens == [6, 8]


def test_verify(batch):
    """Drafts that follow are kept; the sequences end with them."""
    batch.start([[5], [2, 3], [9]], 8)
    out, kept = batch.verify(torch.tensor([6, 4, 10]), torch.tensor([[7, 8], [5, 9], [3, 12]]),
                             torch.full((3, 3), 0.5))
    assert out.tolist() == [[7, 8, 9], [5, 6, -1], [11, -1, -1]] and kept == [3, 2, 1]
    assert batch._lens == [4, 4, 2]
    newest = out.gather(1, torch.tensor(kept)[:, None] - 1)[:, 0]
    out, kept = batch.verify(newest, torch.tensor([[10, -1], [7, 8], [99, -7]]), torch.zeros(3, 3),
                             n_drafts=[1, 0, 2])
    assert out.tolist() == [[10, 11, -1], [7, -1, -1], [12, -1, -1]] and kept == [2, 1, 1]
    assert batch._lens == [6, 5, 3] and batch.runs[-1][1] == [4, 5, 6, 4, 5, 6, 2, 3, 4]
    out, kept = batch.verify(out.gather(1, torch.tensor(kept)[:, None] - 1)[:, 0],
                             torch.empty(3, 0, dtype=torch.int64), torch.zeros(3, 1))
    assert out.tolist() == [[12], [8], [13]] and batch._lens == [7, 6, 4]


def test_verify_refusals(batch):
    t, d, u = torch.tensor([1, 2]), torch.tensor([[1], [2]]), torch.zeros(2, 2)
    with pytest.raises(ValueError):
        batch.verify(t, d, u)                                       # nothing was started
    batch.start([[5], [6]], 4)
    for call in (lambda: batch.verify(t, d, u, temperature=0.0), lambda: batch.verify(t[:1], d, u),
                 lambda: batch.verify(t, d[:1], u), lambda: batch.verify(t, t, u),
                 lambda: batch.verify(t, d, u, n_drafts=[1]), lambda: batch.sample([[1]], 3, drafts=-1),
                 lambda: batch.verify(t, d, u, temperature=float("nan")),
                 lambda: batch.sample([[1]], 3, temperature=-1.0)):
        with pytest.raises(ValueError):
            call()

    def broken(*args):
        raise RuntimeError("not verified")
    batch.ops.verify_drafts = broken
    with pytest.raises(RuntimeError, match="not verified"):
        batch.verify(t, d, u)
    assert batch._lens == [1, 1]                                    # as before


@pytest.mark.parametrize("drafts", [0, 1, 4, 9])
def test_sample(batch, drafts):
    """Tokens that repeat are found and kept; every sequence gets its tokens; rows and
    pages suffice and come back."""
    batch.model.period = 5
    batch.set_prefix([0, 1, 2])
    batch.runs = []
    said = batch.sample([[3, 4, 0, 1], [7]], 14, drafts=drafts)
    assert said == [[(2 + i) % 5 for i in range(14)], [(8 + i) % 5 if i else 3 for i in range(14)]]
    assert len(batch.runs) == 14 if drafts == 0 else len(batch.runs) < 14
    assert len(batch.pool._free) == 39 and not batch._own
    assert batch.sample([[3]], 0) == [[]] and batch.sample([[3]], 1, drafts=drafts) == [[4]]


def test_sample_room():
    """As tight as the pool can be: prompts, new tokens, drafts."""
    batch = Batch(Model(), n_pages=32, page=1)
    batch.model.period = 3
    assert batch.sample([[0, 1, 2, 0], [7]], 8, drafts=5) == [[1, 2, 0, 1, 2, 0, 1, 2],
                                                              [2, 0, 1, 2, 0, 1, 2, 0]]
    with pytest.raises(RuntimeError, match="pages"):
        batch.sample([[0, 1, 2, 0], [7, 8]], 8, drafts=6)
    assert len(batch.pool._free) == 32


def test_sample_without_numbers(batch):
    batch.model.linears["lm_head"] = lambda x: torch.full((len(x), VOCAB), float("nan"))
    with pytest.raises(RuntimeError, match="no numbers"):
        batch.sample([[1, 2]], 4)
    assert len(batch.pool._free) == 40 and not batch._own
    assert batch.generate([[1]], 0) == [[]]


def test_text():
    text = _Text([1, 2, 3], [1, 2])
    assert text.guess(2) == [3, 1] and text.guess(9) == [3, 1, 2] and text.guess(0) == []
    text.add([4, 1, 2])
    assert text.guess(3) == [4, 1, 2]
    text.add([5])
    assert text.guess(3) == [] and _Text([1]).guess(3) == [] and _Text([], []).guess(1) == []


def test_q4_pool():
    for head_dim in (4, 96, 512):
        with pytest.raises(ValueError, match="q4"):
            Batch(Model(head_dim), n_pages=2, page=4, dtype="q4")
    with pytest.raises(ValueError, match="q5"):
        Batch(Model(64), n_pages=2, page=4, dtype="q5")
    kc, kp, vc, vp = Batch(Model(128), n_pages=2, page=4, dtype="q4").pool.layer(0)
    assert kc.shape == vc.shape == (2, 1, 4, 64) and kp.shape == vp.shape == (2, 1, 4, 2, 2)
    assert kc.dtype == torch.uint8 and kp.dtype == torch.bfloat16 and kc.stride() == vc.stride()
