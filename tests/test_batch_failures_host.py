"""BatchDecoder when a step or a call fails, on the CPU (test_batch_sampling_host.py's
model): sequences and pages as before."""
import pytest
import torch

from test_batch_sampling_host import VOCAB, Batch, Model


@pytest.fixture(params=[torch.float32, "q4"], ids=str)
def batch(request):
    return Batch(Model(64 if request.param == "q4" else 4), n_pages=40, page=4, dtype=request.param)


def test_head_fails(batch):
    """A step whose head raises leaves the lengths: no unverified draft is kept, and the
    same step is run again from the same positions."""
    t, d, u = torch.tensor([6, 4]), torch.tensor([[7, 8, 9], [5, 9, 1]]), torch.full((2, 4), 0.5)
    batch.start([[5], [2, 3]], 8)
    head = batch.model.linears["lm_head"]

    def broken(x):
        raise RuntimeError("no memory for the logits")
    for call in (lambda: batch.verify(t, d, u), lambda: batch.step(t),
                 lambda: batch.step(torch.cat([t[:, None], d], 1))):
        batch.model.linears["lm_head"] = broken
        with pytest.raises(RuntimeError, match="no memory"):
            call()
        assert batch._lens == [1, 2]
        batch.model.linears["lm_head"] = head
    out, kept = batch.verify(t, d, u)
    assert out.tolist() == [[7, 8, 9, 10], [5, 6, -1, -1]] and kept == [4, 2]
    assert batch._lens == [5, 4] and batch.runs[-1] == batch.runs[1]


def test_refused_sample(batch):
    """A sample() that is refused leaves the sequences that were started, as generate()
    does; one that fails later gives its pages back."""
    batch.start([[5], [2, 3]], 8)
    own, free = [list(r) for r in batch._own], len(batch.pool._free)
    for call in (lambda: batch.generate([[1]], 61), lambda: batch.sample([[1]], 61),
                 lambda: batch.sample([[1]], 50, drafts=40), lambda: batch.sample([], 3),
                 lambda: batch.sample([[1], []], 3), lambda: batch.sample([[1]], 3, temperature=0.0)):
        with pytest.raises(ValueError):
            call()
        assert batch._own == own and batch._lens == [1, 2] and len(batch.pool._free) == free
    assert batch.step(torch.tensor([6, 4])).argmax(-1).tolist() == [7, 5]

    def broken(*args):
        raise RuntimeError("not verified")
    batch.ops.verify_drafts = broken
    with pytest.raises(RuntimeError, match="not verified"):
        batch.sample([[1]], 3)
    assert len(batch.pool._free) == 40 and not batch._own
