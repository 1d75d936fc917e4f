"""The checks of the attention over the 4-bit cache (q4_checks.py) on the CPU: they pass
outputs that are rounded once, and none where keys are lost or count twice."""
import pytest
import torch

import q4_checks as qc
import q4_oracle as qo

SHAPES = [([40, 3, 17], 1601, 2, 11, 128, 16, 3), ([1, 70], 1500, 2, 5, 256, 32, 1),
          ([130, 600, 31, 5], 900, 1, 4, 64, 32, 2), ([900, 31], 0, 2, 4, 64, 16, 1)]


def fails(check, *args):
    try:
        check(*args, "planted")
    except AssertionError:
        return True
    return False


@pytest.fixture(scope="module", params=[(s, t) for s in SHAPES for t in ("bf16", "f16", "f32")],
                ids=lambda p: f"{p[1]}-{p[0][1]}-{p[0][4]}")
def case(request):
    (lens, prefix, n_kv, rep, hd, page, tokens), dtype = request.param
    batch = qo.Batch(lens, prefix, n_kv, rep, hd, page, dtype, seed=hd + prefix)
    return batch, tokens, hd ** -0.5


def test_exact(case):
    """The same sums as q4_oracle's."""
    batch, tokens, scale = case
    q = batch.queries(tokens, 1.5)
    want, _ = qo.attend(batch, q, tokens, scale)
    assert ((qc.exact(batch, q, tokens, scale) - want).abs() <= 1e-12).all()


def test_rows(case):
    batch, tokens, scale = case
    q = batch.queries(tokens, 1.5)
    want, bar = qc.exact(batch, q, tokens, scale), qc.bound(batch)
    assert not fails(qc.near_rows, want.to(batch.dtype), want, bar)
    assert fails(qc.near_rows, torch.zeros_like(want), want, bar)
    n = batch.prefix + max(batch.lens)
    for first in (0, 32, batch.prefix // 32 * 32):              # a tile that is lost, or counts twice
        for times in (0.0, 2.0):
            count = torch.ones(n)
            count[first:first + 32] = times
            got = qc.exact(batch, q, tokens, scale, count).to(batch.dtype)
            assert fails(qc.near_rows, got, want, bar), (first, times)


def test_single_keys(case):
    """Each border's key: of the prefix's ends, of tiles' ends, and the first and last own one."""
    batch, tokens, scale = case
    q, two = qc.planted(batch, tokens, scale)
    want = qc.exact(batch, q, tokens, scale)
    assert not fails(qc.near_planted, want.to(batch.dtype), want, two, batch)
    assert fails(qc.near_planted, torch.zeros_like(want), want, two, batch)
    weights = 0
    for j in sorted({0, 31, 32, batch.prefix - 1, batch.prefix} & set(range(batch.prefix + max(batch.lens)))):
        for times in (0.0, 2.0):
            count = torch.ones(batch.prefix + max(batch.lens))
            count[j] = times
            got = qc.exact(batch, q, tokens, scale, count)
            moved = (got - want).norm(dim=-1) > 0.1 * (two[0] - two[1]).norm(dim=-1) + 1e-9
            weights += int(moved.sum())
            if bool(moved.any()):                               # a row has that key
                assert fails(qc.near_planted, got.to(batch.dtype), want, two, batch), (j, times)
    assert weights > 0


def test_borders():
    assert sorted(qc.borders(1)) == [0] and sorted(qc.borders(33)) == [0, 1, 31, 32]
    assert sorted(qc.borders(100)) == [0, 1, 31, 32, 33, 63, 64, 65, 95, 96, 97, 99]
