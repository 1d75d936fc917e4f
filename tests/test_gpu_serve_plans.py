"""Every kernel that the paged attention's plans choose, against the float64 form
(serve_oracle.py): hidden pages, rows that the causal mask cuts, values that are not
finite.  tests/test_serve_plans.py checks that the shapes get the kernels they are for."""
import pytest
import torch

import serve_oracle as so
import serve_shapes as sh
from serve_oracle import Batch
from test_gpu_serve import check_decode, decode, ops, prompt, starts  # noqa: F401

pytestmark = pytest.mark.gpu

TYPES = {2: ("bf16", "f16"), 4: ("f32",)}


@pytest.mark.parametrize("dtype,hd,runs,prefix,n_kv,rep,room", [
    (t, shape[0], *shape[2:7]) for shape in sh.PROMPTS for t in TYPES[shape[1]]])
def test_prompts(cuda, ops, dtype, hd, runs, prefix, n_kv, rep, room):
    """A page of the prefix and one of the first run's own are not there; then an
    infinite value of the last run reaches the tokens from its own on, none before."""
    b = Batch(runs, prefix, n_kv, rep, hd, sh.PAGE, dtype, seed=hd + len(runs), room=room)
    b.prefix_table[1] = b.tables[0, 0] = -1
    q, q_start, scale = b.queries(sum(runs), 1.5), starts(runs), hd ** -0.5
    what = f"prompt {dtype} hd={hd} runs={runs} prefix={prefix} heads={n_kv}x{rep} room={room}"
    print(what, flush=True)
    want, tol = so.attend_prompt(b, q, q_start, scale)
    got = prompt(ops, b, q, q_start, scale)
    so.near(got, want, tol, what)
    assert torch.equal(got, prompt(ops, b, q, q_start, scale))
    n, h, d = runs[-1], n_kv - 1, hd - 3
    at = n // 2 if len(runs) > 1 else max(n // 2, sh.PAGE)       # of a page that is there
    b.v[int(b.tables[-1, at // sh.PAGE]), h, at % sh.PAGE, d] = -float("inf")
    got = prompt(ops, b, q, q_start, scale).cpu()
    hit = torch.zeros(got.shape, dtype=torch.bool)
    hit[sum(runs) - n + at:, h * rep:, d] = True
    assert (got[hit] == -float("inf")).all() and got[~hit].isfinite().all()
    so.near(got[~hit], want[~hit], tol[~hit], "beside an infinite value, " + what)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("dtype,lens,prefix,rep,room", [
    (t, *shape[1:5]) for shape in sh.DECODES for t in TYPES[shape[0]]])
def test_decodes(cuda, ops, dtype, hd, lens, prefix, rep, room):
    """Pages of the prefix and of own keys that are not there, and a sequence whose
    own are all so: what its parts left is not read."""
    b = Batch(lens, prefix, 2, rep, hd, sh.PAGE, dtype, seed=hd + len(lens), room=room)
    what = f"{dtype} hd={hd} {len(lens)} sequences prefix={prefix} room={room}"
    print("decode " + what, flush=True)
    b.prefix_table[1] = 1 << 30
    if prefix > 1000:
        b.prefix_table[20:40] = -1
    if max(lens) > 40:
        b.tables[lens.index(max(lens)), 2:9] = -1
        b.tables[-1] = -1
    q = b.queries(len(lens), 1.5)
    out = check_decode(ops, b, what, q=q)
    assert torch.equal(out, decode(ops, b, q, hd ** -0.5))


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("dtype,lens,prefix,rep,room", [
    (t, *shape[1:5]) for shape in sh.JOINTS + sh.MERGES for t in TYPES[shape[0]]])
def test_large_batches(cuda, ops, dtype, hd, lens, prefix, rep, room):
    """Few keys, in one walk and in parts, and many rows of many parts; of a large
    batch some sequences."""
    b = Batch(lens, prefix, 2, rep, hd, sh.PAGE, dtype, seed=hd + len(lens), room=room)
    b.tables[-1] = -1
    q, what = b.queries(len(lens), 1.5), f"{dtype} hd={hd} {len(lens)} sequences prefix={prefix}"
    print("large batch " + what, flush=True)
    out = decode(ops, b, q, hd ** -0.5)
    some = sorted({*range(min(9, len(lens))), len(lens) // 2, *range(max(len(lens) - 9, 0), len(lens))})
    b.lens, b.tables, b.lengths = [lens[i] for i in some], b.tables[some], b.lengths[some]
    so.near(out[some], *so.attend(b, q[some], starts([1] * len(some)), hd ** -0.5), what)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_hidden_parts(cuda, ops, dtype, hd):
    """Several parts of everything, nothing there: zeros."""
    b = Batch([700, 3, 1500], 1100, 2, 8, hd, sh.PAGE, dtype, seed=7)
    b.prefix_table[:] = -1
    b.tables[1:] = -1
    out = check_decode(ops, b, f"hidden parts {dtype} hd={hd}")
    assert out[0].any() and not out[1:].any()
