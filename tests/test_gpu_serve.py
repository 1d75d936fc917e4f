"""Batched serving on the GPU: paged_append, prefix_attention_decode and
prefix_attention_prompt of torch.ops.cbq against their plain float64 forms
(serve_oracle.py derives the tolerances)."""
import pytest
import torch

import serve_oracle as so
from serve_oracle import Batch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(cuda):
    import cbq_ops
    return cbq_ops.load()


def starts(runs):
    return torch.tensor([0] + list(runs), dtype=torch.int64).cumsum(0).to(torch.int32)


def decode(ops, batch, q, scale):
    k, v, prefix_table, tables, lengths = batch.cuda()
    return ops.prefix_attention_decode(q.cuda(), k, v, prefix_table, batch.prefix, tables, lengths,
                                       scale)


def prompt(ops, batch, q, q_start, scale):
    k, v, prefix_table, tables, lengths = batch.cuda()
    return ops.prefix_attention_prompt(q.cuda(), q_start.cuda(), k, v, prefix_table, batch.prefix,
                                       tables, lengths, scale)


def check_decode(ops, batch, what, scale=None, q=None):
    scale = batch.hd ** -0.5 if scale is None else scale
    q = batch.queries(len(batch.lens), 1.5) if q is None else q
    print(f"decode {what}", flush=True)
    out = decode(ops, batch, q, scale)
    assert out.dtype == batch.dtype
    so.near(out, *so.attend(batch, q, starts([1] * len(batch.lens)), scale), what)
    return out


def check_prompt(ops, batch, runs, what, scale=None):
    scale = batch.hd ** -0.5 if scale is None else scale
    q, q_start = batch.queries(sum(runs), 1.5), starts(runs)
    print(f"prompt {what}", flush=True)
    out = prompt(ops, batch, q, q_start, scale)
    assert out.dtype == batch.dtype
    so.near(out, *so.attend(batch, q, q_start, scale), what)
    return out


# ---- append -------------------------------------------------------------------

@pytest.mark.parametrize("x_type,c_type", [("f32", "f32"), ("f32", "bf16"), ("f32", "f16"),
                                           ("bf16", "bf16"), ("f16", "f16")])
@pytest.mark.parametrize("N,n_q,n_kv,hd,page,rot,norm,rows_first,shift", [
    (1, 4, 2, 128, 16, 128, True, False, 0),
    (33, 6, 2, 64, 3, 32, True, True, 0),
    (70, 4, 1, 256, 64, 256, False, False, 0),
    (9, 3, 3, 100, 5, 34, True, False, 0),          # one value at a time
    (5, 2, 1, 128, 16, 128, True, False, 1),        # q, k, v off 16-byte alignment
    (4, 1, 1, 2, 1, 2, False, False, 0),
    (3, 2, 1, 254, 7, 2, True, True, 0),
])
def test_append(cuda, ops, x_type, c_type, N, n_q, n_kv, hd, page, rot, norm, rows_first, shift):
    print(f"append {x_type} {c_type} N={N} hd={hd} page={page} rot={rot}", flush=True)
    g = torch.Generator().manual_seed(N * hd)
    xt, ct = so.TYPES[x_type], so.TYPES[c_type]
    n_pages = -(-N // page) + 3
    shape = (n_pages, 2, page, n_kv, hd) if rows_first else (n_pages, 2, n_kv, page, hd)
    pages = torch.randn(shape, generator=g).to(ct).cuda()
    pages = pages.transpose(2, 3) if rows_first else pages
    before = pages.double().cpu()
    wide = torch.randn(N, (n_q + 2 * n_kv) * hd + shift, generator=g).to(xt)
    y = wide.cuda()[:, shift:].unflatten(1, (-1, hd))           # cut from one stacked product
    q, k, v = y[:, :n_q], y[:, n_q:n_q + n_kv], y[:, n_q + n_kv:]
    P = 50
    angles = torch.rand(P, rot // 2, generator=g, dtype=torch.float64) * 100
    cos, sin = (torch.cat([t, t], 1).float() for t in (angles.cos(), angles.sin()))
    positions = torch.randint(0, P, (N,), generator=g)
    slots = torch.randperm(n_pages * page, generator=g)[:N]
    if N > 4:                                                   # tokens that store nothing
        positions[1], positions[2], slots[3], slots[4] = -1, P, -1, n_pages * page
    w = [1 + 0.1 * torch.randn(hd, generator=g) for _ in range(2)] if norm and N != 33 else [None] * 2
    eps = 1e-6
    out = ops.paged_append(q, k, v, cos.cuda(), sin.cuda(), positions.cuda(), slots.cuda(),
                           pages[:, 0], pages[:, 1], norm, *[x if x is None else x.cuda() for x in w],
                           eps)
    assert out.dtype == ct and out.is_contiguous()
    small = 2.0 ** -25 if ct == torch.float16 else 0.0          # half of fp16's smallest step
    yc = wide[:, shift:].unflatten(1, (-1, hd))
    for what, x, wt, got in (("q", yc[:, :n_q], w[0], out), ("k", yc[:, n_q:n_q + n_kv], w[1], None)):
        want, mag = so.append_rows(x, wt, cos, sin, positions, norm, eps)
        tol = so.half_step(ct) * want.abs() + 32 * so.HALF * mag + small
        if what == "q":
            so.near(got, want, tol, "append q")
        else:
            keys, key_tol = want, tol
    after, want = pages.double().cpu(), before.clone()
    tol = torch.zeros_like(want)
    for t in range(N):
        p, s = int(positions[t]), int(slots[t])
        if not 0 <= p < P or not 0 <= s < n_pages * page:
            continue
        want[s // page, 0, :, s % page], tol[s // page, 0, :, s % page] = keys[t], key_tol[t]
        want[s // page, 1, :, s % page] = yc[t, n_q + n_kv:].to(ct).double()
    so.near(after, want, tol, "append pages")


def test_append_nothing(cuda, ops):
    pages = torch.zeros(2, 2, 1, 16, 64, device=cuda)
    z = torch.zeros(0, 1, 64, device=cuda)
    i = torch.zeros(0, dtype=torch.int64, device=cuda)
    t = torch.zeros(4, 64, device=cuda)
    out = ops.paged_append(z, z, z, t, t, i, i, pages[:, 0], pages[:, 1], False, None, None, 0.0)
    assert out.shape == (0, 1, 64) and not pages.any()


# ---- one token a sequence -------------------------------------------------------

@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("lens,prefix,n_kv,rep,page", [
    ([1], 0, 1, 1, 16),
    ([0, 1, 16, 17, 0, 300], 0, 2, 4, 16),          # sequences that see nothing
    ([0, 5, 700], 1, 1, 16, 3),                     # 48 prefix rows, pages end inside a tile
    ([33, 0], 129, 2, 5, 64),                       # 10 prefix rows
    ([1, 2, 3] * 11, 400, 1, 3, 128),               # 99 prefix rows
    ([40], 1000, 1, 33, 256),                       # three 16-row tiles of one token's heads
])
def test_decode(cuda, ops, dtype, hd, lens, prefix, n_kv, rep, page):
    check_decode(ops, Batch(lens, prefix, n_kv, rep, hd, page, dtype, rows_first=page == 3,
                            seed=hd + len(lens)), f"{dtype} hd={hd} {lens[:6]} prefix={prefix}")


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_decode_long(cuda, ops, dtype, hd):
    """Several own parts a sequence, of very different lengths, and many of the prefix."""
    check_decode(ops, Batch([2500, 3, 1111], 2049, 1, 6, hd, 32, dtype, seed=5, room=9),
                 f"long {dtype} hd={hd}")


# ---- runs of new tokens -----------------------------------------------------------

@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("runs,past,prefix,n_kv,rep,page", [
    ([1], 0, 0, 1, 1, 16),
    ([1, 0, 2, 17, 5], 40, 0, 2, 4, 16),            # an empty run
    ([130, 1, 63], 3, 77, 1, 3, 3),
    ([3, 1, 4], 900, 300, 1, 4, 64),                # few rows, many keys: parts
    ([260], 0, 0, 1, 2, 128),
    ([65, 64], 513, 129, 1, 1, 17),
])
def test_prompt(cuda, ops, dtype, hd, runs, past, prefix, n_kv, rep, page):
    b = Batch([past + n for n in runs], prefix, n_kv, rep, hd, page, dtype, rows_first=page == 3,
              seed=hd + len(runs))
    check_prompt(ops, b, runs, f"{dtype} hd={hd} runs={runs} past={past} prefix={prefix}")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("page", [1, 300, 4096])
def test_pages_of_any_size(cuda, ops, dtype, page):
    b = Batch([70, 1, 333], 401, 1, 4, 64, page, dtype, seed=page)
    check_decode(ops, b, f"page {page}")
    check_prompt(ops, b, [30, 1, 90], f"page {page}")


@pytest.mark.parametrize("n_kv,rep", [(1, 1), (8, 4)])
def test_many_sequences(cuda, ops, n_kv, rep):
    """More runs than a wave has lanes, empty ones among them."""
    rng = torch.Generator().manual_seed(2)
    runs = [int(x) for x in torch.randint(0, 7, (150,), generator=rng)]
    b = Batch([n + 3 for n in runs], 20, n_kv, rep, 64, 16, "bf16", seed=21)
    check_prompt(ops, b, runs, "150 runs")
    check_decode(ops, b, "150 sequences")


def test_nothing_of_one_kind(cuda, ops):
    """Tables without pages, no tokens, no sequences."""
    b = Batch([0, 0], 33, 1, 2, 64, 16, "bf16", seed=22, room=0)
    assert b.tables.shape == (2, 0)
    check_decode(ops, b, "the prefix alone")
    b2 = Batch([0, 0], 900, 2, 20, 64, 16, "bf16", seed=22, room=0)
    check_decode(ops, b2, "a long prefix alone")
    k, v, prefix_table, tables, lengths = b.cuda()
    q = b.queries(5).cuda()
    none = torch.zeros(0, dtype=torch.int32, device=cuda)
    out = ops.prefix_attention_prompt(q, none.new_zeros(1), k, v, prefix_table, 33, tables[:0], none, 0.1)
    assert out.shape == q.shape and not out.any()
    for x in (ops.prefix_attention_decode(q[:0], k, v, prefix_table, 33, tables[:0], none, 0.1),
              ops.prefix_attention_prompt(q[:0], none.new_zeros(3), k, v, prefix_table, 33, tables,
                                          lengths, 0.1)):
        assert x.shape == (0, 2, 64)
    out = decode(ops, Batch([0], 0, 1, 2, 64, 16, "f32", room=0), torch.ones(1, 2, 64), 0.1)
    assert not out.any()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rep", [4, 7])
def test_prompt_many_rows(cuda, ops, dtype, rep):
    """Enough rows for the widest tiles: whole and part-full ones, masks that
    begin inside a tile."""
    runs = [300, 45, 129]
    b = Batch([n + 10 for n in runs], 70, 8, rep, 64, 16, dtype, seed=rep)
    check_prompt(ops, b, runs, f"many rows {dtype} rep={rep}")


# Prompts of a block or less a CU: two streams of keys a block (the plan of each is
# checked by tests/native/cbq_paged_host.cpp).
STREAMS = [
    ([191], 100, 500, 8, 8, 64, 64),
    ([191], 100, 500, 8, 8, 128, 64),
    ([191], 100, 500, 8, 8, 256, 64),
    ([84, 67, 0], 10, 1900, 8, 16, 64, 17),
    ([84, 67, 0], 10, 1900, 8, 16, 128, 17),
]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("runs,past,prefix,n_kv,rep,hd,page", STREAMS)
def test_prompt_streams(cuda, ops, dtype, runs, past, prefix, n_kv, rep, hd, page):
    """With a page of the prefix and one of the first run's own that are not there."""
    b = Batch([past + n for n in runs], prefix, n_kv, rep, hd, page, dtype, seed=hd)
    b.prefix_table[3] = -1
    b.tables[0, 1] = 1 << 30
    q, q_start = b.queries(sum(runs), 2.0), starts(runs)
    want, tol = so.attend_prompt(b, q, q_start, hd ** -0.5)
    first = prompt(ops, b, q, q_start, hd ** -0.5)
    so.near(first, want, tol, f"streams {dtype} hd={hd} {runs}")
    assert torch.equal(first, prompt(ops, b, q, q_start, hd ** -0.5))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("at", [101, 200, 290])
def test_prompt_streams_values_not_finite(cuda, ops, dtype, at):
    """An infinite value of an own key reaches the tokens from it on, none before."""
    runs, past, prefix, n_kv, rep, hd, page = STREAMS[1]
    b = Batch([past + n for n in runs], prefix, n_kv, rep, hd, page, dtype, seed=at)
    q, q_start = b.queries(sum(runs)), starts(runs)
    want, tol = so.attend_prompt(b, q, q_start, hd ** -0.5)
    b.v[int(b.tables[0, at // page]), 2, at % page, 7] = float("inf")
    got = prompt(ops, b, q, q_start, hd ** -0.5).cpu()
    hit = torch.zeros(got.shape, dtype=torch.bool)
    hit[at - past:, 2 * rep:3 * rep, 7] = True
    assert (got[hit] == float("inf")).all() and got[~hit].isfinite().all()
    so.near(got[~hit], want[~hit], tol[~hit], f"beside an infinite value {dtype}")


@pytest.mark.parametrize("prefix", [0, 20])
def test_prompt_rows_without_keys(cuda, ops, prefix):
    """Fewer own keys than tokens: the first tokens see the prefix alone, or nothing."""
    runs = [40, 90]
    b = Batch([10, 0], prefix, 2, 2, 64, 16, "bf16", seed=3)
    out = check_prompt(ops, b, runs, f"rows without keys, prefix={prefix}")
    if prefix == 0:
        assert not out[:30].any() and not out[40:].any()


@pytest.mark.parametrize("n", [40, 2000])
def test_prompt_tokens_of_no_run(cuda, ops, n):
    b = Batch([n // 2], 0, 1, 1, 64, 16, "f32", seed=4)
    q = b.queries(n)
    q_start = torch.tensor([3, 3 + n // 2], dtype=torch.int32)
    out = prompt(ops, b, q, q_start, 0.125)
    so.near(out, *so.attend(b, q, q_start, 0.125), "tokens of no run")
    assert not out[:3].any() and not out[3 + n // 2:].any()


def test_prompt_one_token_runs_are_decode(cuda, ops):
    b = Batch([5, 300, 70], 100, 2, 4, 128, 16, "f32", seed=6)
    q = b.queries(3)
    x, y = decode(ops, b, q, 0.1), prompt(ops, b, q, starts([1, 1, 1]), 0.1)
    want, tol = so.attend(b, q, starts([1, 1, 1]), 0.1)
    so.near(x, want, tol, "decode")
    so.near(y, want, tol, "prompt")


# ---- masks, hidden pages, values that are not numbers -------------------------------

@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("bad", [-1, 1 << 30, -(1 << 31)])
def test_hidden_pages(cuda, ops, dtype, bad):
    """Table entries outside the pool hide their keys, in the prefix too; a
    sequence of hidden pages alone gets zeros."""
    b = Batch([100, 33, 400], 90, 2, 3, 64, 16, dtype, seed=8)
    b.prefix_table[2] = bad
    b.tables[0, 1] = b.tables[2, 0] = b.tables[2, 24] = bad
    check_decode(ops, b, f"hidden pages {dtype}")
    check_prompt(ops, b, [20, 33, 150], f"hidden pages {dtype}")
    b.prefix_table[:] = bad
    b.tables[1] = bad
    out = check_decode(ops, b, f"all hidden {dtype}")
    assert not out[1].any()


def test_lengths_out_of_range(cuda, ops):
    """Below 0 as 0, above the table as what it names."""
    b = Batch([64, 64, 64], 0, 1, 2, 64, 16, "bf16", room=0, seed=9)
    q = b.queries(3)
    want, tol = so.attend(b, q, starts([1] * 3), 0.125)
    b.lengths[0], b.lengths[2] = -7, 1 << 30
    got = decode(ops, b, q, 0.125)
    want[0], tol[0] = 0, 0
    so.near(got, want, tol, "lengths out of range")


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("scale", [-0.2, 0.0, 1e-38, 3.0])
def test_scale(cuda, ops, dtype, scale):
    b = Batch([50, 200], 30, 1, 4, 64, 16, dtype, seed=10)
    check_decode(ops, b, f"scale {scale}", scale)
    check_prompt(ops, b, [50, 20], f"scale {scale}", scale)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_large_scores(cuda, ops, dtype):
    """Scores in the hundreds, of either sign: one key takes all the weight."""
    b = Batch([300, 40], 200, 1, 2, 64, 16, dtype, seed=11, scale_k=30.0)
    check_decode(ops, b, f"large scores {dtype}")
    check_prompt(ops, b, [40, 40], f"large scores {dtype}")


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_not_numbers_stay_in_their_rows(cuda, ops, dtype):
    """A query of NaN touches its own outputs only; a key of NaN the queries that see it."""
    b = Batch([90, 70], 0, 1, 2, 64, 16, dtype, seed=12)
    q = b.queries(120)
    q_start = starts([60, 60])
    want, tol = so.attend(b, q, q_start, 0.125)
    q[7, 1, 5] = float("nan")
    k = b.k.clone()
    b.k[int(b.tables[1, 3]), :, 2] = float("nan")               # own key 50 of sequence 1
    out = prompt(ops, b, q, q_start, 0.125).double().cpu()
    b.k.copy_(k)
    nan = torch.zeros(120, 2, dtype=torch.bool)
    nan[7, 1] = True
    nan[60 + 40:] = True                                        # tokens at own position 50 and later
    assert torch.equal(out.isnan().any(-1), nan) and torch.equal(out.isnan().all(-1), nan)
    so.near(out[~nan], want[~nan], tol[~nan], "beside NaN")


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("hd,runs,past,n_kv,rep", [
    (64, [60, 60], 10, 1, 2),                                   # 16 rows a block
    (128, [60, 60], 10, 1, 2),
    (256, [40, 33], 3, 2, 1),
    (64, [12] * 30, 7, 8, 4),                                   # 64 rows a block
    (128, [12] * 30, 7, 8, 4),
    (256, [12] * 30, 7, 8, 4),
    (64, [300, 129], 20, 8, 4),                                 # the widest
    (128, [300, 129], 20, 8, 4),
    (256, [300, 129], 20, 8, 4),
    (64, [30, 40], 3000, 1, 4),                                 # keys in parts
    (128, [3, 5], 2500, 1, 2),
])
def test_values_not_finite(cuda, ops, dtype, hd, runs, past, n_kv, rep):
    """Infinite values and NaN among the own keys: tokens before them keep their
    outputs, tokens from them on get inf or NaN in the same places."""
    b = Batch([past + n for n in runs], 0, n_kv, rep, hd, 16, dtype, seed=hd)
    inf, nan = float("inf"), float("nan")
    for i, (d, x) in enumerate([(3, inf), (17, -inf), (40, nan), (40, inf), (63, inf), (63, -inf)]):
        j = past + 4 + 3 * (i // 2) - i % 2                     # keys of the last run, two side by side
        p, r = int(b.tables[-1, j // 16]), j % 16
        b.v[p, :, r, d] = x
    for h, j in ((0, past + runs[0] // 2), (n_kv - 1, past + runs[0] - 1)):
        b.v[int(b.tables[0, j // 16]), h, j % 16, hd - 1] = nan if h else -inf
    q, q_start = b.queries(sum(runs), 1.5), starts(runs)
    print(f"values not finite {dtype} hd={hd} runs={runs[:3]}", flush=True)
    got = prompt(ops, b, q, q_start, hd ** -0.5).double().cpu()
    want, tol = so.attend(b, q, q_start, hd ** -0.5)
    odd = ~want.isfinite()
    assert odd.any() and not odd.all()
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got[want.isinf()], want[want.isinf()])
    so.near(got[~odd], want[~odd], tol[~odd], "beside them")


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_nan_queries_without_keys(cuda, ops, dtype):
    """A query of NaN that sees no key gets zeros as any other: hidden pages, no
    keys, tokens before the first own key."""
    b = Batch([40, 0, 40], 0, 2, 2, 64, 16, dtype, seed=20)
    b.tables[0] = -1
    q = torch.full((3, 4, 64), float("nan"), dtype=b.dtype)
    out = decode(ops, b, q, 0.125)
    assert not out[:2].any() and out[2].isnan().all()
    b.lengths[2] = 5
    out = prompt(ops, b, q.repeat(10, 1, 1), starts([10, 10, 10]), 0.125)
    assert not out[:25].any() and out[25:].isnan().all()


@pytest.mark.parametrize("parts", [False, True])
def test_all_scores_nan(cuda, ops, parts):
    b = Batch([3000 if parts else 20], 0, 1, 1, 64, 16, "f32", seed=13)
    b.k.fill_(float("nan"))
    assert decode(ops, b, b.queries(1), 0.125).isnan().all()


# ---- strides, streams, graphs, far offsets -------------------------------------------

@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_strides(cuda, ops, dtype):
    """Queries cut from a wider product, off alignment, and out of order; a table
    cut from a wider one."""
    b = Batch([30, 77], 20, 2, 2, 64, 16, dtype, seed=14)
    q = b.queries(2)
    k, v, prefix_table, tables, lengths = b.cuda()
    want, tol = so.attend(b, q, starts([1, 1]), 0.125)
    wide = torch.full((2, 3 * 4 * 64 + 8), float("nan"), dtype=b.dtype, device=cuda)
    wide[:, 8:8 + 256] = q.cuda().flatten(1)
    odd = torch.zeros(2, 257, dtype=b.dtype, device=cuda)
    odd[:, 1:] = q.cuda().flatten(1)
    big = torch.full((2, tables.shape[1] + 5), 1 << 30, dtype=torch.int32, device=cuda)
    big[:, 2:2 + tables.shape[1]] = tables
    cut = big[:, 2:2 + tables.shape[1]]
    for x in (wide[:, 8:8 + 256].unflatten(1, (4, 64)), odd[:, 1:].unflatten(1, (4, 64)),
              q.cuda().transpose(1, 2).contiguous().transpose(1, 2),
              q.cuda().transpose(0, 1).contiguous().transpose(0, 1)):
        so.near(ops.prefix_attention_decode(x, k, v, prefix_table, 20, cut, lengths, 0.125), want, tol,
                "strides")


def test_separate_pools(cuda, ops):
    """Keys and values in tensors of their own, in different layouts."""
    b = Batch([30, 77], 20, 2, 2, 128, 16, "bf16", seed=15)
    q = b.queries(2)
    k, v, prefix_table, tables, lengths = b.cuda()
    v = v.transpose(1, 2).contiguous().transpose(1, 2)
    want, tol = so.attend(b, q, starts([1, 1]), 0.1)
    so.near(ops.prefix_attention_decode(q.cuda(), k.contiguous(), v, prefix_table, 20, tables, lengths,
                                        0.1), want, tol, "separate pools")


def test_other_stream(cuda, ops):
    b = Batch([900, 77, 5], 300, 2, 2, 128, 16, "bf16", seed=16)
    q = b.queries(3)
    want, tol = so.attend(b, q, starts([1] * 3), 0.1)
    k, v, prefix_table, tables, lengths = b.cuda()
    qd = q.cuda()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        outs = [ops.prefix_attention_decode(qd, k, v, prefix_table, 300, tables, lengths, 0.1)
                for _ in range(4)]
    torch.cuda.current_stream().wait_stream(s)
    for out in outs:
        so.near(out, want, tol, "other stream")
        assert torch.equal(out, outs[0])                        # the same call, the same bits


def test_graph(cuda, ops):
    """A step of append and attention captured once: lengths, positions, slots
    and queries change between replays."""
    b = Batch([40, 500], 64, 2, 4, 64, 16, "bf16", seed=17, room=3, fill=0.0)
    k, v, prefix_table, tables, lengths = b.cuda()
    B, hd = 2, 64
    pos, slot = (torch.zeros(B, dtype=torch.int64, device=cuda) for _ in range(2))
    x = torch.zeros(B, (b.n_q + 4) * hd, dtype=b.dtype, device=cuda).unflatten(1, (-1, hd))
    angles = torch.arange(1000)[:, None] * 0.1 ** torch.linspace(0, 4, hd // 2)
    cos, sin = (torch.cat([t, t], 1).float().cuda() for t in (angles.cos(), angles.sin()))
    # rows for the new tokens in each sequence's own tail
    free = sorted(set(range(b.k.shape[0])) - set(b.prefix_table.tolist()) - set(b.tables.flatten().tolist()))
    for i, page in enumerate(free[:2]):
        row = b.tables[i].tolist()
        tables[i, row.index(-1)] = b.tables[i, row.index(-1)] = page

    def step():
        y = ops.paged_append(x[:, :b.n_q], x[:, b.n_q:b.n_q + 2], x[:, b.n_q + 2:], cos, sin, pos, slot,
                             k, v, True, None, None, 1e-6)
        return ops.prefix_attention_decode(y, k, v, prefix_table, 64, tables, lengths, hd ** -0.5), y

    slot.fill_(-1)
    step()                                                      # loads the code
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, y = step()
    g = torch.Generator().manual_seed(1)
    for i in range(4):
        at = [n + i for n in b.lens]
        x.copy_(torch.randn(x.shape, generator=g).to(b.dtype))
        lengths.copy_(torch.tensor([n + 1 for n in at], dtype=torch.int32))
        pos.copy_(torch.tensor([64 + n for n in at]))
        slot.copy_(torch.tensor([int(b.tables[s, n // 16]) * 16 + n % 16 for s, n in enumerate(at)]))
        graph.replay()
        torch.cuda.synchronize()
        got, turned = out.clone(), y.clone()
        eager, turned2 = step()
        assert torch.equal(turned, turned2) and torch.equal(got, eager)
        b.k.copy_(k.cpu())
        b.v.copy_(v.cpu())
        b.lengths = lengths.cpu()
        so.near(got, *so.attend(b, turned.cpu(), starts([1, 1]), hd ** -0.5), f"replay {i}")


def test_far_pages(cuda, ops):
    """Pages whose offsets pass 2^32 bytes and 2^31 elements."""
    b = Batch([100, 37], 50, 1, 2, 64, 16, "bf16", seed=18)
    n = b.k.shape[0]
    per = 2 * 16 * 64
    far = (2 ** 31 + 2 ** 20) // per                            # 2^31 elements, 4 GiB
    pool = torch.empty(far + n, 2, 1, 16, 64, dtype=b.dtype, device=cuda)
    pool[far:, 0], pool[far:, 1] = b.k.cuda(), b.v.cuda()
    b.prefix_table += far
    b.tables[b.tables >= 0] += far
    q = b.queries(2)
    got = ops.prefix_attention_decode(q.cuda(), pool[:, 0], pool[:, 1], b.prefix_table.cuda(), 50,
                                      b.tables.cuda(), b.lengths.cuda(), 0.125)
    tail = torch.tensor([(far + n) * 16 - 1], device=cuda)
    one = torch.ones(1, 1, 64, dtype=b.dtype, device=cuda)
    t = torch.ones(1, 64, device=cuda)
    ops.paged_append(one, one, one, t, 0 * t, torch.zeros(1, dtype=torch.int64, device=cuda), tail,
                     pool[:, 0], pool[:, 1], False, None, None, 0.0)
    assert (pool[-1, :, 0, 15] == 1).all()
    b.prefix_table -= far
    b.tables[b.tables >= 0] -= far
    so.near(got, *so.attend(b, q, starts([1, 1]), 0.125), "far pages")


# ---- refusals ---------------------------------------------------------------------

def test_refusals(cuda, ops):
    b = Batch([30, 77], 20, 2, 2, 64, 16, "bf16", seed=19)
    k, v, prefix_table, tables, lengths = b.cuda()
    q = b.queries(2).cuda()
    good = dict(q=q, k=k, v=v, pt=prefix_table, p=20, t=tables, n=lengths, s=0.125)

    def call(**kw):
        a = dict(good, **kw)
        return ops.prefix_attention_decode(a["q"], a["k"], a["v"], a["pt"], a["p"], a["t"], a["n"],
                                           a["s"])
    assert call().shape == (2, 4, 64)
    for kw, text in [
            (dict(q=q.float()), "pages' type"), (dict(q=q[:, :3]), "heads of"),
            (dict(q=q[..., :32]), "heads of"), (dict(q=q[:1]), "one token a sequence"),
            (dict(q=q[0]), "device tensor"), (dict(k=k[:1]), "one shape"),
            (dict(v=v.float()), "one type"), (dict(k=k[:0], v=v[:0]), "empty"),
            (dict(k=k[..., :32], v=v[..., :32]), "hd must be"),
            (dict(k=k.transpose(2, 3), v=v.transpose(2, 3)), "last dimension"),
            (dict(pt=prefix_table[:1]), "names 1 pages"), (dict(p=-1), "prefix_table names"),
            (dict(p=33), "prefix_table names"), (dict(t=tables[:1]), "batch"),
            (dict(t=tables.long()), "tables must be"), (dict(n=lengths.long()), "lengths must be"),
            (dict(n=lengths.cpu()), "is on cpu"), (dict(s=float("nan")), "scale"),
            (dict(s=float("inf")), "scale")]:
        with pytest.raises(RuntimeError, match=text):
            call(**kw)
    odd = torch.zeros(k.numel() + 1, dtype=k.dtype, device=cuda)[1:].view(k.shape)
    with pytest.raises(RuntimeError, match="16-byte aligned"):
        call(k=odd)
    with pytest.raises(RuntimeError, match="q_start"):
        ops.prefix_attention_prompt(q, lengths, k, v, prefix_table, 20, tables, lengths, 0.125)

    x = torch.zeros(2, 4, 64, device=cuda)
    kv = x[:, :2]
    tab = torch.zeros(8, 64, device=cuda)
    at = torch.zeros(2, dtype=torch.int64, device=cuda)
    w = torch.ones(64, device=cuda)
    good = dict(q=x, k=kv, v=kv, c=tab, s=tab, p=at, l=at, kp=k, vp=v, n=True, qw=w, kw=w, e=1e-6)

    def add(**kw):
        a = dict(good, **kw)
        return ops.paged_append(*a.values())
    kept = k.clone()
    for kw, text in [
            (dict(k=x), "k must be"), (dict(v=kv.bfloat16()), "q's type"),
            (dict(q=x.half(), k=kv.half(), v=kv.half()), "own type"), (dict(q=x.double()), "float32"),
            (dict(c=tab[:, :32]), "one shape"), (dict(c=tab[:, :0], s=tab[:, :0]), "width"),
            (dict(c=tab[:, :33].contiguous(), s=tab[:, :33].contiguous()), "even width"),
            (dict(p=at[:1]), "one a token"), (dict(l=at.int()), "slots must be"),
            (dict(n=False), "without the norm"), (dict(qw=w[:32]), "q_weight"),
            (dict(e=float("nan")), "eps"), (dict(e=-1.0), "eps"), (dict(s=tab.cpu()), "is on cpu")]:
        with pytest.raises(RuntimeError, match=text):
            add(**kw)
    assert torch.equal(kept, k) or (kept.isnan() == k.isnan()).all()
