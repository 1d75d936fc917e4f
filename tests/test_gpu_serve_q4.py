"""The 4-bit paged cache on the GPU: paged_append_q4, paged_read_q4 and
prefix_attention_decode_q4 of torch.ops.cbq against their plain float64 forms
(q4_oracle.py derives the tolerances)."""
import pytest
import torch

import q4_oracle as qo
import serve_oracle as so

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(cuda):
    import cbq_ops
    return cbq_ops.load()


# ---- append -------------------------------------------------------------------

def pool(n_pages, n_kv, page, hd, g, rows_first=False):
    """Random bytes as the pool's former content: (codes, pairs) [n_pages, 2, n_kv, page, ..]"""
    lead = (n_pages, 2, page, n_kv) if rows_first else (n_pages, 2, n_kv, page)
    codes = torch.randint(0, 256, (*lead, hd // 2), generator=g, dtype=torch.uint8)
    pairs = torch.randn(*lead, hd // 64, 2, generator=g).bfloat16()
    return [x.transpose(2, 3) if rows_first else x for x in (codes, pairs)]


def split(codes, pairs):
    return codes[:, 0], pairs[:, 0], codes[:, 1], pairs[:, 1]


def on_gpu(x):
    return torch.empty_strided(x.shape, x.stride(), dtype=x.dtype, device="cuda").copy_(x)


@pytest.mark.parametrize("x_type", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("N,n_q,n_kv,hd,page,rot,norm,rows_first,shift", [
    (1, 4, 2, 128, 16, 128, True, False, 0),
    (33, 6, 2, 64, 3, 32, True, True, 0),
    (70, 4, 1, 256, 64, 256, False, False, 0),
    (9, 3, 3, 128, 5, 34, True, False, 0),          # halves that are no whole fours
    (5, 2, 1, 128, 16, 128, True, False, 1),        # q, k, v off alignment: one value at a time
    (4, 1, 1, 64, 1, 2, False, False, 0),
    (19, 2, 1, 256, 7, 200, True, True, 0),
    (300, 8, 4, 64, 32, 64, True, False, 0),
])
def test_append(cuda, ops, x_type, N, n_q, n_kv, hd, page, rot, norm, rows_first, shift):
    """Queries within rounding; codes, scales and mids as the 64-bit form's, every one;
    rows of no token untouched."""
    print(f"append {x_type} N={N} hd={hd} page={page} rot={rot}", flush=True)
    g = torch.Generator().manual_seed(N * hd)
    xt = so.TYPES[x_type]
    n_pages = -(-N // page) + 3
    codes, pairs = pool(n_pages, n_kv, page, hd, g, rows_first)
    dev = [on_gpu(codes), on_gpu(pairs)]
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
    out = ops.paged_append_q4(q, k, v, cos.cuda(), sin.cuda(), positions.cuda(), slots.cuda(),
                              *split(*dev), norm, *[x if x is None else x.cuda() for x in w], eps)
    assert out.dtype == xt and out.is_contiguous()
    yc = wide[:, shift:].unflatten(1, (-1, hd))
    want, mag = so.append_rows(yc[:, :n_q], w[0], cos, sin, positions, norm, eps)
    small = 2.0 ** -25 if xt == torch.float16 else 0.0
    so.near(out, want, so.half_step(xt) * want.abs() + 32 * so.HALF * mag + small, "append q")
    keys, _ = so.append_rows(yc[:, n_q:n_q + n_kv], w[1], cos, sin, positions, norm, eps)
    new = [qo.quantise(x) for x in (keys, yc[:, n_q + n_kv:])]
    for t in range(N):
        p, s = int(positions[t]), int(slots[t])
        if 0 <= p < P and 0 <= s < n_pages * page:
            for i in range(2):
                codes[s // page, i, :, s % page], pairs[s // page, i, :, s % page] = new[i][0][t], new[i][1][t]
    assert torch.equal(dev[0].cpu(), codes), "codes"
    assert torch.equal(dev[1].cpu().view(torch.int16), pairs.view(torch.int16)), "pairs"


def test_append_groups(cuda, ops):
    """Groups at the format's edges, as values (64 bits have no order of sums there):
    constants, zeros, two levels, steps on borders, huge, tiny and mixed magnitudes,
    NaN and infinities beside sound groups."""
    hd, nan, inf = 128, float("nan"), float("inf")
    step = torch.arange(64, dtype=torch.float64)
    groups = [torch.zeros(64), torch.full((64,), 3.7), step % 2, step % 16 - 7.5, (step % 31) / 2 - 7.5,
              step % 15 - 7, 0.125 * (step % 61), 1e30 * (step - 20), 1e-30 * (step - 50), 1e4 + step / 64,
              torch.where(step == 9, 1e6, 1e-3 * step), torch.where(step == 5, nan, step),
              torch.where(step == 63, inf, step), torch.where(step == 0, -inf, step),
              torch.full((64,), 3.4e38), 3.0e38 * (step % 2 * 2 - 1), 1e-41 * step, -step]
    x = torch.stack([torch.cat([a, b]) for a in groups for b in (groups[3], a)]).float()[:, None]
    N = len(x)
    codes = torch.zeros(N, 1, 1, hd // 2, dtype=torch.uint8, device="cuda")
    pairs = torch.zeros(N, 1, 1, 2, 2, dtype=torch.bfloat16, device="cuda")
    pools = codes, pairs, codes.clone(), pairs.clone()
    table = torch.ones(1, 2, device="cuda"), torch.zeros(1, 2, device="cuda")
    i = torch.arange(N, device="cuda")
    d = x.cuda()
    ops.paged_append_q4(d, d, d, *table, i * 0, i, *pools, False, None, None, 0.0)
    c, p = qo.quantise(x)
    finite = x.reshape(N, 2, 64).isfinite().all(-1)
    for what, gc, gp in (("values", pools[2], pools[3]), ("keys", pools[0], pools[1])):
        gc, gp = gc.cpu().reshape(N, 1, -1), gp.cpu().reshape(N, 1, 2, 2)
        if what == "values":
            ok = (gc == c).all(-1).flatten()
            assert ok.all(), f"codes of rows {(~ok).nonzero().flatten().tolist()}"
            assert torch.equal(gp.nan_to_num(7e7), p.nan_to_num(7e7))
        got = qo.values(gc, gp).reshape(N, 2, 64)
        # within half a step, and what the two roundings of the range's ends add
        tol = gp.double()[..., 0].reshape(N, 2, 1) * 0.52
        near = (got - x.double().reshape(N, 2, 64)).abs() <= tol
        sound = finite & (x.reshape(N, 2, 64).abs().amax(-1) < 3.3e38)
        if what == "values":
            assert near[sound].all()
        assert got[~finite].isnan().all()
    k, v = ops.paged_read_q4(*pools, i, torch.float32)
    want = qo.values(c, p).float()
    assert torch.equal(v.cpu().nan_to_num(7e7), want.nan_to_num(7e7))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n_kv,hd,page,rows_first,N", [(2, 128, 16, False, 200), (1, 64, 3, True, 7),
                                                       (3, 256, 64, False, 90), (8, 128, 1, False, 1)])
def test_read(cuda, ops, dtype, n_kv, hd, page, rows_first, N):
    """Any rows in any order, the same one twice, slots that name none."""
    g = torch.Generator().manual_seed(N)
    n_pages = 90 // page + 2
    codes, pairs = pool(n_pages, n_kv, page, hd, g, rows_first)
    slots = torch.randint(0, n_pages * page, (N,), generator=g)
    if N > 4:
        slots[1], slots[3], slots[4] = -1, n_pages * page, slots[0]
    got = ops.paged_read_q4(*split(on_gpu(codes), on_gpu(pairs)), slots.cuda(), so.TYPES[dtype])
    ok = (slots >= 0) & (slots < n_pages * page)
    at = torch.where(ok, slots, 0)
    for i, x in enumerate(got):
        assert x.dtype == so.TYPES[dtype] and x.is_contiguous() and x.shape == (N, n_kv, hd)
        want = qo.values(codes[at // page, i, :, at % page], pairs[at // page, i, :, at % page])
        want = torch.where(ok[:, None, None], want, 0.0)
        assert torch.equal(x.cpu(), want.float().to(so.TYPES[dtype]))


# ---- attention ------------------------------------------------------------------

def decode(ops, batch, q, scale):
    cache, tables = batch.cuda()
    return ops.prefix_attention_decode_q4(q.cuda(), *cache, tables[0], batch.prefix, *tables[1:], scale)


def check(ops, batch, tokens, what, scale=None, q=None):
    scale = batch.hd ** -0.5 if scale is None else scale
    q = batch.queries(tokens, 1.5) if q is None else q
    print(f"decode q4 {what}", flush=True)
    out = decode(ops, batch, q, scale)
    assert out.dtype == batch.dtype and out.is_contiguous()
    want, tol = qo.attend(batch, q, tokens, scale)
    none = want.isnan()                                 # a row that sees NaN, and only such a row
    got = out.double().cpu()
    assert torch.equal(got.isnan(), none)
    got, want, tol = (x.masked_fill(none, 0.0) for x in (got, want, tol))
    so.near(got, want, tol, what)
    worst = float(((got - want).abs() / tol.clamp(min=1e-30)).max())
    print(f"  largest error {worst:.2f} of its tolerance", flush=True)
    return out


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("lens,prefix,n_kv,rep,page,tokens,rows_first,room", [
    ([1], 0, 1, 1, 16, 1, False, 0),
    ([40, 1, 0, 97, 33], 0, 2, 4, 16, 1, False, 1),
    ([5, 64, 31], 70, 2, 3, 3, 1, True, 2),
    ([90, 7, 12], 33, 1, 7, 17, 4, False, 1),           # 28 rows a sequence
    ([3, 1, 40], 5, 2, 12, 64, 3, False, 0),            # 36 rows; lengths below the tokens'
    ([700, 0, 2], 0, 2, 2, 16, 1, False, 30),           # parts, some of them empty
    ([130, 600, 31, 5], 900, 1, 4, 32, 2, False, 3),    # parts of prefix and own keys
])
def test_decode(cuda, ops, dtype, hd, lens, prefix, n_kv, rep, page, tokens, rows_first, room):
    batch = qo.Batch(lens, prefix, n_kv, rep, hd, page, dtype, rows_first, room, seed=len(lens) + hd)
    check(ops, batch, tokens, f"{dtype} hd={hd} {lens} behind {prefix}, {tokens} tokens")


def test_decode_many_rows(cuda, ops):
    """Prefix rows past one, two and four tiles, and a last tile that is part full."""
    for n, rep, tokens in ((5, 5, 1), (9, 6, 1), (11, 4, 2), (37, 4, 1)):
        for dtype, hd in (("bf16", 128), ("f16", 64), ("f32", 256), ("bf16", 256)):
            batch = qo.Batch([i * 7 % 50 for i in range(n)], 700, 1, rep, hd, 16, dtype, seed=n)
            check(ops, batch, tokens, f"{dtype} hd={hd} {n} sequences of {rep} heads, {tokens} tokens")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0, 1e-45, 1e-30])
def test_scales(cuda, ops, dtype, scale):
    batch = qo.Batch([50, 3, 90], 40, 2, 2, 64, 16, dtype, seed=3)
    factor = 1e29 if scale == 1e-30 else 1.0
    q = batch.queries(1, factor)
    check(ops, batch, 1, f"{dtype} scale {scale}", scale, q)


def test_offsets(cuda, ops):
    """Keys and values whose middle is far from 0, and large scores."""
    for dtype in ("f32", "bf16", "f16"):
        batch = qo.Batch([60, 200], 100, 1, 4, 128, 16, dtype, seed=8, offset=5.0)
        check(ops, batch, 2, f"{dtype} offset", q=batch.queries(2, 6.0))


def test_lengths_and_pages_out_of_range(cuda, ops):
    """A length counts inside 0 .. its row's capacity; a page outside the pool hides its
    keys; a sequence that sees nothing gets zeros."""
    batch = qo.Batch([40, 50, 60, 30, 20, 600], 100, 2, 3, 64, 16, "f32", room=2, seed=5)
    n = batch.codes.shape[0]
    batch.tables[1, 1] = n
    batch.tables[2, :] = -7
    batch.tables[5, 3:30] = 1 << 30
    batch.prefix_table[2] = -1
    batch.lengths[0] = -4
    batch.lengths[3] = 1 << 30                          # the unused pages are -1
    check(ops, batch, 1, "out of range")
    check(ops, batch, 3, "out of range, three tokens")
    lone = qo.Batch([0, 20, 900], 0, 1, 2, 128, 16, "bf16", seed=6)
    lone.tables[1, :] = -1
    lone.tables[2, :] = -1
    out = check(ops, lone, 2, "nothing to see")
    assert not out.any()


def test_hidden_nan(cuda, ops):
    """What a token does not see may be NaN: keys of later tokens, rows behind the
    length; one that it sees reaches its own rows and heads alone."""
    tokens = 4
    for dtype in ("f32", "bf16"):
        batch = qo.Batch([70, 33, 4], 40, 2, 2, 64, 16, dtype, seed=9)
        q = batch.queries(tokens, 1.5)
        clean = decode(ops, batch, q, 0.125)
        for b, last in enumerate((69, 32, 3)):          # the newest key, of both kinds
            p, r = int(batch.tables[b, last // 16]), last % 16
            batch.pairs[p, b % 2, 0, r] = float("nan")
        out = decode(ops, batch, q, 0.125).reshape(3, tokens, 2, 2, 64)
        clean = clean.reshape(out.shape)
        assert torch.equal(out[:, :, 1], clean[:, :, 1])            # the other kv head
        assert torch.equal(out[:, :-1], clean[:, :-1])              # tokens before the newest
        assert out[:, -1, 0].isnan().all()


def test_queries(cuda, ops):
    """Strided and unaligned queries; one that is not finite is its own row's matter."""
    batch = qo.Batch([50, 80], 40, 2, 2, 128, 16, "bf16", seed=10)
    q = batch.queries(1)
    cache, tables = batch.cuda()
    want = decode(ops, batch, q, 0.1)
    wide = torch.zeros(2, 4, 200, dtype=torch.bfloat16, device="cuda")
    wide[:, :, 1:129] = q.cuda()
    turned = q.cuda().permute(2, 0, 1).contiguous().permute(1, 2, 0)
    for x in (wide[:, :, 1:129], turned):
        got = ops.prefix_attention_decode_q4(x, *cache, tables[0], batch.prefix, *tables[1:], 0.1)
        assert torch.equal(got, want)
    for bad in (float("nan"), float("inf"), -float("inf")):
        x = q.clone()
        x[1, 2, 77] = bad
        got = decode(ops, batch, x, 0.1)
        assert got[1, 2].isnan().all()
        got[1, 2] = want[1, 2]
        assert torch.equal(got, want)


def test_empty(cuda, ops):
    batch = qo.Batch([5, 9], 0, 1, 2, 64, 16, "f32", seed=1)
    cache, (pt, tables, lengths) = batch.cuda()
    q = torch.zeros(0, 2, 64, device="cuda")
    assert ops.prefix_attention_decode_q4(q, *cache, pt, 0, tables[:0], lengths[:0], 1.0).shape == (0, 2, 64)
    assert ops.prefix_attention_decode_q4(q, *cache, pt, 0, tables, lengths, 1.0).shape == (0, 2, 64)
    none = torch.zeros(2, 0, dtype=torch.int32, device="cuda")
    got = ops.prefix_attention_decode_q4(torch.ones(2, 2, 64, device="cuda"), *cache, pt, 0, none, lengths, 1.0)
    assert not got.any()
    k, v = ops.paged_read_q4(*cache, torch.zeros(0, dtype=torch.int64, device="cuda"), torch.float32)
    assert k.shape == v.shape == (0, 1, 64)
