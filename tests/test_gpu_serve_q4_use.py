"""The 4-bit paged cache and the verification of drafts in use, on the GPU: prefixes that
many rows share, pages far apart, other streams, captured steps replayed, refusals."""
import pytest
import torch

import q4_oracle as qo
import serve_oracle as so
from test_gpu_serve_q4 import check, decode

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(cuda):
    import cbq_ops
    return cbq_ops.load()


# ---- many tokens: several heads a thread ----------------------------------------------

@pytest.mark.parametrize("dtype,hd,rot,norm", [("bf16", 128, 128, True), ("f32", 64, 64, True),
                                               ("f16", 256, 256, False), ("bf16", 64, 16, True)])
def test_append_many(cuda, ops, dtype, hd, rot, norm):
    """70000 head rows, among them some whose groups are no ordinary ones: constants, zeros,
    one value far from the others, numbers too large or small, NaN.  Queries within
    rounding; every code, scale and mid as the 64-bit form's."""
    N, H, page, eps = 5900, 4, 16, 1e-6
    g = torch.Generator().manual_seed(hd)
    x = torch.randn(N, 3 * H, hd, generator=g)
    x[7::50, 5] = 2.5
    x[9::50, 9] = 0.0
    x[11::50, 10] = 40.0 + 0.001 * x[11::50, 10]
    x[13::50, 11, 3] = 3e4
    x[15::50, 8] *= 6e-8 if dtype == "f16" else 1e-36
    x[17::50, 9] *= 1.5e4 if dtype == "f16" else 1e36
    x[19::50, 10, 1] = float("nan")
    x[21::50, 4, hd - 1] = float("inf")
    x = x.to(so.TYPES[dtype])
    n_pages = -(-N // page) + 1
    codes = torch.zeros(n_pages, 2, H, page, hd // 2, dtype=torch.uint8)
    pairs = torch.zeros(n_pages, 2, H, page, hd // 64, 2, dtype=torch.bfloat16)
    dev = codes.cuda(), pairs.cuda()
    angles = torch.rand(90, rot // 2, generator=g, dtype=torch.float64) * 100
    cos, sin = (torch.cat([t, t], 1).float() for t in (angles.cos(), angles.sin()))
    positions = torch.randint(0, 90, (N,), generator=g)
    slots = torch.randperm(n_pages * page, generator=g)[:N]
    w = [1 + 0.1 * torch.randn(hd, generator=g) if norm else None for _ in range(2)]
    y = x.cuda()
    out = ops.paged_append_q4(y[:, :H], y[:, H:2 * H], y[:, 2 * H:], cos.cuda(), sin.cuda(), positions.cuda(),
                              slots.cuda(), dev[0][:, 0], dev[1][:, 0], dev[0][:, 1], dev[1][:, 1], norm,
                              *[t if t is None else t.cuda() for t in w], eps)
    want, mag = so.append_rows(x[:, :H], w[0], cos, sin, positions, norm, eps)
    small = 2.0 ** -25 if dtype == "f16" else 0.0
    so.near(out, want, so.half_step(out.dtype) * want.abs() + 32 * so.HALF * mag + small, "append q")
    keys, _ = so.append_rows(x[:, H:2 * H], w[1], cos, sin, positions, norm, eps)
    for i, v in enumerate((keys, x[:, 2 * H:])):
        codes[slots // page, i, :, slots % page], pairs[slots // page, i, :, slots % page] = qo.quantise(v)
    assert torch.equal(dev[0].cpu(), codes), "codes"
    assert torch.equal(dev[1].cpu().nan_to_num(7e7), pairs.nan_to_num(7e7)), "pairs"


# ---- a long prefix, many rows: tiles of it made into values once ----------------------

@pytest.mark.parametrize("hd,lens,prefix,n_kv,rep,tokens,page,rows_first", [
    (64, [5, 0], 5500, 12, 64, 1, 64, False),           # 128 rows: one whole block
    (128, [40, 3, 17], 5601, 16, 11, 3, 16, False),     # 99 rows, pages inside a tile
    (256, [1, 70], 5500, 16, 50, 1, 32, True),          # 100 rows: two blocks of 64
    (128, [9], 8300, 32, 18, 1, 48, False),             # 18 rows, a block of 64
])
def test_shared(cuda, ops, hd, lens, prefix, n_kv, rep, tokens, page, rows_first):
    batch = qo.Batch(lens, prefix, n_kv, rep, hd, page, "bf16", rows_first, 1, seed=hd)
    check(ops, batch, tokens, f"hd={hd} {lens} behind {prefix}, {n_kv} x {rep} heads")


def test_shared_hidden(cuda, ops):
    """Pages of the prefix outside the pool, a NaN among its keys and one among its
    values: the rows and heads that see them alone."""
    for page in (64, 24):
        batch = qo.Batch([30, 2], 5600, 12, 64, 64, page, "bf16", seed=page)
        n = batch.codes.shape[0]
        batch.prefix_table[3], batch.prefix_table[-1], batch.prefix_table[50] = -1, n, 1 << 30
        q = batch.queries(1, 1.5)
        clean = check(ops, batch, 1, f"hidden pages of {page}", q=q)
        for i, h in ((0, 2), (1, 7)):
            p = int(batch.prefix_table[10 + i])
            batch.pairs[p, i, h, 5] = float("nan")
        got = decode(ops, batch, q, 0.125).reshape(2, 12, 64, 64)
        clean = clean.reshape(got.shape)
        others = [h for h in range(12) if h not in (2, 7)]
        assert got[:, [2, 7]].isnan().all() and torch.equal(got[:, others], clean[:, others])
        batch.prefix_table[:] = -1                      # nothing of the prefix is there
        check(ops, batch, 1, "no prefix in the pool", q=q)
        bad = q.clone()
        bad[1, 64 * 5 + 3, 7] = float("inf")
        got = decode(ops, batch, bad, 0.125)
        want = decode(ops, batch, q, 0.125)
        assert got[1, 64 * 5 + 3].isnan().all()
        got[1, 64 * 5 + 3] = want[1, 64 * 5 + 3]
        assert torch.equal(got, want)


def test_shared_large_scores(cuda, ops):
    """Maxima that move over the tiles, weights of 0, a scale below 0."""
    batch = qo.Batch([30, 2], 5600, 12, 64, 64, 32, "bf16", seed=1, offset=2.0)
    for scale in (1.0, -0.5, 0.0):
        check(ops, batch, 1, f"scale {scale}", scale, batch.queries(1, 3.0))


# ---- many sequences: a block for all of a sequence's keys --------------------------------

@pytest.mark.parametrize("dtype,hd,prefix,page", [("bf16", 64, 500, 32), ("f16", 128, 0, 24), ("f32", 64, 77, 64),
                                                  ("bf16", 256, 300, 16)])
def test_many_sequences(cuda, ops, dtype, hd, prefix, page):
    """520 blocks and more, prefix and own keys in one walk, lengths of 0 to 900."""
    batch = qo.Batch([i * 61 % 900 for i in range(130)], prefix, 4, 2, hd, page, dtype, room=0, seed=hd + prefix)
    check(ops, batch, 1, f"{dtype} hd={hd} 130 sequences behind {prefix}")


@pytest.mark.parametrize("dtype,hd,page", [("bf16", 128, 96), ("f32", 64, 160), ("f16", 256, 33), ("bf16", 64, 1000)])
def test_odd_pages(cuda, ops, dtype, hd, page):
    """Pages of whole tiles whose count is no power of two, pages that end inside one."""
    batch = qo.Batch([5, 700, 161, 96, 1500], 490, 2, 3, hd, page, dtype, room=1, seed=page)
    check(ops, batch, 2, f"{dtype} hd={hd} pages of {page}")


# ---- far pages, streams, graphs ---------------------------------------------------------

def test_far_pages(cuda, ops):
    """Pages whose codes lie more than 2^32 bytes on."""
    batch = qo.Batch([100, 37], 50, 1, 2, 256, 16, "bf16", seed=18)
    n = batch.codes.shape[0]
    far = (2 ** 32 + 2 ** 20) // (2 * 16 * 128)
    codes = torch.empty(far + n, 2, 1, 16, 128, dtype=torch.uint8, device=cuda)
    pairs = torch.empty(far + n, 2, 1, 16, 4, 2, dtype=torch.bfloat16, device=cuda)
    codes[far:], pairs[far:] = batch.codes.cuda(), batch.pairs.cuda()
    cache = codes[:, 0], pairs[:, 0], codes[:, 1], pairs[:, 1]
    tables = torch.where(batch.tables >= 0, batch.tables + far, -1).int().cuda()
    q = batch.queries(1)
    got = ops.prefix_attention_decode_q4(q.cuda(), *cache, batch.prefix_table.cuda() + far, 50, tables,
                                         batch.lengths.cuda(), 0.0625)
    so.near(got, *qo.attend(batch, q, 1, 0.0625), "far pages")
    last = torch.tensor([(far + n) * 16 - 1], device=cuda)
    x = torch.randn(1, 1, 256)
    d, t = x.cuda(), torch.ones(1, 256, device=cuda)
    ops.paged_append_q4(d, d, d, t, 0 * t, 0 * last, last, *cache, False, None, None, 0.0)
    want = qo.quantise(x)
    assert torch.equal(codes[-1, 0, 0, 15].cpu(), want[0][0, 0])
    assert torch.equal(pairs[-1, 1, 0, 15].cpu(), want[1][0, 0])
    k, v = ops.paged_read_q4(*cache, last, torch.float32)
    assert torch.equal(k.cpu(), qo.values(*want).float()) and torch.equal(k, v)


def test_other_stream(cuda, ops):
    """The same bits from every call, on whichever stream it is queued."""
    batch = qo.Batch([900, 77, 5], 1300, 2, 8, 128, 16, "bf16", seed=16)
    q = batch.queries(1)
    cache, (pt, tables, lengths) = batch.cuda()
    qd = q.cuda()
    probs = torch.softmax(torch.randn(3, 4, 5000, device=cuda), -1)
    drafts, u = torch.randint(0, 5000, (3, 3), device=cuda), torch.rand(3, 4, device=cuda)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append((ops.prefix_attention_decode_q4(qd, *cache, pt, 1300, tables, lengths, 0.1),
                             *ops.verify_drafts(probs, drafts, probs[:, :3].sqrt(), None, u)))
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    so.near(outs[0][0], *qo.attend(batch, q, 1, 0.1), "other streams")
    for out in outs:
        assert all(torch.equal(a, b) for a, b in zip(out, outs[0]))


class Step:
    """A step of verification on static tensors: append the newest tokens and drafts,
    attend, take the outputs' softmax for probabilities, verify."""

    def __init__(self, ops, dtype, hd, seed, prefix):
        self.ops, self.tokens, self.hd = ops, 3, hd
        b = self.batch = qo.Batch([40, 500], prefix, 2, 4, hd, 16, dtype, room=2, seed=seed)
        self.cache, (self.pt, self.tables, self.lengths) = b.cuda()
        free = sorted(set(range(b.codes.shape[0])) - set(b.prefix_table.tolist())
                      - set(b.tables.flatten().tolist()))
        for i, page in enumerate(free[:2]):                 # pages for the new tokens
            b.tables[i, b.tables[i].tolist().index(-1)] = page
        self.tables.copy_(b.tables)
        N, dev = 2 * self.tokens, "cuda"
        self.pos, self.slot = (torch.zeros(N, dtype=torch.int64, device=dev) for _ in range(2))
        self.x = torch.zeros(N, b.n_q + 4, hd, dtype=b.dtype, device=dev)
        angles = torch.arange(2500)[:, None] * 0.1 ** torch.linspace(0, 4, hd // 2)
        self.cos, self.sin = (torch.cat([t, t], 1).float().cuda() for t in (angles.cos(), angles.sin()))
        self.drafts = torch.zeros(2, 2, dtype=torch.int64, device=dev)
        self.u = torch.zeros(2, 3, device=dev)

    def fill(self, i, g):
        b = self.batch
        at = [n + 2 * i + t for n in b.lens for t in range(self.tokens)]
        rows = [int(b.tables[s, n // 16]) * 16 + n % 16
                for n, s in zip(at, [0] * self.tokens + [1] * self.tokens)]
        self.x.copy_(torch.randn(self.x.shape, generator=g).to(b.dtype))
        self.lengths.copy_(torch.tensor([n + 2 * i + self.tokens for n in b.lens], dtype=torch.int32))
        self.pos.copy_(torch.tensor([b.prefix + n for n in at]))
        self.slot.copy_(torch.tensor(rows))
        self.drafts.copy_(torch.randint(0, b.n_q * self.hd, (2, 2), generator=g))
        self.u.copy_(torch.rand(2, 3, generator=g) * 1e-3)

    def __call__(self):
        n, b = self.batch.n_q, self.batch
        y = self.ops.paged_append_q4(self.x[:, :n], self.x[:, n:n + 2], self.x[:, n + 2:], self.cos, self.sin,
                                     self.pos, self.slot, *self.cache, True, None, None, 1e-6)
        out = self.ops.prefix_attention_decode_q4(y, *self.cache, self.pt, b.prefix, self.tables, self.lengths,
                                                  self.hd ** -0.5)
        probs = torch.softmax(out.float().reshape(2, 3, -1), -1)
        return (y, out, probs, *self.ops.verify_drafts(probs, self.drafts, None, None, self.u))

    def check(self, got, what):
        """Against the plain forms on what the cache holds."""
        y, out, probs, tokens, counts = got
        b = self.batch
        b.codes.copy_(torch.stack([self.cache[0], self.cache[2]], 1).cpu())
        b.pairs.copy_(torch.stack([self.cache[1], self.cache[3]], 1).cpu())
        lengths, b.lengths = b.lengths, self.lengths.cpu()
        want, tol = qo.attend(b, y.cpu(), self.tokens, self.hd ** -0.5)
        b.lengths = lengths
        none = want.isnan()         # positions past the tables store nothing: rows stay NaN
        assert torch.equal(out.isnan().cpu(), none)
        so.near(out.masked_fill(none.cuda(), 0.0), *(x.masked_fill(none, 0.0) for x in (want, tol)), what)
        want = qo.verify(probs.cpu(), self.drafts.cpu(), None, None, self.u.cpu())
        assert torch.equal(tokens.cpu(), want[0]) and torch.equal(counts.cpu(), want[1])


def test_graphs(cuda, ops):
    """Two steps captured once, of one pool of workspaces, replayed in turn with eager
    calls between: lengths, rows, queries and drafts change between replays."""
    steps = [Step(ops, "bf16", 64, 17, 200), Step(ops, "f32", 128, 18, 1200)]
    for s in steps:
        s.slot.fill_(-1)
        s()                                                 # loads the code
    torch.cuda.synchronize()
    graphs, outs = [torch.cuda.CUDAGraph() for _ in steps], []
    mempool = torch.cuda.graph_pool_handle()
    for s, graph in zip(steps, graphs):
        with torch.cuda.graph(graph, pool=mempool):
            outs.append(s())
    g = torch.Generator().manual_seed(1)
    for i in range(4):
        for n, (s, graph, out) in enumerate(zip(steps, graphs, outs)):
            s.fill(i, g)
            graph.replay()
            torch.cuda.synchronize()
            got = [x.clone() for x in out]
            eager = s()
            assert all(torch.equal(a, b) for a, b in zip(got, eager)), f"replay {i} of {n}"
            s.check(got, f"replay {i} of {n}")


@pytest.mark.parametrize("dtype,hd,prefix", [("f32", 64, 0), ("f16", 128, 77), ("bf16", 256, 1900),
                                             ("bf16", 256, 2000)])
def test_together(cuda, ops, dtype, hd, prefix):
    """Append, attend and verify, step by step, each against its plain form."""
    step = Step(ops, dtype, hd, 30 + hd, prefix)
    g = torch.Generator().manual_seed(hd)
    for i in range(3):
        step.fill(i, g)
        step.check(step(), f"{dtype} hd={hd} step {i}")


# ---- gradients, refusals ------------------------------------------------------------------

def test_no_gradients(cuda, ops):
    """These operators serve: the same outputs, no graph in the cache, and a backward
    pass through them says that there is none."""
    step = Step(ops, "f32", 64, 3, 20)
    step.fill(0, torch.Generator().manual_seed(0))
    want = step()
    step.x.requires_grad_()
    got = step()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    with pytest.warns(UserWarning, match="autograd kernel was not registered"):
        got[1].sum().backward()
    assert step.x.grad is None or not step.x.grad.any()
    assert not any(t.requires_grad for t in step.cache)


def test_attention_refusals(cuda, ops):
    batch = qo.Batch([30, 77], 20, 2, 2, 64, 16, "bf16", seed=19)
    (kc, ks, vc, vs), (pt, tables, lengths) = batch.cuda()
    q = batch.queries(1).cuda()
    good = dict(q=q, kc=kc, ks=ks, vc=vc, vs=vs, pt=pt, p=20, t=tables, n=lengths, s=0.125)

    def call(**kw):
        return ops.prefix_attention_decode_q4(*{**good, **kw}.values())
    assert call().shape == (2, 4, 64)
    odd = torch.zeros(kc.numel() + 64, dtype=kc.dtype, device=cuda)[8:]
    odd = odd[:kc.numel()].view(kc.shape)
    for kw, text in [
            (dict(q=q.double()), "float32, bfloat16"), (dict(q=q[:, :3]), "heads of"),
            (dict(q=q[..., :32]), "heads of"), (dict(q=q[:1]), "tokens for every"), (dict(q=q[0]), "device tensor"),
            (dict(kc=kc[:1]), "one shape"), (dict(kc=kc.int()), "uint8"), (dict(vs=vs.half()), "bfloat16"),
            (dict(ks=ks[:1], vs=vs[:1]), "codes are"), (dict(kc=kc[:0], vc=vc[:0]), "empty"),
            (dict(kc=kc[..., :16], vc=vc[..., :16]), "hd must be"), (dict(vc=vc.contiguous()), "one layout"),
            (dict(ks=ks[..., :1], vs=vs[..., :1]), "pairs"), (dict(kc=odd, vc=odd), "aligned"),
            (dict(kc=kc.transpose(2, 3).contiguous().transpose(2, 3),
                  vc=vc.transpose(2, 3).contiguous().transpose(2, 3)), "contiguous"),
            (dict(pt=pt[:1]), "names 1 pages"), (dict(p=-1), "prefix_table names"),
            (dict(p=33), "prefix_table names"), (dict(t=tables[:1]), "contiguous"),
            (dict(t=tables.long()), "tables must be"), (dict(n=lengths.long()), "lengths must be"),
            (dict(n=lengths.cpu()), "is on cpu"), (dict(kc=kc.cpu()), "is on cpu"),
            (dict(s=float("nan")), "scale"), (dict(s=float("inf")), "scale")]:
        with pytest.raises(RuntimeError, match=text):
            call(**kw)


def test_append_and_read_refusals(cuda, ops):
    batch = qo.Batch([30, 77], 20, 2, 2, 64, 16, "bf16", seed=19)
    (kc, ks, vc, vs), _ = batch.cuda()
    x = torch.zeros(2, 4, 64, device=cuda)
    kv, tab, at = x[:, :2], torch.zeros(8, 64, device=cuda), torch.zeros(2, dtype=torch.int64, device=cuda)
    w = torch.ones(64, device=cuda)
    good = dict(q=x, k=kv, v=kv, cos=tab, sin=tab, pos=at, slot=at, kc=kc, ks=ks, vc=vc, vs=vs, norm=True, qw=w,
                kw=w, eps=1e-6)

    def call(**kw):
        return ops.paged_append_q4(*{**good, **kw}.values())
    before = kc.clone()
    for kw, text in [
            (dict(k=x), "k must be"), (dict(v=kv.half()), "q's type"), (dict(q=x.double()), "float32, bfloat16"),
            (dict(cos=tab[:0], sin=tab[:0]), "need a row"), (dict(sin=tab[:4]), "one shape"),
            (dict(cos=tab[:, :63].contiguous(), sin=tab[:, :63].contiguous()), "even width"),
            (dict(cos=tab.half()), "cos and sin"), (dict(pos=at[:1]), "one a token"), (dict(slot=at.int()), "slots must be"),
            (dict(slot=at.cpu()), "is on cpu"), (dict(norm=False), "without the norm"), (dict(qw=w[:32]), "q_weight"),
            (dict(kw=w.half()), "k_weight"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
            (dict(vc=vc[:1]), "one shape")]:
        with pytest.raises(RuntimeError, match=text):
            call(**kw)
    assert torch.equal(kc, before)
    for slots, dtype, text in ((at.int(), torch.float32, "slots must be"), (at.cpu(), torch.float32, "device|CPU|cpu"),
                               (at, torch.float64, "float32, bfloat16"), (at[::2].expand(2, 1), torch.float32, "slots"),
                               (torch.zeros(4, dtype=torch.int64, device=cuda)[::2], torch.float32, "contiguous")):
        with pytest.raises(RuntimeError, match=text):
            ops.paged_read_q4(kc, ks, vc, vs, slots, dtype)


def test_verify_refusals(cuda, ops):
    p = torch.rand(2, 4, 100, device=cuda)
    good = dict(p=p, d=torch.zeros(2, 3, dtype=torch.int64, device=cuda), q=p[:, :3], n=None,
                u=torch.zeros(2, 4, device=cuda))
    n = torch.zeros(4, dtype=torch.int32, device=cuda)
    assert ops.verify_drafts(*good.values())[0].shape == (2, 4)
    for kw, text in [
            (dict(p=p[0]), "probs must be"), (dict(p=p.double()), "float32, bfloat16"), (dict(p=p[:, :0]), "probs is"),
            (dict(p=p[..., :0]), "probs is"), (dict(d=good["d"].int()), "drafts must be"),
            (dict(d=good["d"][:, :2]), "drafts is"), (dict(q=p), "draft_probs must be"),
            (dict(q=p[:, :3].half()), "draft_probs must be"), (dict(q=p[:, :3].cpu()), "is on cpu"),
            (dict(n=n), "one a sequence"), (dict(n=n[::2]), "contiguous"), (dict(n=n[:2].long()), "n_drafts must be"),
            (dict(u=good["u"][:, :3]), "uniforms is"), (dict(u=good["u"].double()), "uniforms must be")]:
        with pytest.raises(RuntimeError, match=text):
            ops.verify_drafts(*{**good, **kw}.values())
