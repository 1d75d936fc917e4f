"""verify_drafts of torch.ops.cbq against the rule in 64 bits (q4_oracle.verify):
the same tokens, every one."""
import pytest
import torch

import q4_oracle as qo

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


@pytest.fixture(scope="module")
def ops(cuda):
    import cbq_ops
    return cbq_ops.load()


def check(ops, probs, drafts, draft_probs, n_drafts, uniforms, what):
    print(f"verify {what}", flush=True)
    dev = [None if x is None else x.cuda() for x in (probs, drafts, draft_probs, n_drafts, uniforms)]
    tokens, counts = ops.verify_drafts(*dev)
    assert tokens.dtype == torch.int64 and counts.dtype == torch.int32
    want = qo.verify(probs, drafts, draft_probs, n_drafts, uniforms)
    assert torch.equal(counts.cpu(), want[1]), (counts, want[1])
    assert torch.equal(tokens.cpu(), want[0]), (tokens, want[0])
    return want


def inputs(B, K, V, dtype, seed, spread=0.7):
    g = torch.Generator().manual_seed(seed)
    logits = 2.5 * torch.randn(B, K + 1, V, generator=g)
    near = torch.softmax(logits[:, :K] + spread * torch.randn(B, K, V, generator=g), -1).to(TYPES[dtype])
    drafts = torch.multinomial(near.float().reshape(B * K, V), 1, generator=g).reshape(B, K) \
        if K else torch.zeros(B, 0, dtype=torch.int64)
    return (torch.softmax(logits, -1).to(TYPES[dtype]), drafts, near,
            torch.rand(B, K + 1, generator=g), g)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("B,K,V", [(1, 4, 151936), (3, 7, 1000), (40, 2, 2048), (5, 1, 2049), (9, 3, 63),
                                   (4, 0, 4097), (6, 5, 1), (2, 70, 300), (300, 3, 17)])
def test_verify(cuda, ops, dtype, B, K, V):
    probs, drafts, near, u, g = inputs(B, K, V, dtype, B + K)
    check(ops, probs, drafts, near, None, u, f"{dtype} {B}x{K} of {V}")
    check(ops, probs, drafts, None, None, u, f"{dtype} {B}x{K} of {V}, certain drafts")
    some = torch.randint(-1, K + 2, (B,), generator=g, dtype=torch.int32)
    check(ops, probs, drafts, near, some, u, f"{dtype} {B}x{K} of {V}, some drafts")


def test_chain(cuda, ops):
    """Drafts from the target itself are all kept (u q < p where q = p), none of a token
    that the target never gives."""
    probs, drafts, _, u, _ = inputs(20, 5, 500, "f32", 1)
    drafts = torch.multinomial(probs[:, :5].reshape(-1, 500), 1).reshape(20, 5)
    _, counts = check(ops, probs, drafts, probs[:, :5].contiguous(), None, u, "the target's own")
    assert (counts == 6).all()
    probs.scatter_(2, drafts[:, :, None], 0.0)
    _, counts = check(ops, probs, drafts, None, None, torch.zeros_like(u), "impossible")
    assert (counts == 1).all()


def test_borders(cuda, ops):
    """Random numbers on the sums' borders, at both ends and beside a chunk's: dyadic
    probabilities, whose sums are exact in any order."""
    V = 8192
    p = torch.zeros(1, 1, V)
    p[0, 0, ::2] = 2.0 / V
    for u in (0.0, 0.25, 0.5, 0.5 - 2 ** -20, 0.75, 1 - 2.0 ** -24, 2046 / V, 2048 / V, 2050 / V, 1.0, 1.5, -1.0):
        check(ops, p, torch.zeros(1, 0, dtype=torch.int64), None, None, torch.tensor([[u]]), f"u = {u}")
    q = torch.zeros(1, 1, V)
    q[0, 0, 5] = 0.5                                    # u q = p: refused
    t = torch.zeros(1, 2, V)
    t[0, 0, 5], t[0, 0, 7] = 0.25, 0.75
    t[0, 1, 9] = 1
    d = torch.tensor([[5]])
    assert check(ops, t, d, q, None, torch.tensor([[0.5, 0.0]]), "on the border")[0].tolist() == [[7, -1]]
    assert check(ops, t, d, q, None, torch.tensor([[0.5 - 2 ** -25, 0.0]]), "below it")[0].tolist() == [[5, 9]]


def test_odd_values(cuda, ops):
    """Rows without a remainder, without anything, with NaN and negative numbers; drafts
    outside the vocabulary; random numbers that are NaN."""
    nan = float("nan")
    p = torch.tensor([[[0.2, 0.3, 0.5], [0.1, 0.2, 0.7]], [[0.0, 0.0, 0.0], [0.0, 1.0, 0.0]],
                      [[nan, 0.5, -0.5], [nan, nan, 0.5]], [[0.2, 0.3, 0.5], [0.1, 0.2, 0.7]],
                      [[0.2, 0.3, 0.5], [0.0, 0.0, 0.0]]])
    q = p[:, :1].clone()
    for drafts in ([2, 0, 0, 3, 1], [0, 1, 1, -1, 1 << 40]):
        d = torch.tensor(drafts)[:, None]
        for u0, u1 in ((0.0, 0.3), (0.999, 0.999), (1.0, 0.0), (nan, 0.5)):
            u = torch.full((5, 2), u0)
            u[:, 1] = u1
            for draft_probs in (q, 2 * q, None):
                check(ops, p, d, draft_probs, None, u, f"{drafts} {u0} {u1}")


def test_layouts(cuda, ops):
    """Rows in any strides, a vocabulary that is not contiguous, broadcast rows."""
    probs, drafts, near, u, _ = inputs(4, 3, 777, "f32", 5)
    want = qo.verify(probs, drafts, near, None, u)
    wide = torch.zeros(4, 4, 1000, device="cuda")
    wide[:, :, 3:780] = probs.cuda()
    p2 = probs.cuda().permute(2, 0, 1).contiguous().permute(1, 2, 0)
    n2 = near.cuda().transpose(0, 1).contiguous().transpose(0, 1)
    d2 = drafts.cuda().t().contiguous().t()
    for p, n, d in ((wide[:, :, 3:780], near.cuda(), d2), (p2, n2, drafts.cuda())):
        tokens, counts = ops.verify_drafts(p, d, n, None, u.cuda())
        assert torch.equal(tokens.cpu(), want[0]) and torch.equal(counts.cpu(), want[1])
    one = probs[:1, :1].expand(4, 4, 777)
    check(ops, one.contiguous(), drafts, None, None, u, "one row for all")
    got = ops.verify_drafts(probs[:1, :1].cuda().expand(4, 4, 777), drafts.cuda(), None, None, u.cuda())
    assert torch.equal(got[0].cpu(), qo.verify(one, drafts, None, None, u)[0])
    none = ops.verify_drafts(probs[:0].cuda(), drafts[:0].cuda(), None, None, u[:0].cuda())
    assert none[0].shape == (0, 4) and none[1].shape == (0,)


def test_distribution(cuda, ops):
    """What is kept and drawn is distributed as the target: 2^16 sequences of one draft
    over five tokens, each share within five standard deviations."""
    n = 1 << 16
    g = torch.Generator().manual_seed(4)
    p, q = torch.tensor([0.1, 0.4, 0.05, 0.3, 0.15]), torch.tensor([0.3, 0.1, 0.2, 0.2, 0.2])
    drafts = torch.multinomial(q, n, replacement=True, generator=g)[:, None]
    u = torch.rand(n, 2, generator=g)
    tokens, _ = ops.verify_drafts(p.cuda().expand(n, 2, 5), drafts.cuda(), q.cuda().expand(n, 1, 5), None,
                                  u.cuda())
    share = torch.bincount(tokens[:, 0].cpu(), minlength=5) / n
    assert ((share - p).abs() <= 5 * (p * (1 - p) / n).sqrt()).all(), share
