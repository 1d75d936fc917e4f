"""Batched serving at the ends of its ranges: launches of more threads than one
grid dimension holds, values and scales at the ends of their types.  Tolerances:
serve_oracle.py."""
import math

import pytest
import torch

import serve_oracle as so
from serve_oracle import Batch
from test_gpu_serve import check_decode, ops, prompt, starts  # noqa: F401

pytestmark = pytest.mark.gpu


# ---- launches of 2^24 blocks and more ---------------------------------------------

def test_append_many_rows(cuda, ops):
    """2^26 + 40 head rows, a wave each."""
    N, n_q, n_kv, page = 2 ** 23 + 5, 6, 1, 4096
    g = torch.Generator(device=cuda).manual_seed(1)
    y = torch.randn(N, n_q + 2, 2, generator=g, device=cuda, dtype=torch.float16)
    pages = torch.zeros(-(-N // page), 2, n_kv, page, 2, device=cuda, dtype=torch.float16)
    angles = torch.rand(50, 1, generator=g, device=cuda, dtype=torch.float64) * 100
    cos, sin = (torch.cat([t, t], 1).float() for t in (angles.cos(), angles.sin()))
    positions = torch.randint(0, 50, (N,), generator=g, device=cuda)
    slots = torch.randperm(N, generator=g, device=cuda)
    print("append of 2^26 + 40 rows", flush=True)
    out = ops.paged_append(y[:, :n_q], y[:, n_q:n_q + 1], y[:, n_q + 1:], cos, sin, positions, slots,
                           pages[:, 0], pages[:, 1], False, None, None, 0.0)
    rows = pages.permute(0, 3, 1, 2, 4).reshape(-1, 2, 2)[slots]        # [N, key and value, 2]
    assert torch.equal(rows[:, 1], y[:, n_q + 1])
    for lo in range(0, N, 1 << 20):
        at = slice(lo, lo + (1 << 20))
        want, mag = so.append_rows(y[at, :n_q + 1], None, cos, sin, positions[at], False, 0.0)
        tol = 2.0 ** -11 * want.abs() + 32 * so.HALF * mag + 2.0 ** -25
        got = torch.cat([out[at], rows[at, :1]], 1).double()
        assert ((got - want).abs() <= tol).all(), lo


def test_decode_many_blocks(cuda, ops):
    """17 sequences of 2^20 - 1 heads, two parts of the own keys: 2^25 blocks and
    more, and as many rows to merge as 2^24."""
    heads, page, width = 2 ** 20 - 1, 2, 1100
    g = torch.Generator(device=cuda).manual_seed(2)
    pool = torch.randn(5, 2, heads, page, 64, generator=g, device=cuda, dtype=torch.bfloat16)
    lens = [2100, 0, 1, 3] + [2] * 13
    tables = torch.randint(0, 5, (17, width), dtype=torch.int32, generator=torch.Generator().manual_seed(3))
    q = torch.randn(17, heads, 64, generator=g, device=cuda, dtype=torch.bfloat16)
    print("decode of 2^25 blocks", flush=True)
    out = ops.prefix_attention_decode(q, pool[:, 0], pool[:, 1], tables.new_zeros(0).cuda(), 0,
                                      tables.cuda(), torch.tensor(lens, dtype=torch.int32, device=cuda),
                                      0.125)
    # some heads as a batch of their own: the first, the last, around 2^22 and 2^24 rows
    some = [0, 1, 2 ** 18 - 1, 2 ** 18, heads // 2, 987654, heads - 2, heads - 1]
    b = Batch([], 0, len(some), 1, 64, page, "bf16", room=0)
    b.k, b.v = pool[:, 0, some].cpu(), pool[:, 1, some].cpu()
    b.lens, b.tables, b.lengths = lens, tables, torch.tensor(lens)
    so.near(out[:, some], *so.attend(b, q[:, some].cpu(), starts([1] * 17), 0.125), "some heads")
    # one key a sequence: its value, whatever the query
    one = pool[int(tables[2, 0]), 1, :, 0]
    assert torch.equal(out[2], one) and not out[1].any()


def test_prompt_many_blocks(cuda, ops):
    """Five one-token runs of 2^20 - 1 heads: more than 2^22 blocks."""
    heads = 2 ** 20 - 1
    g = torch.Generator(device=cuda).manual_seed(4)
    pool = torch.randn(3, 2, heads, 1, 64, generator=g, device=cuda, dtype=torch.bfloat16)
    q = torch.randn(5, heads, 64, generator=g, device=cuda, dtype=torch.bfloat16)
    tables = torch.tensor([[0, -1], [1, -1], [2, 0], [0, 1], [-1, -1]], dtype=torch.int32)
    lens = [1, 1, 2, 2, 0]
    print("prompt of 5 * 2^20 blocks", flush=True)
    out = ops.prefix_attention_prompt(q, starts([1] * 5).cuda(), pool[:, 0], pool[:, 1],
                                      tables.new_zeros(0).cuda(), 0, tables.cuda(),
                                      torch.tensor(lens, dtype=torch.int32, device=cuda), 0.125)
    assert torch.equal(out[0], pool[0, 1, :, 0]) and torch.equal(out[1], pool[1, 1, :, 0])
    assert not out[4].any()
    some = [0, 1, 2 ** 18, heads // 2, 987654, heads - 1]
    b = Batch([], 0, len(some), 1, 64, 1, "bf16", room=0)
    b.k, b.v = pool[:, 0, some].cpu(), pool[:, 1, some].cpu()
    b.lens, b.tables, b.lengths = lens, tables, torch.tensor(lens)
    so.near(out[:, some], *so.attend(b, q[:, some].cpu(), starts([1] * 5), 0.125), "some heads")


# ---- large values -------------------------------------------------------------------

def _late_key(dtype, prefix, lens, at, value, n_kv=1, rep=2, hd=64):
    """Scores 0 but for own key `at` of every sequence, which is 5.5 more (244 times
    the others' weight), and values of one large magnitude."""
    b = Batch(lens, prefix, n_kv, rep, hd, 16, dtype, seed=30)
    b.k.zero_()
    sign = torch.where(torch.rand(hd, generator=b.g) < 0.5, -1.0, 1.0)
    b.v.copy_(value * sign * (1 - 0.5 * torch.rand(b.v.shape, generator=b.g)))
    for row in b.tables:
        b.k[int(row[at // 16]), :, at % 16, 0] = 5.5
    q = torch.zeros(len(lens), b.n_q, hd, dtype=b.dtype)
    q[:, :, 0] = 1.0
    return b, q


# fp16's largest values; of the other types, values whose sums stay below 2^128
# while 2^8 times a value does not.
LARGE = {"f32": 2.0 ** 122, "bf16": 2.0 ** 122, "f16": 60000.0}


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("prefix,n,hd", [(0, 400, 64), (0, 300, 128), (1200, 400, 64), (0, 3000, 128),
                                         (600, 200, 256)])
def test_large_values_decode(cuda, ops, dtype, prefix, n, hd):
    """A later key's score above those before it by less than the slack that the
    running maximum has."""
    b, q = _late_key(dtype, prefix, [n, n], n - 7, LARGE[dtype], hd=hd)
    out = check_decode(ops, b, f"large values {dtype} prefix={prefix} n={n} hd={hd}", 1.0, q)
    assert out.isfinite().all()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("prefix", [300, 1100])
@pytest.mark.parametrize("n_kv,rep", [(1, 1), (8, 4), (8, 16)])
def test_large_values_prompt(cuda, ops, dtype, prefix, n_kv, rep):
    """The same in a prompt: blocks of 16, 64 and 128 rows, and row by row beside an
    infinite value that the last token alone sees."""
    n = 130
    b, q1 = _late_key(dtype, prefix, [n], 0, LARGE[dtype], n_kv, rep)
    q, q_start = q1.expand(n, -1, -1).contiguous(), starts([n])
    want, tol = so.attend_prompt(b, q, q_start, 1.0)
    print(f"large values {dtype} prefix={prefix} heads={n_kv}x{rep}", flush=True)
    so.near(prompt(ops, b, q, q_start, 1.0), want, tol, "large values")
    b.v[int(b.tables[0, (n - 1) // 16]), :, (n - 1) % 16, 3] = float("inf")
    got = prompt(ops, b, q, q_start, 1.0)
    assert (got[-1, :, 3] == float("inf")).all()
    so.near(got[:-1], want[:-1], tol[:-1], "before an infinite value")


# ---- small scales -------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("scale", [1e-31, -1e-31, 2.0 ** -126, 2.0 ** -130])
def test_small_scale_of_large_products(cuda, ops, dtype, scale):
    """Queries and keys whose products are as large as the scale is small."""
    large = min(abs(scale) ** -0.5, 2.0 ** 63)                  # products within fp32's range
    b = Batch([300, 40], 100, 1, 2, 64, 16, dtype, seed=31, scale_k=large / 32)
    q = b.queries(2, large)
    check_decode(ops, b, f"scale {scale} {dtype}", scale, q)
    want, tol = so.attend_prompt(b, q, torch.tensor([0, 1, 2], dtype=torch.int32), scale)
    so.near(prompt(ops, b, q, starts([1, 1]), scale), want, tol, f"prompt, scale {scale} {dtype}")


# ---- rows done key by key beside products ----------------------------------------------

@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_equal_scores_across_parts(cuda, ops, dtype):
    """Every score the same, from exact products, in parts of which the last, with an
    infinite value, is done key by key: the mean of the values.  No score's rounding
    enters (one score, one weight), so the tolerance is the sums'."""
    for scale in (1.0, 0.7, 1.1, 0.9, 0.3, 0.77):
        b = Batch([3040], 0, 1, 4, 64, 16, dtype, seed=32)
        b.k.zero_()
        b.k[..., 0] = 60.0
        q = torch.zeros(40, 4, 64, dtype=b.dtype)
        q[..., 0] = 60.0
        q_start = starts([40])
        b.v.fill_(-1.0)
        for j in range(2700, 3040):                             # inside the last part
            b.v[int(b.tables[0, j // 16]), :, j % 16] = 1.0
        b.v[int(b.tables[0, 3039 // 16]), 0, 3039 % 16, 5] = float("inf")
        got = prompt(ops, b, q, q_start, scale).double().cpu()
        v = b.dense(0)[1][:, 0]
        for t in range(39):
            n = 3000 + t + 1
            want, mass = v[:n].mean(0), v[:n].abs().mean(0)
            half = so.half_step(b.dtype)
            tol = half * want.abs() + (n / 16 + 64) * so.HALF * mass
            if dtype != "f32":
                tol = tol + half * mass
            if dtype == "f16":
                tol = tol + 2.0 ** -25 * v[:n].abs().amax(0) + 2.0 ** -25
            so.near(got[t], want.expand(4, 64), tol.expand(4, 64), f"scale {scale}, token {t}")
        assert (got[39, :, 5] == math.inf).all()


# ---- inputs that ask for gradients --------------------------------------------------

def test_no_gradients(cuda, ops):
    """These operators serve: the same outputs, no graph in the pages, and a backward
    pass through them says that there is none."""
    b = Batch([30, 77], 20, 2, 2, 64, 16, "f32", seed=33, fill=0.0)
    k, v, prefix_table, tables, lengths = b.cuda()
    x = torch.randn(2, 8, 64, device=cuda)
    at, table = torch.tensor([3, 4], device=cuda), torch.rand(8, 64, device=cuda)
    slots = torch.tensor([int(b.tables[s, n // 16]) * 16 + n % 16 for s, n in enumerate((29, 76))],
                         device=cuda)

    def step(y):
        q = ops.paged_append(y[:, :4], y[:, 4:6], y[:, 6:], table, table, at, slots, k, v, True, None,
                             None, 1e-6)
        return q, ops.prefix_attention_decode(q, k, v, prefix_table, 20, tables, lengths, 0.125), \
            ops.prefix_attention_prompt(q, starts([1, 1]).cuda(), k, v, prefix_table, 20, tables, lengths,
                                        0.125)
    want = step(x)
    y = x.clone().requires_grad_()
    for a, c in zip(want, step(y)):
        assert torch.equal(a, c)
        with pytest.warns(UserWarning, match="autograd kernel was not registered"):
            c.sum().backward(retain_graph=True)
    assert y.grad is None or not y.grad.any()
    assert not k.requires_grad and not v.requires_grad
