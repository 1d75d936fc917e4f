"""prefix_attention_decode_q4 by rows and by single keys (q4_checks.py): small weights beside
a large one, small values beside large ones, keys at every kind of border."""
import math

import pytest
import torch

import q4_checks as qc
import q4_oracle as qo
import serve_oracle as so
from test_gpu_serve_q4 import decode

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(cuda):
    import cbq_ops
    return cbq_ops.load()


@pytest.mark.parametrize("dtype,hd,n_kv,rep,prefix", [
    ("bf16", 64, 8, 64, 8300), ("bf16", 128, 8, 64, 8300), ("bf16", 256, 8, 64, 8300),      # tiles shared
    ("bf16", 128, 2, 4, 2000), ("f16", 64, 2, 4, 2000)])
@pytest.mark.parametrize("gap", [12.0, 21.7, 23.4])
def test_weak_keys(cuda, ops, dtype, hd, n_kv, rep, prefix, gap):
    """One key in sixteen has the weight 1 and the value 0, the others 2^-gap and values
    around 4096: the output is theirs alone.  A weight holds fp16's 11 bits down to 2^-25
    of the largest one, where the maximum stands 4 times above it: half a step of the
    output, of each weight and (twice) of each value, below four."""
    batch = qo.Batch([0, 3], prefix, n_kv, rep, hd, 16, dtype, seed=hd)
    batch.pairs[:, 0] = 0.0                             # keys: scale 0, mid 0
    for page in batch.prefix_table.tolist():
        batch.codes[page, 1], batch.pairs[page, 1] = qo.quantise(
            4096 * (1 + torch.randn(n_kv, 16, hd, generator=batch.g)))
        batch.pairs[page, 0, :, 5, 0, 1] = 1.0          # the strong key: 64 ones
        batch.pairs[page, 1, :, 5] = 0.0
    page = int(batch.tables[1, 0])
    batch.codes[page, 1], batch.pairs[page, 1] = qo.quantise(4096 + torch.zeros(n_kv, 16, hd))
    q = torch.zeros(2, n_kv * rep, hd, dtype=batch.dtype)
    q[..., :64] = 1.0
    out = decode(ops, batch, q, gap * math.log(2) / 64)
    j = torch.arange(prefix)
    at = batch.prefix_table[j // 16].long(), j % 16
    v = qo.values(batch.codes[at[0], 1, :, at[1]], batch.pairs[at[0], 1, :, at[1]])     # [keys, n_kv, hd]
    strong = int((j % 16 == 5).sum())
    w = 2.0 ** -gap
    for b, own in enumerate((0, 3)):
        want = w * (v.sum(0) + own * 4096.0) / (strong + w * (prefix - strong + own))
        qc.near_rows(out[b], want.repeat_interleave(rep, 0), 4 * so.half_step(batch.dtype), f"sequence {b}")


def test_small_values(cuda, ops):
    """Values of one group 2^-27 of the other's, in tiles that are made into fp16 numbers
    against the largest.  The largest scale becomes 2^10 or more, so the group's s are 2^-18.8
    or more, rounded to fp16's smallest number: off by 2^-25, 2^-6.2 of them, 3.5 half steps of
    bf16; their middles and sums by 2^-25 each, of values of 4 s and more 0.9; the output by
    one.  Seven half steps of a row in all; the other group's, whose scales are exact, two."""
    batch = qo.Batch([0, 3], 8300, 8, 64, 128, 16, "bf16", seed=5)
    scales = batch.pairs[batch.prefix_table.long(), 1, :, :12, :, 0].float()
    assert float(scales[..., 1].min() / scales.amax()) >= 2.0 ** -1.8
    batch.pairs[:, 1, :, :, 1] *= 2.0 ** -27
    q = batch.queries(1, 1.5)
    out = decode(ops, batch, q, 128 ** -0.5)
    want = qc.exact(batch, q, 1, 128 ** -0.5)
    for half, steps in ((slice(0, 64), 2), (slice(64, 128), 7)):
        qc.near_rows(out[..., half], want[..., half], steps * so.half_step(batch.dtype), f"values {half}")


SHAPES = [  # lens, prefix, n_kv, rep, hd, page, tokens, rows_first, room, types
    ([5, 0], 5500, 12, 64, 64, 64, 1, False, 1, ["bf16", "f16"]),       # shared tiles, 128 rows a block
    ([40, 3, 17], 5601, 16, 11, 128, 16, 3, False, 1, ["bf16", "f32"]),
    ([1, 70], 5500, 16, 50, 256, 32, 1, True, 1, ["bf16"]),             # 64 rows a block
    ([9], 8300, 32, 18, 128, 48, 1, False, 1, ["bf16"]),
    ([130, 600, 31, 5], 900, 1, 4, 64, 32, 2, False, 3, ["f32", "bf16", "f16"]),
    ([130, 600, 31, 5], 900, 2, 4, 256, 24, 2, False, 3, ["f32", "bf16", "f16"]),
    ([90, 7, 1200], 33, 2, 7, 128, 17, 4, False, 1, ["f32", "bf16", "f16"]),        # 28 rows a sequence
    ([9000, 31, 4000], 0, 2, 4, 128, 64, 1, False, 9, ["f32", "bf16", "f16"]),
    ([2500, 8100], 3000, 4, 12, 64, 256, 5, False, 0, ["bf16", "f16"]),
    ([i * 61 % 900 for i in range(130)], 300, 4, 2, 64, 32, 1, False, 0, ["bf16", "f32"]),  # a block a sequence
    ([i * 37 % 300 for i in range(130)], 700, 4, 2, 128, 24, 1, False, 0, ["f16"]),
    ([i * 37 % 300 for i in range(130)], 0, 4, 2, 256, 32, 1, False, 0, ["bf16"]),
    ([i * 7 % 90 for i in range(130)], 2900, 8, 2, 64, 16, 1, False, 0, ["bf16", "f16", "f32"]),  # few own keys
]


@pytest.mark.parametrize("dtype,shape", [(t, s[:-1]) for s in SHAPES for t in s[-1]],
                         ids=[f"{t}-{i}" for i, s in enumerate(SHAPES) for t in s[-1]])
def test_rows_and_borders(cuda, ops, dtype, shape):
    """Every row within its roundings; rows of two keys, one at a border of tiles or at
    either end, of prefix and own keys alike: each counts, and once."""
    lens, prefix, n_kv, rep, hd, page, tokens, rows_first, room = shape
    batch = qo.Batch(lens, prefix, n_kv, rep, hd, page, dtype, rows_first, room, seed=hd + prefix)
    scale = hd ** -0.5
    q = batch.queries(tokens, 1.5)
    worst = qc.near_rows(decode(ops, batch, q, scale), qc.exact(batch, q, tokens, scale), qc.bound(batch), dtype)
    print(f"{dtype} hd={hd} prefix={prefix}: rows within {worst / qc.bound(batch):.2f} of the bound", flush=True)
    q, two = qc.planted(batch, tokens, scale)
    worst = qc.near_planted(decode(ops, batch, q, scale), qc.exact(batch, q, tokens, scale), two, batch, dtype)
    print(f"  two keys: {16 * worst:.2f} of the bound", flush=True)
