"""paged_append_q4 of rows with an infinity, normed: its factor is 0, as paged_append's."""
import pytest
import torch

import q4_oracle as qo
import serve_oracle as so

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("hd,rot", [(128, 128), (256, 64), (256, 16), (128, 34)])
def test_infinite_rows(cuda, dtype, hd, rot):
    """Groups that the infinity does not reach hold zeros, those that it does NaN."""
    import cbq_ops
    ops = cbq_ops.load()
    N = 9
    g = torch.Generator().manual_seed(hd + rot)
    x = torch.randn(N, 1, hd, generator=g)
    x[1, 0, hd - 1], x[4, 0, 3], x[7, 0, 70] = float("inf"), -float("inf"), float("nan")
    x = x.to(so.TYPES[dtype])
    angles = torch.rand(5, rot // 2, generator=g, dtype=torch.float64) * 100
    cos, sin = (torch.cat([t, t], 1).float() for t in (angles.cos(), angles.sin()))
    positions, slots = torch.arange(N) % 5, torch.arange(N)
    codes = torch.zeros(1, 1, N, hd // 2, dtype=torch.uint8, device=cuda)
    pairs = torch.zeros(1, 1, N, hd // 64, 2, dtype=torch.bfloat16, device=cuda)
    cache = codes, pairs, codes.clone(), pairs.clone()
    d = x.cuda()
    ops.paged_append_q4(d, d, d, cos.cuda(), sin.cuda(), positions.cuda(), slots.cuda(), *cache, True, None, None, 1e-6)
    keys, _ = so.append_rows(x, None, cos, sin, positions, True, 1e-6)
    want = qo.quantise(keys[:, 0])
    assert torch.equal(cache[1][0, 0].cpu().nan_to_num(7e7), want[1].nan_to_num(7e7))
    assert torch.equal(cache[0][0, 0].cpu(), want[0])
