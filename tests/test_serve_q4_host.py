"""The 4-bit cache and the verification of drafts without a GPU: launch plans under
sanitizers, refusals of the C entry points before any launch, the operators' schemas
and shape functions, the plain forms' own arithmetic."""
import ctypes
import os
import subprocess

import pytest
import torch

import cbq_native
import q4_oracle as qo

NATIVE = os.path.join(os.path.dirname(os.path.abspath(__file__)), "native")


@pytest.fixture(scope="module")
def lib():
    try:
        return cbq_native.load()
    except RuntimeError as e:
        pytest.fail(str(e))


def test_plans():
    r = subprocess.run(["make", "-s", "-C", NATIVE, "q4"], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stderr[-3000:]
    r = subprocess.run([os.path.join(NATIVE, "cbq_q4_host")], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0 and "all cases passed" in r.stdout, (r.stdout + r.stderr)[-4000:]


def _cache(p, **kw):
    c = cbq_native.PagedQ4(k_codes=p, v_codes=p, k_scales=p, v_scales=p, n_pages=4, page=16, n_kv=2, hd=64)
    for i, (codes, scales) in enumerate(((1024, 64), (512, 32), (32, 2))):
        c.code_stride[i], c.scale_stride[i] = codes, scales
    for name, value in kw.items():
        if name in ("code_stride", "scale_stride"):
            getattr(c, name)[value[0]] = value[1]
        else:
            setattr(c, name, value)
    return c


POOLS = [dict(hd=96), dict(hd=0), dict(hd=512), dict(page=0), dict(page=65537), dict(n_pages=0),
         dict(n_pages=1 << 28), dict(n_kv=0), dict(code_stride=(2, 24)), dict(code_stride=(0, -1024)),
         dict(code_stride=(0, 1 << 41)), dict(scale_stride=(2, 3)), dict(scale_stride=(1, -2)),
         dict(code_stride=(0, 1 << 35)), dict(scale_stride=(0, 1 << 32))]
POINTERS = ["k_codes", "v_codes", "k_scales", "v_scales"]


def _pointers(p):
    return [dict(zip([n], [None])) for n in POINTERS] + [{n: p + (8 if "codes" in n else 2)} for n in POINTERS]


def _buffer():
    buf = ctypes.create_string_buffer(256)
    return buf, (ctypes.addressof(buf) + 15) // 16 * 16


def test_attention_refusals(lib):
    buf, p = _buffer()
    st = (ctypes.c_int64 * 2)(256, 64)

    def call(c, q=p, strides=st, dtype=1, pt=p, prefix=10, t=p, width=300, lens=p, batch=2, tokens=3, n_q=4,
             scale=0.1, out=p, ws=p, nws=1 << 40):
        return lib.cbq_prefix_attn_decode_q4(q, strides, dtype, ctypes.byref(c), pt, prefix, t, 300, width,
                                             lens, batch, tokens, n_q, scale, out, ws, nws, None)
    need = lib.cbq_prefix_attn_decode_q4_workspace(ctypes.byref(_cache(p)), 10, 300, 2, 3, 4, 1)
    assert need > 0
    for kw in (dict(q=None), dict(strides=None), dict(pt=None), dict(t=None), dict(lens=None), dict(out=None),
               dict(ws=None), dict(nws=need - 1), dict(ws=p + 4), dict(q=p + 2), dict(out=p + 8), dict(dtype=3),
               dict(dtype=-1), dict(n_q=3), dict(n_q=0), dict(n_q=1 << 20), dict(prefix=-1), dict(prefix=1 << 31),
               dict(width=-1), dict(width=1 << 28), dict(batch=-1), dict(batch=1 << 30), dict(tokens=0),
               dict(tokens=-1), dict(tokens=1 << 28), dict(scale=float("nan")), dict(scale=float("inf")),
               dict(strides=(ctypes.c_int64 * 2)(255, 64))):
        assert call(_cache(p), **kw) == 2, kw
    for kw in POOLS + _pointers(p):
        assert call(_cache(p, **kw)) == 2, kw
    one = _cache(p, page=1)                                     # tables of 2^30 entries
    assert call(one, width=1 << 30) == 2 and call(one, prefix=1 << 30) == 2
    assert call(_cache(p), batch=0) == 0                        # nothing to do
    assert lib.cbq_prefix_attn_decode_q4_workspace(ctypes.byref(_cache(p, hd=65)), 10, 3, 2, 1, 4, 1) == 0


def test_append_and_read_refusals(lib):
    buf, p = _buffer()
    st = (ctypes.c_int64 * 2)(256, 64)

    def append(c, ptrs=(p,) * 3, x=1, strides=(st,) * 3, tables=(p, p), n_pos=8, rot=64, at=(p, p), out=p, N=3,
               n_q=4, norm=1, eps=1e-6):
        return lib.cbq_paged_append_q4(*ptrs, x, *strides, *tables, n_pos, rot, *at, norm, None, None, eps, out,
                                       ctypes.byref(c), N, n_q, None)
    for kw in (dict(ptrs=(None, p, p)), dict(ptrs=(p, None, p)), dict(ptrs=(p, p, None)), dict(x=3), dict(x=-1),
               dict(strides=(st, None, st)), dict(tables=(None, p)), dict(n_pos=0), dict(rot=0), dict(rot=63),
               dict(rot=66), dict(at=(p, None)), dict(out=None), dict(out=p + 4), dict(N=-1), dict(n_q=0),
               dict(N=1 << 31), dict(N=1 << 29), dict(eps=-1.0), dict(eps=float("nan"))):
        assert append(_cache(p), **kw) == 2, kw

    def read(c, slots=p, N=3, dtype=0, k=p, v=p):
        return lib.cbq_paged_read_q4(ctypes.byref(c), slots, N, dtype, k, v, None)
    for kw in (dict(slots=None), dict(N=-1), dict(N=1 << 32), dict(dtype=3), dict(dtype=-1), dict(k=None),
               dict(v=None), dict(k=p + 8)):
        assert read(_cache(p), **kw) == 2, kw
    for kw in POOLS + _pointers(p):
        assert append(_cache(p, **kw)) == 2 and read(_cache(p, **kw)) == 2, kw
    assert append(_cache(p), N=0) == 0 and read(_cache(p), N=0) == 0


def test_verify_refusals(lib):
    buf, p = _buffer()
    st = (ctypes.c_int64 * 2)(256, 64)

    def call(probs=p, ps=st, drafts=p, q=p, qs=st, dtype=0, n=None, u=p, batch=2, n_max=3, vocab=1000, tokens=p,
             counts=p, ws=p, nws=1 << 40):
        return lib.cbq_verify_drafts(probs, ps, drafts, q, qs, dtype, n, u, batch, n_max, vocab, tokens, counts,
                                     ws, nws, None)
    need = lib.cbq_verify_drafts_workspace(2, 1000)
    assert need > 0
    for kw in (dict(probs=None), dict(ps=None), dict(drafts=None), dict(qs=None), dict(dtype=3), dict(dtype=-1),
               dict(u=None), dict(batch=-1), dict(batch=1 << 24), dict(n_max=-1), dict(n_max=1 << 20),
               dict(batch=1 << 23, n_max=1 << 10), dict(vocab=0), dict(vocab=1 << 31), dict(tokens=None),
               dict(counts=None), dict(ws=None), dict(ws=p + 8), dict(nws=need - 1)):
        assert call(**kw) == 2, kw
    assert call(batch=0) == 0
    assert lib.cbq_verify_drafts_workspace(-1, 10) == 0 and lib.cbq_verify_drafts_workspace(1, 0) == 0


def test_schemas_and_shapes():
    import cbq_ops
    ops = cbq_ops.load()
    assert ("Tensor(a!) k_codes, Tensor(b!) k_scales, Tensor(c!) v_codes, Tensor(d!) v_scales"
            in str(ops.paged_append_q4.default._schema))
    m = torch.device("meta")
    codes = torch.empty(4, 2, 16, 32, device=m, dtype=torch.uint8)
    scales = torch.empty(4, 2, 16, 1, 2, device=m, dtype=torch.bfloat16)
    cache = codes, scales, codes, scales
    q, kv = torch.empty(6, 4, 64, device=m), torch.empty(6, 2, 64, device=m)
    i, t = torch.empty(6, dtype=torch.int64, device=m), torch.empty(9, 64, device=m)
    out = ops.paged_append_q4(q, kv, kv, t, t, i, i, *cache, False, None, None, 0.0)
    assert out.shape == q.shape and out.dtype == q.dtype
    k, v = ops.paged_read_q4(*cache, i, torch.float16)
    assert k.shape == v.shape == (6, 2, 64) and k.dtype == torch.float16
    n, rows = torch.empty(3, dtype=torch.int32, device=m), torch.empty(3, 2, dtype=torch.int32, device=m)
    out = ops.prefix_attention_decode_q4(q, *cache, n, 0, rows, n, 0.1)
    assert out.shape == q.shape and out.dtype == q.dtype
    probs, drafts = torch.empty(3, 5, 70, device=m), torch.empty(3, 4, dtype=torch.int64, device=m)
    tokens, counts = ops.verify_drafts(probs, drafts, None, None, torch.empty(3, 5, device=m))
    assert tokens.shape == (3, 5) and tokens.dtype == torch.int64
    assert counts.shape == (3,) and counts.dtype == torch.int32
    cpu = torch.zeros(1, 2, 5)
    with pytest.raises(NotImplementedError):            # no kernel for host tensors
        ops.verify_drafts(cpu, torch.zeros(1, 1, dtype=torch.int64), None, None, torch.zeros(1, 2))


def test_format():
    """Values come back within 0.52 of a step (half of it, and what the roundings of the
    middle and the step add: 2^-8 of 7.5 steps at most each way), in the order they went."""
    g = torch.Generator().manual_seed(0)
    for hd in (64, 128, 256):
        assert sorted(qo.order(hd).tolist()) == list(range(hd))
        x = torch.randn(40, hd, generator=g, dtype=torch.float64) * torch.logspace(-6, 6, 40)[:, None] + 0.3
        codes, pairs = qo.quantise(x)
        assert codes.shape == (40, hd // 2) and pairs.shape == (40, hd // 64, 2)
        step = pairs.double()[..., 0].repeat_interleave(64, -1)
        assert ((qo.values(codes, pairs) - x).abs() <= 0.53 * step).all()
        # byte (e / 4) (hd / 32) + 2 g + e % 4 / 2, even values low
        c = (qo.parts(codes, pairs)[0] + 7.5).to(torch.uint8)
        for d in (0, 1, 63, hd - 1, hd // 2):
            group, e = d // 64, d % 64
            byte = codes[:, e // 4 * (hd // 32) + 2 * group + e % 4 // 2]
            assert torch.equal(byte >> 4 if e % 2 else byte & 15, c[:, d])
    codes, pairs = qo.quantise(torch.tensor([[float("nan")] + [1.0] * 63, [2.0] * 64, [0.0] * 64]))
    v = qo.values(codes, pairs)
    assert v[0].isnan().all() and (v[1] == 2).all() and (v[2] == 0).all()
