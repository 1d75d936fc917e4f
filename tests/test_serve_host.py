"""Batched serving without a GPU: addresses and launch plans of the paged cache
under sanitizers, refusals of the C entry points before any launch, the
operators' schemas and shape functions."""
import ctypes
import os
import subprocess

import pytest
import torch

import cbq_native

NATIVE = os.path.join(os.path.dirname(os.path.abspath(__file__)), "native")


@pytest.fixture(scope="module")
def lib():
    try:
        return cbq_native.load()
    except RuntimeError as e:
        pytest.fail(str(e))


def test_addresses_and_plans():
    r = subprocess.run(["make", "-s", "-C", NATIVE, "paged"], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stderr[-3000:]
    r = subprocess.run([os.path.join(NATIVE, "cbq_paged_host")], capture_output=True, text=True,
                       timeout=600)
    assert r.returncode == 0 and "all cases passed" in r.stdout, (r.stdout + r.stderr)[-4000:]


def _cache(p, **kw):
    c = cbq_native.PagedKV(k=p, v=p, n_pages=4, page=16, n_kv=2, hd=64, dtype=1)
    for s in (c.k_stride, c.v_stride):
        s[0], s[1], s[2] = 2048, 1024, 64
    for name, value in kw.items():
        setattr(c, name, value)
    return c


def test_attention_refusals(lib):
    buf = ctypes.create_string_buffer(256)
    p = (ctypes.addressof(buf) + 15) // 16 * 16
    st = (ctypes.c_int64 * 2)(256, 64)

    def call(c, q=p, strides=st, pt=p, prefix=10, t=p, width=300, lens=p, batch=2, n_q=4, scale=0.1,
             out=p, ws=p, nws=1 << 40):
        return lib.cbq_prefix_attn_decode(q, strides, ctypes.byref(c), pt, prefix, t, 300, width, lens,
                                          batch, n_q, scale, out, ws, nws, None)
    need = lib.cbq_prefix_attn_decode_workspace(ctypes.byref(_cache(p)), 10, 300, 2, 4)
    assert need > 0
    bad = [dict(q=None), dict(strides=None), dict(pt=None), dict(t=None), dict(lens=None),
           dict(out=None), dict(ws=None), dict(nws=need - 1), dict(ws=p + 4), dict(q=p + 2),
           dict(n_q=3), dict(n_q=0), dict(prefix=-1), dict(prefix=1 << 31), dict(width=-1),
           dict(width=1 << 28), dict(batch=-1), dict(scale=float("nan")), dict(scale=float("inf")),
           dict(strides=(ctypes.c_int64 * 2)(255, 64))]
    for kw in bad:
        assert call(_cache(p), **kw) == 2, kw
    for kw in (dict(hd=96), dict(hd=0), dict(page=0), dict(page=65537), dict(n_pages=0),
               dict(n_pages=1 << 28), dict(n_kv=0), dict(dtype=3), dict(dtype=-1), dict(k=None),
               dict(v=p + 8)):
        assert call(_cache(p, **kw)) == 2, kw
    c = _cache(p)
    c.v_stride[2] = 65
    assert call(c) == 2
    c = _cache(p, n_pages=1 << 26)
    c.k_stride[0] = (1 << 20) + 8                               # 2^50 bytes in units of 16
    assert call(c) == 2
    c.k_stride[0], c.k_stride[2] = 1024, -64
    assert call(c) == 2
    assert call(_cache(p), batch=0) == 0                        # nothing to do
    prompt = lib.cbq_prefix_attn_prompt
    args = (ctypes.byref(_cache(p)), p, 10, p, 3, 3, p, 2)
    assert prompt(p, st, None, *args, 7, 4, 0.1, p, p, 1 << 40, None) == 2      # no q_start
    assert prompt(p, st, p, *args, -1, 4, 0.1, p, p, 1 << 40, None) == 2
    assert prompt(p, st, p, *args, 1 << 31, 4, 0.1, p, p, 1 << 40, None) == 2
    assert prompt(p, st, p, *args, 0, 4, 0.1, p, p, 1 << 40, None) == 0
    assert lib.cbq_prefix_attn_prompt_workspace(ctypes.byref(_cache(p, hd=65)), 10, 3, 2, 7, 4) == 0


def test_append_refusals(lib):
    buf = ctypes.create_string_buffer(256)
    p = (ctypes.addressof(buf) + 15) // 16 * 16
    st = (ctypes.c_int64 * 2)(256, 64)

    def call(c, ptrs=(p,) * 3, x=1, strides=(st,) * 3, tables=(p, p), n_pos=8, rot=64, at=(p, p),
             out=p, N=3, n_q=4):
        return lib.cbq_paged_append(*ptrs, x, *strides, *tables, n_pos, rot, *at, 1, None, None, 1e-6,
                                    out, ctypes.byref(c), N, n_q, None)
    for kw in (dict(ptrs=(None, p, p)), dict(ptrs=(p, None, p)), dict(ptrs=(p, p, None)), dict(x=2),
               dict(x=3), dict(x=-1), dict(strides=(st, None, st)), dict(tables=(None, p)),
               dict(n_pos=0), dict(rot=0), dict(rot=63), dict(rot=66), dict(at=(p, None)),
               dict(out=None), dict(N=-1), dict(n_q=0), dict(N=1 << 31), dict(N=1 << 29)):
        assert call(_cache(p), **kw) == 2, kw
    for kw in (dict(hd=258), dict(hd=63), dict(hd=0), dict(page=0), dict(n_pages=0),
               dict(n_pages=1 << 27), dict(n_kv=0), dict(dtype=7), dict(k=None)):
        assert call(_cache(p, **kw)) == 2, kw
    assert call(_cache(p), N=0) == 0


def test_schemas_and_shapes():
    import cbq_ops
    ops = cbq_ops.load()
    assert "Tensor(a!) k_pages, Tensor(b!) v_pages" in str(ops.paged_append.default._schema)
    m = torch.device("meta")
    pages = torch.empty(4, 2, 16, 64, device=m, dtype=torch.float16)
    q, kv = torch.empty(3, 4, 64, device=m), torch.empty(3, 2, 64, device=m)
    i = torch.empty(3, dtype=torch.int64, device=m)
    t = torch.empty(9, 64, device=m)
    out = ops.paged_append(q, kv, kv, t, t, i, i, pages, pages, False, None, None, 0.0)
    assert out.shape == q.shape and out.dtype == torch.float16
    q = q.half()
    n = torch.empty(3, dtype=torch.int32, device=m)
    rows = torch.empty(3, 2, dtype=torch.int32, device=m)
    out = ops.prefix_attention_decode(q, pages, pages, n, 0, rows, n, 0.1)
    assert out.shape == q.shape and out.dtype == q.dtype
    out = ops.prefix_attention_prompt(q, n, pages, pages, n, 0, rows[:2], n[:2], 0.1)
    assert out.shape == q.shape
    cpu = torch.zeros(1, 2, 16, 64)
    with pytest.raises(NotImplementedError):            # no kernel for host tensors
        ops.prefix_attention_decode(torch.zeros(1, 2, 64), cpu, cpu, torch.zeros(0, dtype=torch.int32),
                                    0, torch.zeros(1, 1, dtype=torch.int32),
                                    torch.zeros(1, dtype=torch.int32), 0.1)
