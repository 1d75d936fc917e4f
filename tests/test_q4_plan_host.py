"""Launch plans of the attention over the 4-bit cache by what they ask for: no workspace where
one block takes all keys of a sequence, else room for the parts' sums."""
import ctypes

import pytest

import cbq_native


def joint(batch, prefix, capacity, n_kv=8, rep=4, hd=128, tokens=1, dtype=1):
    lib = cbq_native.load()
    cache = cbq_native.PagedQ4(page=16, n_kv=n_kv, hd=hd)
    return lib.cbq_prefix_attn_decode_q4_workspace(ctypes.byref(cache), prefix, -(-capacity // 16), batch, tokens,
                                                   n_kv * rep, dtype) == 0


@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_prefix_of_many_sequences(dtype):
    """A prefix is read for many sequences at a time, unless it is short."""
    for batch, short, long in ((64, 100, 1000), (256, 100, 1000), (1024, 100, 1000), (1024, 100, 2900)):
        assert joint(batch, short, 100, dtype=dtype) and not joint(batch, long, 100, dtype=dtype)
    assert not joint(486, 2777, 68, rep=1, hd=256, dtype=dtype)
    assert joint(603, 10, 16, rep=12, hd=64, tokens=4, dtype=dtype)


def test_own_keys():
    """Without a prefix as before: few keys, or sequences that fill the CUs."""
    assert joint(1, 0, 128) and not joint(1, 0, 1200) and joint(64, 0, 1900) and not joint(64, 0, 3200)
    assert joint(1, 64, 64) and not joint(1, 64, 1200)


def test_once():
    """Rows that share no tile with another sequence's have nothing to lose."""
    for tokens in (4, 8):
        assert joint(64, 1000, 100, tokens=tokens)          # 16 and 32 rows a sequence
