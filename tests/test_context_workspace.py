"""The decode workspace sized once, for the largest batch and the longest
context to come, does for every call on less: its size never falls when nseq
or max_len grows.  On the CPU: the size is computed on the host, from a zeroed
stand-in for the context's memory."""
import numpy as np
import pytest

from test_context_refusals import cache, call  # noqa: F401 (call is a fixture)


def sized(c, heads, kv_heads, dim):
    desc = cache(kv_heads=kv_heads, head_dim=dim, page_stride=16 * kv_heads * dim, token_stride=kv_heads * dim,
                 head_stride=dim)
    return lambda nseq, max_len: c.attn_decode_workspace(desc, heads, nseq, max_len)


SHAPES = [(16, 2, 256), (32, 8, 128), (8, 8, 64), (12, 4, 128), (7, 1, 64), (40, 2, 128), (1024, 64, 256), (1024, 1, 256)]


@pytest.mark.parametrize("heads,kv_heads,dim", SHAPES)
def test_size_grows_with_sequences(call, heads, kv_heads, dim):  # noqa: F811
    size = sized(call, heads, kv_heads, dim)
    most = (1 << 22) // heads
    counts = [n for n in list(range(0, 1100)) + [2000, 4096, most] if n <= most]
    for max_len in (0, 1, 128, 129, 4096, 32769, 131071, 1 << 30, (1 << 30) + 1, 2 ** 31 - 1):
        sizes = [size(n, max_len) for n in counts]
        assert sizes == sorted(sizes), max_len


@pytest.mark.parametrize("heads,kv_heads,dim", SHAPES)
def test_size_grows_with_length(call, heads, kv_heads, dim):  # noqa: F811
    size = sized(call, heads, kv_heads, dim)
    edges = [m * 128 * p + d for m in (1, 2, 3, 16, 257) for p in (1, 3, 64, 255, 256, 512) for d in (-1, 0, 1)]
    lens = sorted(set(list(range(0, 2000, 7)) + edges + [32768, 32769, 33000, 1 << 30, (1 << 30) + 1, 2 ** 31 - 1]))
    for nseq in (1, 2, 3, 64, 129, 255, 256, 511, 512, 1023, 1024, 4096):
        sizes = [size(nseq, n) for n in lens]
        assert sizes == sorted(sizes), nseq


def test_size_stays_small(call):  # noqa: F811
    """It is for as many parts as run at once, not for every sequence's: at
    most twice four a CU and key head's tile, of a row of fp32 and two sums."""
    for heads, kv_heads, dim in SHAPES:
        tiles = -(-heads // kv_heads // 16)
        most = 2 * (4 * 256 // (kv_heads * tiles) + 1) * heads * (dim + 2) * 4
        assert sized(call, heads, kv_heads, dim)((1 << 22) // heads, 2 ** 31 - 1) <= most, (heads, kv_heads, dim)


def test_drawn_pairs(call):  # noqa: F811
    """Any call on fewer sequences, shorter ones or both needs no more."""
    rng = np.random.default_rng(17)
    size = sized(call, 16, 2, 256)
    for _ in range(3000):
        n, m = (int(2 ** rng.uniform(0, 12)) for _ in range(2))
        a, b = (int(2 ** rng.uniform(0, 31)) for _ in range(2))
        assert size(min(n, m), min(a, b)) <= size(max(n, m), max(a, b))
