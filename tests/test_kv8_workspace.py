"""The workspaces of attention over the cache in 8 bits, sized once for the
most sequences, tokens and the longest context to come, do for every call on
less: their sizes never fall when one of them grows.  On the CPU, as in
test_context_workspace.py."""
import numpy as np
import pytest

from test_context_refusals import call  # noqa: F401 (a fixture)
from test_context_workspace import SHAPES
from test_kv8_refusals import cache8


def desc(kv_heads, dim):
    return cache8(kv_heads=kv_heads, head_dim=dim, page_stride=16 * kv_heads * dim, token_stride=kv_heads * dim, head_stride=dim)


@pytest.mark.parametrize("heads,kv_heads,dim", SHAPES)
def test_decode_size(call, heads, kv_heads, dim):  # noqa: F811
    d, most = desc(kv_heads, dim), (1 << 22) // heads
    size = lambda n, m: call.attn8_decode_workspace(d, heads, n, m)
    counts = [n for n in [*range(0, 1100), 2000, 4095, 4096, 4097, 5000, most] if n <= most]
    for max_len in (0, 1, 2048, 2049, 131071, 2 ** 31 - 1):
        sizes = [size(n, max_len) for n in counts]
        assert sizes == sorted(sizes), max_len
    for n in (1, 2, 63, 64, 65, 128, 129, 255, 256, 512, 513, 4096, 4097):
        sizes = [size(n, m) for m in (0, 1, 127, 128, 129, 2048, 2049, 65536, 2 ** 30, 2 ** 31 - 1)]
        assert sizes == sorted(sizes), n
    # rows for as many pieces as run at once and one a sequence, of those that are cut
    pieces = 4 * 256 // (kv_heads * -(-heads // kv_heads // 16)) + 2 + 4096
    assert size(most, 2 ** 31 - 1) <= pieces * heads * (dim + 2) * 4 + 4096 * 8


@pytest.mark.parametrize("heads,kv_heads,dim", SHAPES)
def test_prompt_size(call, heads, kv_heads, dim):  # noqa: F811
    d = desc(kv_heads, dim)
    size = lambda n, t, q, m: call.attn8_prompt_workspace(d, heads, n, t, q, m)
    rng, rows = np.random.default_rng(heads), min(1 << 22, (1 << 30) // heads)
    for _ in range(2000):
        n, t, q, m = (sorted(int(2 ** rng.uniform(0, top)) for _ in range(2)) for top in (22 - np.log2(heads), np.log2(rows), 22, 31))
        assert size(n[0], t[0], q[0], m[0]) <= size(n[1], t[1], q[1], m[1]), (n, t, q, m)
    # partial rows for as many blocks of 128 as run at once, twice
    assert size(1, rows, rows, 2 ** 31 - 1) <= 2 * 128 * 256 * (dim + 2) * 4

