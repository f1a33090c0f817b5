"""GPU: the context operators as a program uses them: a workspace sized once
for all that is to come, scores of minus infinity, the performance cases'
order."""
import os
import subprocess
import sys

import numpy as np
import pytest

import context_oracle as O
import nmoe_hip as nh
from test_gpu_context import Decode, ctx, within  # noqa: F401 (ctx is a fixture)

pytestmark = pytest.mark.gpu


def lse_tol(q, k, scale, lse):
    """The error of a logarithm of a sum of exponentials: the scores' (fp32
    sums of D products, D + 8 half steps of their magnitudes), the sum's own
    (half steps of n terms, added up as their root, twice over for the parts),
    the exponentials' 2^-21, and four half steps of the logarithm, of the
    maximum (in powers of two) and of what they add up to."""
    n, D = k.shape
    mag = (np.abs(k) @ np.abs(q)).max() * abs(scale)
    return (D + 8) * 2.0 ** -24 * mag + n ** 0.5 * 2.0 ** -23 + 2.0 ** -21 + 4 * 2.0 ** -24 * (abs(lse) * 1.45 + 16 + mag)


def test_decode_workspace_sized_once(ctx):  # noqa: F811
    """Sized for the most and the longest, then calls on fewer and shorter
    sequences, which are cut into more parts than those were."""
    H, K, D, page = 4, 1, 64, 16
    rng = np.random.default_rng(40)
    calls = [[65537], [65536], [9, 700, 4097], rng.integers(0, 300, 1023).tolist(), rng.integers(0, 300, 1024).tolist()]
    size = ws = None
    for lens in calls:
        d = Decode(ctx, rng, nh.BF16, H, K, D, page, lens)
        if ws is None:
            size = ctx.attn_decode_workspace(d.cache.desc, H, 1024, 65537)
            ws = ctx.to_device(np.full(size, 0xFF, np.uint8))
        ctx._check(ctx.attn_decode(d.cache.desc, d.dq, H, len(lens), d.dlens, d.dtable, d.max_pages, max(lens), d.scale,
                                   d.out, d.lse, ws, size))
        ctx.sync()
        d.check(skip=set(range(3, len(lens))) - set(range(3, len(lens), 101)))


@pytest.mark.parametrize("dtype,H,K,D", [(nh.BF16, 16, 2, 256), (nh.F16, 4, 4, 128), (nh.F16, 7, 1, 64)])
@pytest.mark.parametrize("max_len", [1, 5000])
def test_decode_keys_of_minus_infinity(ctx, dtype, H, K, D, max_len):  # noqa: F811
    """Keys whose score is minus infinity weigh nothing, also where a
    wavefront's step, a workgroup's or a whole part has no others."""
    gone = [range(0, 32), range(0, 128), range(128, 512), [*range(32, 300), 700], range(0, 31), range(0)]
    d = Decode(ctx, np.random.default_rng(41), dtype, H, K, D, 16, [500, 300, 777, 901, 33, 64])
    d.q[..., 3] = O.pack(np.ones(1), dtype)[0]
    d.dq.upload(d.q)
    q = O.value(d.q, dtype)
    for b, js in enumerate(gone):
        js = np.array(js, np.int64)
        slots = d.table[b, js // 16].astype(np.int64) * 16 + js % 16
        rows = d.k[b][js].astype(np.float32)
        rows[..., 3] = -np.inf
        d.cache.put(0, slots, O.pack(rows, dtype))
    d.cache.upload()
    d.run(max_len)
    ctx.sync()
    got, got_lse = d.read()
    for b, js in enumerate(gone):
        keep = np.setdiff1d(np.arange(d.lens[b]), np.array(js, np.int64))
        for h in range(H):
            k, v = d.k[b][keep, h // (H // K)], d.v[b][keep, h // (H // K)]
            o, ls, tol = O.attention(q[b, h][None], k, v, [len(keep)], d.scale, dtype)
            within(got[b, h], o[0], tol[0], f"seq {b} head {h}")
            assert abs(got_lse[b, h] - ls[0]) <= lse_tol(q[b, h], k, d.scale, ls[0]), (b, h)


def test_performance_cases_are_ordered():
    """Their inputs, calls and outputs without a wait between (a program of its
    own: the library then uses the HIP runtime that torch brings)."""
    client = os.path.join(os.path.dirname(os.path.abspath(__file__)), "ordered_cases_client.py")
    r = subprocess.run([sys.executable, client], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and "ordered" in r.stdout, r.stdout + r.stderr
