"""GPU: the context operators as a program uses them: a workspace sized once
for all that is to come."""
import os
import subprocess
import sys

import numpy as np
import pytest

import nmoe_hip as nh
from test_gpu_context import Decode, ctx  # noqa: F401 (ctx is a fixture)

pytestmark = pytest.mark.gpu


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


def test_performance_cases_are_ordered():
    """Their inputs, calls and outputs without a wait between (a program of its
    own: the library then uses the HIP runtime that torch brings)."""
    client = os.path.join(os.path.dirname(os.path.abspath(__file__)), "ordered_cases_client.py")
    r = subprocess.run([sys.executable, client], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and "ordered" in r.stdout, r.stdout + r.stderr
