"""GPU: the context operators as a program uses them: a workspace sized once
for all that is to come, scores of minus infinity, that every key counts once
and no other, one context on two streams, rows far apart, the performance
cases' order."""
import ctypes
import os
import subprocess
import sys

import numpy as np
import pytest

import context_oracle as O
import nmoe_hip as nh
from static_capture_client import hip
from test_gpu_context import Decode, Delta, Prompt, ctx, randn, within  # noqa: F401 (ctx is a fixture)

pytestmark = pytest.mark.gpu


def lse_tol(q, k, scale, lse):
    """The error of a logarithm of a sum of exponentials: the scores' (fp32
    sums of D products, D + 8 half steps of their magnitudes), the sum's own
    (half steps of n terms, added up as their root, twice over for the parts),
    the exponentials' 2^-21, and four half steps of the logarithm, of the
    maximum (in powers of two) and of what they add up to."""
    n, D = k.shape
    mag = (np.abs(k) @ np.abs(q)).max() * abs(scale)
    last = 4 * 2.0 ** -24 * (abs(lse) * 1.45 + 16 + mag)
    return (D + 8) * 2.0 ** -24 * mag + n ** 0.5 * 2.0 ** -23 + 2.0 ** -21 + last


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


def marked_keys(rng, n, count, step):
    """Key numbers below n: the first and the last, both sides of `step`'s multiples, and some more."""
    edges = np.arange(0, n + step, step)[:, None] + np.array([-1, 0])
    edges = np.concatenate([[0, n - 1], edges[(edges >= 0) & (edges < n)]])
    if len(edges) > count:
        edges = np.concatenate([edges[:2], rng.choice(edges, count - 2, replace=False)])
    return np.concatenate([edges, rng.integers(0, n, count - len(edges))]).astype(np.int64)


# equal scores: weights are exact powers of two and their sum is exact, so out is its one rounding and a division's
# (2^-22) off; lse is off by a step of log2 of up to 2^12 * 2^17 (2^-19), by its factor's rounding and its own (2^-21
# each): 0.7 * 2^-19 + 2^-20
LSE_OF_EQUALS = 2.0 ** -18


@pytest.mark.parametrize("dtype,H,K,D,page,lens", [
    (nh.BF16, 16, 2, 256, 16, [777, 1, 33, 128, 129]),
    (nh.F16, 8, 8, 128, 64, [4097, 31, 512]),
    (nh.BF16, 8, 8, 64, 48, [3000, 2, 96]),
    (nh.F16, 16, 2, 256, 256, [40000]),
    (nh.BF16, 2, 2, 128, 16, [65537]),
])
@pytest.mark.parametrize("max_len", [1, None])
def test_decode_every_key_counts(ctx, dtype, H, K, D, page, lens, max_len):  # noqa: F811
    """Equal scores, and a value of 1 at one key a dimension: out is 1 / len
    wherever that key was taken (once), and lse the logarithm of how many
    were."""
    rng = np.random.default_rng(42)
    d = Decode(ctx, rng, dtype, H, K, D, page, lens)
    d.q[:] = 0
    d.dq.upload(d.q)
    for b, n in enumerate(lens):
        v = np.zeros((n, K, D), np.float32)
        v[marked_keys(rng, n, K * D, 32).reshape(K, D), np.arange(K)[:, None], np.arange(D)] = 1.0
        j = np.arange(n)
        d.cache.put(1, d.table[b, j // page].astype(np.int64) * page + j % page, O.pack(v, dtype))
    d.cache.upload()
    d.run(max_len)
    ctx.sync()
    got, lse = d.read()
    for b, n in enumerate(lens):
        within(got[b], np.full((H, D), 1.0 / n), (O.HALF[dtype] + 2.0 ** -22) / n + O.TINY[dtype], f"seq {b}")
        assert (np.abs(lse[b] - np.log(n)) <= LSE_OF_EQUALS).all(), (b, lse[b] - np.log(n))


@pytest.mark.parametrize("dtype,H,K,D,lq,lk,causal", [
    (nh.BF16, 16, 2, 256, [130, 1, 33, 64], None, True),
    (nh.BF16, 32, 2, 256, [700], None, True),
    (nh.F16, 32, 2, 256, [1100], None, True),
    (nh.BF16, 64, 8, 256, [600, 500], None, True),
    (nh.F16, 8, 8, 64, [63, 65, 129, 7, 200], None, True),
    (nh.BF16, 32, 4, 64, [2100, 300], None, True),
    (nh.F16, 4, 2, 128, [40, 31], [2000, 65], True),
    (nh.BF16, 32, 2, 128, [333, 280], [900, 280], True),
    (nh.BF16, 64, 8, 128, [500, 600], None, True),
    (nh.F16, 4, 4, 128, [130, 9], [70, 0], True),
    (nh.BF16, 4, 2, 256, [70, 3], [513, 96], False),
])
def test_prompt_every_key_counts(ctx, dtype, H, K, D, lq, lk, causal):  # noqa: F811
    """The same for prompts, every query: the keys that it sees, once each."""
    rng = np.random.default_rng(43)
    p = Prompt(ctx, rng, dtype, H, K, D, lq, lk, causal)
    p.q[:] = 0
    marks = []
    v = np.zeros((p.nk, K, D), np.float32)
    for b in range(len(lq)):
        n = p.ck[b + 1] - p.ck[b]
        marks.append(marked_keys(rng, n, K * D, 32).reshape(K, D) if n else None)
        if n:
            v[p.ck[b] + marks[b], np.arange(K)[:, None], np.arange(D)] = 1.0
    p.v[:] = O.pack(v.reshape(p.nk, K * D), dtype)
    p.dev[0].upload(p.q)
    p.dev[2].upload(p.v)
    p.run()
    ctx.sync()
    got, lse = p.read()
    for b in range(len(lq)):
        nq, nk = p.cq[b + 1] - p.cq[b], p.ck[b + 1] - p.ck[b]
        see = np.clip(np.arange(nq) + 1 + nk - nq, 0, nk) if causal else np.full(nq, nk)
        rows = slice(p.cq[b], p.cq[b + 1])
        inv = np.where(see > 0, 1.0 / np.maximum(see, 1), 0.0)
        for h in range(H):
            want = (marks[b][h // (H // K)][None] < see[:, None]) * inv[:, None] if nk else np.zeros((nq, D))
            within(got[rows, h], want, (O.HALF[dtype] + 2.0 ** -22) * want + O.TINY[dtype], f"seq {b} head {h}")
            assert np.isneginf(lse[rows, h][see == 0]).all()
            assert (np.abs(lse[rows, h] - np.log(np.maximum(see, 1)))[see > 0] <= LSE_OF_EQUALS).all(), (b, h)


def test_one_context_two_streams(ctx):  # noqa: F811
    """Calls of one context on two streams at once, a workspace and outputs
    each: the bits of the same calls alone, every time."""
    hp, rng = hip(), np.random.default_rng(44)
    streams = [ctypes.c_void_p(), ctypes.c_void_p()]
    for s in streams:
        assert hp.hipStreamCreate(ctypes.byref(s)) == 0
    jobs = []
    for i in range(2):
        d = Decode(ctx, rng, nh.BF16, 16, 2, 256, 16, [3000, 5, 800 + i])
        r = Delta(ctx, rng, nh.BF16, 2, 4, 128, 128, [150, 20 + i])
        t = Delta(ctx, rng, nh.F32, 2, 4, 128, 128, [1] * (9 + i))
        wd = ctx.alloc(ctx.attn_decode_workspace(d.cache.desc, 16, 3, int(d.lens.max())))
        wr = ctx.alloc(ctx.delta_prompt_workspace(r.desc, 2, r.T))
        jobs.append((d, Prompt(ctx, rng, nh.F16, 4, 2, 128, [300, 100 + i]), r, t, wd, wr))

    def go(job, stream):
        d, p, r, t, wd, wr = job
        d.run(ws=wd, stream=stream)
        p.run(stream=stream)
        r.run(ws=wr, stream=stream)
        t.step(stream=stream)

    def bits(job):
        d, p, r, t = job[:4]
        return [x.tobytes() for x in (*d.read(), *p.read(), r.state(), t.state())]

    try:
        alone = []
        for job in jobs:
            go(job, None)
            ctx.sync()
            alone.append(bits(job))
        for _ in range(5):
            for job, s in zip(jobs, streams):
                go(job, s.value)
            for s in streams:
                assert hp.hipStreamSynchronize(s) == 0
            assert [bits(job) for job in jobs] == alone
        for d, p, r, t, _, _ in jobs:
            d.check()
            p.check()
            r.check()
            t.check()
    finally:
        for s in streams:
            assert hp.hipStreamDestroy(s) == 0


FAR = (1 << 24) - 8  # elements from one row to the next: 130 rows are past 2^31


def far_rows(ctx, parts):  # noqa: F811
    """Rows of several inputs side by side, FAR apart: where each begins."""
    n, es = parts[0].shape[0], parts[0].itemsize
    big = ctx.alloc(n * FAR * es)
    at = np.cumsum([0] + [p.shape[1] for p in parts])[:-1]
    for p, a in zip(parts, at):
        for i in range(n):
            big.upload(p[i], (i * FAR + int(a)) * es)
    return [big + int(a) * es for a in at]


def test_prompt_rows_far_apart(ctx):  # noqa: F811
    p = Prompt(ctx, np.random.default_rng(45), nh.BF16, 4, 2, 128, [70, 60], behind=0)
    q, k, v = far_rows(ctx, [p.q, p.k, p.v])
    p.desc = ctx.qkv_rows(q, k, v, nh.BF16, 4, 2, 128, FAR, 128, FAR, 128, FAR, 128)
    p.run()
    ctx.sync()
    p.check()


@pytest.mark.parametrize("lens", [[70, 60], [1] * 130])
def test_delta_rows_far_apart(ctx, lens):  # noqa: F811
    d = Delta(ctx, np.random.default_rng(46), nh.F16, 1, 2, 64, 64, lens, behind=0)
    d.dev[:3] = far_rows(ctx, [d.q, d.k, d.v])
    d.w = [FAR] * 3
    d.bind(d.dev[5], d.ds_out)
    d.w = [64, 64, 128]
    if len(lens) > 2:
        d.step()
    else:
        d.run()
    ctx.sync()
    d.check()


def test_append_rows_and_pages_far_apart(ctx):  # noqa: F811
    T, H, K, D, page, stride = 130, 2, 1, 64, 80, 3 << 30
    x = O.pack(randn(np.random.default_rng(47), T, H + 2 * K, D), nh.BF16)
    q, k, v = far_rows(ctx, [x[:, :H].reshape(T, -1), x[:, H].reshape(T, -1), x[:, H + 1].reshape(T, -1)])
    rows = ctx.qkv_rows(q, k, v, nh.BF16, H, K, D, FAR, D, FAR, D, FAR, D)
    half = page * K * D * 2  # v lies behind k
    big = ctx.alloc(stride * 2 + 2 * half)
    desc = ctx.kv_cache(big, big + half, nh.BF16, K, D, page, 2, stride, K * D, D)
    slots = np.arange(2 * page, dtype=np.int64)[::-1][:T].copy()
    q_out = ctx.alloc(T * H * D * 2)
    ctx._check(ctx.kv_append(desc, rows, None, T, ctx.to_device(np.zeros(T, np.int32)), ctx.to_device(slots), q_out))
    ctx.sync()
    np.testing.assert_array_equal(q_out.download(np.uint16, (T, H, D)), x[:, :H])
    for which in (0, 1):
        got = np.concatenate([big.download(np.uint16, (page, D), p * stride * 2 + which * half) for p in range(2)])
        np.testing.assert_array_equal(got[slots], x[:, H + which])


def test_performance_cases_are_ordered():
    """Their inputs, calls and outputs without a wait between (a program of its
    own: the library then uses the HIP runtime that torch brings)."""
    client = os.path.join(os.path.dirname(os.path.abspath(__file__)), "ordered_cases_client.py")
    r = subprocess.run([sys.executable, client], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and "ordered" in r.stdout, r.stdout + r.stderr
