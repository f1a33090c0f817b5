"""GPU: the context in 8 bits as a program uses it: batches of very unlike
lengths, a workspace sized once, that every key counts once and no other,
scores of minus infinity, pages far apart, appends in a captured graph, two
graphs on one workspace, the performance cases' order."""
import os
import subprocess
import sys

import numpy as np
import pytest

import context_oracle as O
import kv8_oracle as O8
import nmoe_hip as nh
from static_capture_client import hip
from test_gpu_context import ctx, randn, within  # noqa: F401 (ctx is a fixture)
from test_gpu_context_use import lse_tol
from test_gpu_graph import Graph
from test_gpu_kv8 import Append8, Attend8

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("H,K,D,lens,hint", [
    (4, 1, 64, [3] * 299 + [9000], None),
    (4, 1, 64, [9000] + [129] * 511, None),  # as many as half the blocks that run at once
    (4, 1, 64, [128] * 512 + [4100], None),
    (4, 1, 64, [7] * 300 + [12000] + [40] * 723, 1),  # too many to cut, by the hint
    (16, 2, 256, [20] * 60 + [7000, 0, 6000, 1], None),
    (16, 2, 256, [5, 1, 20000, 129], 2 ** 31 - 1),
    (32, 8, 128, [60] * 40 + [5000, 2049, 2048, 0], None),
    (2, 1, 64, [11] * 4095 + [3000], 3000),
    (2, 1, 64, [11] * 4096 + [3000], 3000),  # more than are looked through
])
def test_decode_unlike_lengths(ctx, H, K, D, lens, hint):  # noqa: F811
    """Every sequence is as by itself, however long the others are."""
    d = Attend8(ctx, np.random.default_rng(len(lens)), nh.BF16, H, K, D, 16, lens)
    d.run(hint)
    ctx.sync()
    far = np.argsort(lens)[-4:].tolist() + [0, 1, len(lens) - 1, len(lens) // 2]
    d.check(skip=set(range(len(lens))) - set(far))


def test_workspace_sized_once(ctx):  # noqa: F811
    """Sized for the most and the longest, then calls on fewer and shorter
    sequences; it holds NaN before each."""
    rng = np.random.default_rng(71)
    size = ws = None
    for lens, lq in (([9000], None), ([20] * 600 + [8000], None), ([9, 700, 4097], None), ([3], None), ([9000], [9]), ([5000, 20], [300, 20]),
                     ([2000, 1030, 7], [1, 1, 1])):
        d = Attend8(ctx, rng, nh.BF16, 4, 1, 64, 16, lens, lq=lq)
        if ws is None:
            size = max(ctx.attn8_decode_workspace(d.cache.desc, 4, 601, 9000), ctx.attn8_prompt_workspace(d.cache.desc, 4, 3, 330, 300, 9000))
            ws = ctx.alloc(size + 16)
        assert d.size() <= size
        ws.upload(np.full(size + 16, 0xFF, np.uint8))
        d.run(ws=ws)
        ctx.sync()
        d.ws = None
        d.check(skip=set(range(2, len(lens) - 2)))
        assert (ws.download(np.uint8, 16, size) == 0xFF).all()


@pytest.mark.parametrize("dtype", [nh.BF16, nh.F16])
@pytest.mark.parametrize("H,K,D,lens,lq", [
    (4, 1, 64, [131071, 1, 127, 128, 129, 2047, 2048, 2049, 0, 33], None),
    (16, 2, 256, [33000, 16, 4095], None), (8, 2, 128, [255, 5000, 31], None), (2, 1, 64, [70001], None),
    (4, 1, 64, [60000, 17, 64], [5, 17, 40]), (16, 2, 256, [20001, 100], [3, 100]), (8, 2, 128, [1000, 1, 130], [1000, 1, 129]),
])
def test_every_key_counts_once(ctx, dtype, H, K, D, lens, lq):  # noqa: F811
    """Equal scores, key j's value 1 in dimension j % D alone: the result is
    how often each comes, by the number of keys; both exact in fp32."""
    rng = np.random.default_rng(72)
    page = 64
    d = Attend8(ctx, rng, dtype, H, K, D, page, [1] * len(lens), lq=[1] * len(lens) if lq else None)  # its buffers made anew below
    d.lens, d.lq = np.array(lens, np.int32), lq
    per = -(-d.lens // page)
    from test_gpu_kv8 import Cache8
    d.cache = c = Cache8(ctx, rng, K, D, page, int(per.sum()) + 1)
    d.max_pages = int(per.max()) + 1
    d.table = np.full((len(lens), d.max_pages), 0x3FFFFFFF, np.int32)
    for x in c.codes:
        x[:] = 0x7F
    at = 0
    for b, p in enumerate(per):
        pages = d.table[b, :p] = c.order[at:at + p]
        at += p
        for j0 in range(0, lens[b], page):
            pg, m = pages[j0 // page], min(page, lens[b] - j0)
            c.codes[0][pg, :m] = 0
            c.codes[1][pg, :m] = 0
            for h in range(K):
                c.codes[1][pg, np.arange(m), h * D + (j0 + np.arange(m)) % D] = 0x38  # 1
            c.scales[0][pg] = c.scales[1][pg] = 1.0
    c.upload()
    d.cu = (np.cumsum([0, *(lq or [1] * len(lens))]) + (2 if lq else 0)).astype(np.int32)
    d.nq = int(d.cu[-1]) + (3 if lq else 1)
    d.dq = ctx.to_device(O.pack(randn(rng, d.nq, H, D), dtype))
    d.dlens, d.dtable, d.dcu = (ctx.to_device(t) for t in (d.lens, d.table, d.cu))
    d.out, d.lse = ctx.to_device(O.pack(np.full((d.nq, H, D), 9.0), dtype)), ctx.to_device(np.full(d.nq * H, 9.0, np.float32))
    d.run()
    ctx.sync()
    got, lse = d.read()
    for b, n in enumerate(lens):
        nq = d.cu[b + 1] - d.cu[b]
        for i in range(nq):
            see = n if lq is None else max(0, i + 1 + n - nq)
            t = d.cu[b] + i
            if see == 0:
                assert (got[t] == 0).all() and np.isneginf(lse[t]).all()
                continue
            want = np.bincount(np.arange(see) % D, minlength=D) / see
            # a quotient (two half steps) and its rounding; the logarithm: four half steps of what is added to it
            within(got[t], np.broadcast_to(want, (H, D)), want * (O.HALF[dtype] + 2.0 ** -22) + O.TINY[dtype], f"{b} {i}")
            assert np.abs(lse[t] - np.log(see)).max() <= 4 * 2.0 ** -24 * (1 + 1.45 * np.log(see)) + 2.0 ** -21


@pytest.mark.parametrize("dtype,H,K,D", [(nh.BF16, 16, 2, 256), (nh.F16, 4, 4, 128), (nh.F16, 7, 1, 64)])
@pytest.mark.parametrize("lq", [None, [3, 20, 1, 60, 1]])
def test_keys_of_minus_infinity(ctx, dtype, H, K, D, lq):  # noqa: F811
    """Keys whose score is minus infinity weigh nothing, also where a tile, a
    workgroup's turn or a whole part has no others."""
    gone = [range(0, 32), range(0, 128), range(128, 512), [*range(32, 300), 700, 707], range(0, 2048)]
    d = Attend8(ctx, np.random.default_rng(73), dtype, H, K, D, 16, [500, 300, 777, 901, 2200], lq=lq)
    q = O.value(d.q, dtype)
    q[..., 3] = -64.0
    d.q = O.pack(q, dtype)
    d.dq.upload(d.q)
    for b, js in enumerate(gone):
        js = np.array(js)
        for j0 in sorted({j // 16 * 16 for j in js}):
            pg = int(d.table[b, j0 // 16])
            m = min(16, d.lens[b] - j0)
            for h in range(K):  # the block: 448 * 2^118 for these, zeros for others; that times -64 is beyond fp32
                c = d.cache.block(0, pg, 0, h)
                c[:m] = 0
                c[js[(js >= j0) & (js < j0 + 16)] - j0, 3] = 0x7E
            d.cache.scales[0][pg, 0] = 2.0 ** 118
            d.k[b][j0:j0 + m] = 0.0
    d.cache.upload()
    d.run()
    ctx.sync()
    got, got_lse = d.read()
    q = O.value(d.q, dtype)
    for b, js in enumerate(gone):
        nq, n = d.cu[b + 1] - d.cu[b], d.lens[b]
        keep = np.setdiff1d(np.arange(n), np.array(js))
        for i in range(nq):
            seen = keep[keep <= (n if lq is None else i + n - nq)]
            for h in range(H):
                k, v = d.k[b][seen, h // (H // K)], d.v[b][seen, h // (H // K)]
                o, ls, tol = O.attention(q[d.cu[b] + i, h][None], k, v, [len(seen)], d.scale, dtype)
                within(got[d.cu[b] + i, h], o[0], tol[0], f"seq {b} query {i} head {h}")
                assert abs(got_lse[d.cu[b] + i, h] - ls[0]) <= lse_tol(q[d.cu[b] + i, h], k, d.scale, ls[0])


def test_attention_far_apart(ctx):  # noqa: F811
    """Pages 3 * 2^30 bytes apart, the second past 2^32, tokens 2^23 bytes apart within."""
    rng, stride, step = np.random.default_rng(74), 3 << 30, 1 << 23
    n, K, D, H = 40, 2, 64, 4
    big = ctx.alloc(2 * stride + 16 * step + (1 << 16))
    scales = [ctx.to_device(np.full((3, 1, K), 2.0 ** -7, np.float32)) for _ in range(2)]
    desc = ctx.kv8_cache(big, big + 4096, *scales, K, D, 16, 3, stride, step, D)
    codes = rng.integers(0, 0x7F, (2, n, K, D)).astype(np.uint8) | (rng.integers(0, 2, (2, n, K, D)) << 7).astype(np.uint8)
    order = [2, 0, 1]
    for which in (0, 1):
        for j in range(n):
            big.upload(codes[which, j], order[j // 16] * stride + j % 16 * step + 4096 * which)
    k, v = (O8.CODES[codes[w]] * 2.0 ** -7 for w in (0, 1))
    table, lens = ctx.to_device(np.array([order], np.int32)), ctx.to_device(np.array([n], np.int32))
    for nq in (1, 40):
        q = O.pack(0.3 * randn(rng, nq, H, D), nh.BF16)
        out, ws = ctx.alloc(nq * H * D * 2), ctx.alloc(1 << 20)
        if nq == 1:
            ctx._check(ctx.attn8_decode(desc, ctx.to_device(q), nh.BF16, H, 1, lens, table, 3, n, 0.125, out, None, ws, 1 << 20))
        else:
            ctx._check(ctx.attn8_prompt(desc, ctx.to_device(q), nh.BF16, H, 1, ctx.to_device(np.array([0, nq], np.int32)), nq, lens, table, 3,
                                        nq, n, True, 0.125, out, None, ws, 1 << 20))
        ctx.sync()
        got = O.value(out.download(np.uint16, (nq, H, D)), nh.BF16)
        for h in range(H):
            o, _, tol = O.attention(O.value(q, nh.BF16)[:, h], k[:, h // 2], v[:, h // 2], np.arange(n - nq + 1, n + 1), 0.125, nh.BF16)
            within(got[:, h], o, tol, f"{nq} queries, head {h}")


@pytest.mark.parametrize("new", [[1, 1, 1], [40, 0, 3]])
def test_append_replays(ctx, new):  # noqa: F811
    """A captured append follows rows and lengths: the same bits as eager
    ones into another cache, step after step."""
    jobs = [Append8(ctx, np.random.default_rng(75), nh.BF16, nh.BF16, 4, 2, 128, 16, "token", [9, 30, 0], [200, 200, 200]) for _ in (0, 1)]
    rng = np.random.default_rng(76)
    inv = ctx.to_device((1e6 ** (-np.arange(0, 64, 2) / 64)).astype(np.float32))
    cu, x = np.cumsum([0, *new]).astype(np.int32), [None, None]
    for a in jobs:
        a.T = int(cu[-1]) - 3  # no rows behind the last: a token each is as many as there are sequences
        a.dcu.upload(cu)
        a.dev = ctx.to_device(a.x)
        base, w, es = a.dev.ptr, a.width, 2
        a.rows = ctx.qkv_rows(base, base + 4 * 136 * es, base + 6 * 136 * es, nh.BF16, 4, 2, 128, w, 136, w, 136, w, 136)
        a.prep = ctx.qk_prep(64, inv, False, True, None, None, 0, 1e-6)
    graph = Graph(hip(), ctx.stream, lambda: jobs[1].run(jobs[1].prep))
    for a in jobs:  # the capture itself has run nothing
        a.cache.upload()
    lens = np.array([9, 30, 0], np.int32)
    for step in range(5):
        lens = lens + np.array(new, np.int32)
        rows = O.pack(2.0 ** (step - 2) * randn(rng, *jobs[0].x.shape), nh.BF16)
        for a in jobs:
            a.dlens.upload(lens)
            a.dev.upload(rows)
        jobs[0].run(jobs[0].prep)
        ctx.sync()
        graph.launch()
        ctx.sync()
        for a, b in zip(*(sum(map(list, a.cache.download()), []) for a in jobs)):
            np.testing.assert_array_equal(a, b)
        np.testing.assert_array_equal(jobs[0].q(), jobs[1].q())
    graph.close()


def test_two_graphs_one_workspace(ctx):  # noqa: F811
    """Decode and prompt captured with the same workspace, replayed in turns."""
    rng = np.random.default_rng(77)
    d = Attend8(ctx, rng, nh.BF16, 16, 2, 256, 16, [3000, 5, 800])
    p = Attend8(ctx, rng, nh.BF16, 4, 2, 128, 16, [2500, 100], [40, 100])
    ws = ctx.alloc(max(d.size(), p.size()) + 16)
    graphs = []
    for a in (d, p):
        a.run(ws=ws)
        ctx.sync()
        graphs.append((a, [t.tobytes() for t in a.read()], Graph(hip(), ctx.stream, lambda a=a: a.run(ws=ws))))
    for _ in range(3):
        for a, _, g in graphs:
            a.out.upload(O.pack(np.full((a.nq, a.H, a.D), 9.0), a.dtype))
            a.lse.upload(np.full(a.nq * a.H, 9.0, np.float32))
        for _, _, g in graphs:
            g.launch()
        ctx.sync()
        for a, bits, _ in graphs:
            assert [t.tobytes() for t in a.read()] == bits
            a.check(heads=[0, a.H - 1])
    for _, _, g in graphs:
        g.close()


def test_performance_cases_are_ordered():
    """As for the context in 16 bits."""
    client = os.path.join(os.path.dirname(os.path.abspath(__file__)), "ordered_cases8_client.py")
    r = subprocess.run([sys.executable, client], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and "ordered" in r.stdout, r.stdout + r.stderr
