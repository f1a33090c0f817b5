"""GPU: the context in 8 bits at its edges: values and scores near fp32's
limits, lengths near 32 bits', hints and row counts far from what there
is, requests that a plan refuses, the searches for a row's sequence, offsets
that fall."""
import numpy as np
import pytest

import context_oracle as O
import kv8_oracle as O8
import nmoe_hip as nh
from static_capture_client import hip
from test_gpu_context import ctx, randn, within  # noqa: F401 (ctx is a fixture)
from test_gpu_context_use import lse_tol
from test_gpu_graph import Graph
from test_gpu_kv8 import Append8, Attend8, Cache8, Plan, mixed, test_append as append_case

pytestmark = pytest.mark.gpu


def blocks_of(d):
    """Every block that a sequence has tokens in: sequence, first token, page, block, tokens."""
    for b, n in enumerate(d.lens):
        for j0 in range(0, int(n), 16):
            yield b, j0, int(d.table[b, j0 // d.page]), j0 % d.page // 16, min(16, int(n) - j0)


# --------------------------------------------------- values and scores far out

@pytest.mark.parametrize("powers", [[118], [118, 100, 80, 20, -8]], ids=str)
@pytest.mark.parametrize("H,K,D,lens,lq", [
    (16, 2, 256, [300, 1, 5000], None), (4, 2, 64, [9000], None), (8, 2, 128, [20] * 40 + [2500], None),
    (4, 2, 64, [300, 40], [300, 40]), (16, 2, 256, [130, 17], [130, 2]), (8, 2, 128, [3000], [17]), (16, 2, 256, [5000], [3]),
])
def test_values_near_the_largest(ctx, H, K, D, lens, lq, powers):  # noqa: F811
    """Values up to 448 * 2^118: their mean is a number, so the result is."""
    rng = np.random.default_rng(len(powers))
    d = Attend8(ctx, rng, nh.BF16, H, K, D, 16, lens, lq=lq)
    for b, j0, pg, blk, m in blocks_of(d):
        e = rng.choice(powers, K)
        d.cache.scales[1][pg, blk] = 2.0 ** e
        for h in range(K):
            c = d.cache.block(1, pg, blk, h)
            c[:m] = rng.integers(0x70, 0x7F, (m, D))  # 128 to 448
            d.v[b][j0:j0 + m, h] = O8.CODES[c[:m]] * 2.0 ** e[h]
    d.cache.upload()
    d.run()
    ctx.sync()
    d.check(skip=set(range(2, len(lens) - 2)))


@pytest.mark.parametrize("H,K,D,lens,lq", [
    (16, 2, 256, [300, 64, 5000], None), (4, 2, 64, [90, 9000], None), (8, 2, 128, [60], None),
    (8, 2, 128, [64, 100], [64, 100]), (4, 2, 64, [300, 33], [300, 33]), (16, 2, 256, [130, 48], [130, 20]), (8, 2, 128, [3000], [17]),
])
def test_great_values_that_weigh_nothing(ctx, H, K, D, lens, lq):  # noqa: F811
    """Blocks of the greatest scale among those of the least, whose keys'
    scores are far below the others': neither queries that do not see them nor those that
    do lose a bit of the small values."""
    rng = np.random.default_rng(94)
    d = Attend8(ctx, rng, nh.BF16, H, K, D, 16, lens, lq=lq, spread=0.5)
    q = O.value(d.q, nh.BF16)
    q[..., 3] = 1.0
    d.q = O.pack(q, nh.BF16)
    d.dq.upload(d.q)
    for b, j0, pg, blk, m in blocks_of(d):
        great = j0 // 16 % 3 == 1 and j0 + 16 < d.lens[b]
        d.cache.scales[1][pg, blk] = 2.0 ** (118 if great else -117)
        for h in range(K):
            for which, x in ((0, d.k), (1, d.v)):
                c = d.cache.block(which, pg, blk, h)
                if which == 0 and great:
                    c[:m] = 0
                    c[:m, 3] = 0xFE  # -448 times 16: scores of -448 and less
                    d.cache.scales[0][pg, blk, h] = 2.0 ** 4
                if which == 1 and not great:
                    c[:m] = rng.integers(0x08, 0x19, (m, D))  # 2^-6 to 2^-4
                x[b][j0:j0 + m, h] = O8.CODES[c[:m]] * float(d.cache.scales[which][pg, blk, h])
    d.cache.upload()
    d.run()
    ctx.sync()
    d.check()


@pytest.mark.parametrize("lq", [None, [2, 30]])
def test_small_keys_great_queries(ctx, lq):  # noqa: F811
    """Codes of the least scale against queries of 2^117: what counts is the key's value, not its code."""
    d = Attend8(ctx, np.random.default_rng(81), nh.BF16, 16, 2, 256, 16, [700, 90], lq=lq, spread=2.0 ** 117)
    for b, j0, pg, blk, m in blocks_of(d):
        d.cache.scales[0][pg, blk] = 2.0 ** -117
        for h in range(2):
            d.k[b][j0:j0 + m, h] = O8.CODES[d.cache.block(0, pg, blk, h)[:m]] * 2.0 ** -117
    d.cache.upload()
    d.scale = 2.0 ** -11
    d.run()
    ctx.sync()
    d.check()


@pytest.mark.parametrize("dtype", [nh.BF16, nh.F16])
@pytest.mark.parametrize("lq", [None, [2, 30]])
def test_great_keys_small_queries(ctx, dtype, lq):  # noqa: F811
    """Queries of zero against keys of the greatest scale, times a scale of 2^12: scores of zero."""
    d = Attend8(ctx, np.random.default_rng(82), dtype, 4, 2, 64, 16, [300, 40], lq=lq)
    for b, j0, pg, blk, m in blocks_of(d):
        d.cache.scales[0][pg, blk] = 2.0 ** 118
        d.k[b][j0:j0 + m] = 0.0  # times zero
    d.cache.upload()
    q = O.value(d.q, dtype)
    d.q = O.pack(np.where(np.isnan(q), q, 0.0), dtype)
    d.dq.upload(d.q)
    d.scale = 2.0 ** 12
    d.run()
    ctx.sync()
    d.check()


@pytest.mark.parametrize("D", [64, 256])
def test_small_weights_of_small_values(ctx, D):  # noqa: F811
    """Keys of a 2^12.9th of the weight of four others, together as much as
    those, all of one value of the least scale: the mean is that value.  Among
    so many sequences none is cut, and each wavefront has one of the four."""
    d = Attend8(ctx, np.random.default_rng(83), nh.BF16, 4, 2, D, 16, [30000] + [1] * 511)
    q = O.value(d.q, nh.BF16)
    q[..., 3] = 1.0
    d.q, d.scale = O.pack(q, nh.BF16), 8.94
    d.dq.upload(d.q)
    for b, j0, pg, blk, m in blocks_of(d):
        for which in (0, 1):
            d.cache.scales[which][pg, blk] = 2.0 ** -117 if which else 1.0
            for h in range(2):
                c = d.cache.block(which, pg, blk, h)
                c[:m] = 0x78 if which else 0  # 256, or 0
                if j0 in (0, 32, 64, 96) and which == 0:
                    c[0, 3] = 0x38  # 1: a score of 8.94, 12.9 in powers of two
        d.k[b][j0:j0 + m], d.v[b][j0:j0 + m] = 0.0, 2.0 ** -109
        if j0 in (0, 32, 64, 96):
            d.k[b][j0, :, 3] = 1.0
    d.cache.upload()
    d.run(1)
    ctx.sync()
    d.check(heads=[0, 3], skip=set(range(3, 512)))


# ------------------------------------------------------------ plan, far lengths

def test_plan_lengths_near_the_largest(ctx):  # noqa: F811
    """A length of 32 bits does not wrap, though the table's row would hold more."""
    top, page, width = 2 ** 31 - 1, 1 << 30, 4
    lens, new = np.array([top, top - 5, top, 7], np.int32), np.array([100, 5, 0, 1], np.int32)
    up = lambda a: ctx.to_device(np.asarray(a))
    d = dict(lens=up(lens), new=up(new), free=up(np.array([1], np.int32)), stack=up(np.zeros(1, np.int32)),
             table=up(np.zeros((4, width), np.int32)), out=up(np.full(4, -9, np.int32)), count=up(np.zeros(1, np.int32)),
             cu=up(np.zeros(5, np.int32)), status=up(np.full(4, -9, np.int32)), positions=up(np.full(200, -9, np.int32)),
             slots=up(np.full(200, -9, np.int64)))
    req = ctx.kv_requests(page, 1, width, 200, d["lens"], d["new"], d["free"], d["stack"], d["table"], d["out"], d["count"],
                          d["cu"], d["status"], d["positions"], d["slots"])
    ctx._check(ctx.kv_plan(req, 4))
    ctx.sync()
    assert d["status"].download(np.int32, 4).tolist() == [1, 0, 0, 0]
    assert d["out"].download(np.int32, 4).tolist() == [top, top, top, 8]
    assert d["cu"].download(np.int32, 5).tolist() == [0, 0, 5, 5, 6]
    assert d["positions"].download(np.int32, 7).tolist() == [*range(top - 5, top), 7, 0]


# --------------------------------------------------- hints far from what there is

def written(d, size):
    """Words of the workspace that the last call wrote."""
    return int((d.ws.download(np.uint32, len(d.guard))[:size // 4] != d.guard[:size // 4]).sum())


@pytest.mark.parametrize("dtype,H,K,D,n", [
    (nh.BF16, 16, 2, 256, 1000), (nh.F16, 32, 8, 128, 777), (nh.BF16, 4, 1, 64, 3), (nh.BF16, 2, 2, 64, 40000), (nh.BF16, 8, 4, 128, 20000),
])
def test_decode_one_sequence_by_its_length(ctx, dtype, H, K, D, n):  # noqa: F811
    """One sequence is cut by its length, whatever max_len says: as many
    partial rows, the same bits; also where a piece does not begin where the hint has it."""
    d = Attend8(ctx, np.random.default_rng(n), dtype, H, K, D, 64, [n])
    seen = []
    for hint in (n, 1, 0, n // 2, 3 * n, 1 << 20, 2 ** 31 - 1):
        d.out.upload(O.pack(np.full((d.nq, H, D), 9.0), dtype))
        d.run(hint)
        ctx.sync()
        seen.append((written(d, d.size(hint)), *[t.tobytes() for t in d.read()]))
        if hint in (n, 1 << 20):
            d.check(heads=[0, H - 1])
    assert all(s == seen[0] for s in seen[1:]), [s[0] for s in seen]


def padded(d, ntok):
    """Its rows as the first of ntok, the others 9."""
    q = np.full((ntok, d.H, d.D), np.nan, np.float32)
    q[:d.nq] = O.value(d.q, d.dtype)
    d.q, d.nq = O.pack(q, d.dtype), ntok
    d.dq = d.ctx.to_device(d.q)
    d.out = d.ctx.to_device(O.pack(np.full((ntok, d.H, d.D), 9.0), d.dtype))
    d.lse = d.ctx.to_device(np.full(ntok * d.H, 9.0, np.float32))


@pytest.mark.parametrize("dtype,H,K,D,lens,lq", [
    (nh.BF16, 16, 2, 256, [9000], [96]), (nh.F16, 32, 8, 128, [5000], [12]), (nh.BF16, 8, 8, 64, [3000, 2900], [30, 30]),
])
def test_prompt_padded_rows(ctx, dtype, H, K, D, lens, lq):  # noqa: F811
    """Rows behind the last sequence's change nothing, neither the way a call
    is cut: the same bits, as many partial rows."""
    d = Attend8(ctx, np.random.default_rng(D), dtype, H, K, D, 64, lens, lq)
    seen = []
    for ntok in (d.nq, 512, 4096):
        padded(d, ntok)
        d.run()
        ctx.sync()
        got, lse = d.read()
        rows = slice(d.cu[0], d.cu[-1])
        seen.append((written(d, d.size()), got[rows].tobytes(), lse[rows].tobytes()))
        if ntok != 512:
            d.check(heads=[0, H - 1], rows=20)
    assert seen[0][0] > 0 and all(s == seen[0] for s in seen[1:]), [s[0] for s in seen]


@pytest.mark.parametrize("lens,lq,first", [([9000, 4000], [300, 700], 0), ([9000, 4000, 2000], [20, 700, 20], 0), ([5000, 3000], [20, 25], 900)])
@pytest.mark.parametrize("max_q", [1, 20, 2 ** 31 - 1])
def test_prompt_more_rows_than_hinted(ctx, lens, lq, first, max_q):  # noqa: F811
    """Sequences whose rows are more than the call was cut for, or lie far
    behind the first, are right, and nothing behind the workspace is written."""
    d = Attend8(ctx, np.random.default_rng(84), nh.BF16, 16, 2, 256, 64, lens, lq)
    if first:
        d.cu = (d.cu + first).astype(np.int32)
        d.dcu = ctx.to_device(d.cu)
        q = np.full((d.nq + first, 16, 256), np.nan, np.float32)
        q[first:] = O.value(d.q, nh.BF16)
        d.q, d.nq = O.pack(q, nh.BF16), d.nq + first
        padded(d, d.nq)
    d.run(max_len=30000, max_q=max_q)
    ctx.sync()
    d.check(heads=[0, 15], rows=20)


# ------------------------------------------------------ rows found by offsets

def by_rows(d, hint=None):
    """nmoe_attn8_decode_rows on a prompt's arguments, which has to leave all but each sequence's last row as it is."""
    ctx, n = d.ctx, len(d.lens)  # noqa: F811
    most = int(d.lens.max()) if hint is None else hint
    size = ctx.attn8_decode_workspace(d.cache.desc, d.H, n, most)
    d.guard = np.full(size // 4 + 8, 0x7FC12345, np.uint32)
    d.ws = ctx.to_device(d.guard)
    ctx._check(ctx.attn8_decode_rows(d.cache.desc, d.dq, d.dtype, d.H, n, d.dcu, d.nq, d.dlens, d.dtable, d.max_pages, most, d.scale,
                                     d.out, d.lse, d.ws, size))
    ctx.sync()


@pytest.mark.parametrize("dtype,H,K,D,lens,lq", [
    (nh.BF16, 16, 2, 256, [700, 300, 5000, 40, 33], [1, 0, 1, 0, 1]),
    (nh.F16, 32, 8, 128, [20, 2500, 9, 700], [0, 1, 3, 0]),
    (nh.BF16, 4, 1, 64, [9000], [1]), (nh.BF16, 4, 1, 64, [9000], [5]), (nh.F16, 7, 1, 64, [90], [0]),
    (nh.BF16, 4, 1, 64, [11] * 300 + [9000] + [7] * 299 + [4000], [1, 0, 2] * 100 + [0] + [1] * 299 + [1]),
    (nh.BF16, 2, 1, 64, [5] * 4200, [0, 1, 1] * 1400),  # a workgroup a sequence
])
@pytest.mark.parametrize("hint", [None, 1, 2 ** 31 - 1])
def test_decode_rows(ctx, dtype, H, K, D, lens, lq, hint):  # noqa: F811
    """The last row of each sequence that has one; the others', whatever their lengths, nowhere."""
    d = Attend8(ctx, np.random.default_rng(D + len(lens)), dtype, H, K, D, 16, lens, lq=lq)
    last = np.zeros(d.nq, bool)
    last[[d.cu[b + 1] - 1 for b in range(len(lens)) if lq[b]]] = True
    by_rows(d, hint)
    got, lse = d.read()
    assert (got[~last] == 9.0).all() and (lse[~last] == 9.0).all()
    np.testing.assert_array_equal(d.ws.download(np.uint32, len(d.guard))[-8:], d.guard[-8:])
    for b in [b for b in range(len(lens)) if lq[b]][:: max(1, len(lens) // 40)] + [len(lens) - 1] * bool(lq[-1]):
        t = d.cu[b + 1] - 1
        for h in range(0, H, 1 if H <= 16 else 5):
            k, v = d.k[b][:, h * K // H], d.v[b][:, h * K // H]
            q = O.value(d.q[t, h], dtype)
            o, ls, tol = O.attention(q[None], k, v, [lens[b]], d.scale, dtype)
            within(got[t, h], o[0], tol[0], f"seq {b} head {h}")
            assert abs(lse[t, h] - ls[0]) <= lse_tol(q, k, d.scale, ls[0])


def test_decode_rows_as_without_offsets(ctx):  # noqa: F811
    """With a row a sequence: the same bits as nmoe_attn8_decode, in place as well."""
    d = Attend8(ctx, np.random.default_rng(85), nh.BF16, 16, 2, 256, 16, [900, 1, 40, 3000])
    d.run()
    ctx.sync()
    want = [t[:4].tobytes() for t in d.read()]
    d.dcu = ctx.to_device(np.arange(5, dtype=np.int32))
    d.out = d.dq
    by_rows(d)
    assert [t[:4].tobytes() for t in d.read()] == want


def test_decode_rows_offsets_that_fall(ctx):  # noqa: F811
    """Offsets outside the rows, or falling: nothing outside out, lse and the
    workspace is written, nor a row that is no sequence's last."""
    d = Attend8(ctx, np.random.default_rng(86), nh.BF16, 4, 2, 128, 16, [50, 300, 20, 700], lq=[4, 5, 6, 2])
    rows = d.nq - 2  # two rows behind those of the call
    for cu, last in (([-100, 7, 3, 9, 10 ** 9], {6, 8, rows - 1}), ([2 ** 31 - 1, -2 ** 31, 5, -1, 2], {4, 1})):
        d.out.upload(O.pack(np.full((d.nq, 4, 128), 9.0), nh.BF16))
        d.lse.upload(np.full(d.nq * 4, 9.0, np.float32))
        d.dcu = ctx.to_device(np.array(cu, np.int32))
        d.nq -= 2
        by_rows(d)
        d.nq += 2
        got, lse = d.read()
        others = np.setdiff1d(np.arange(d.nq), list(last))
        assert (got[others] == 9.0).all() and (lse[others] == 9.0).all()
        np.testing.assert_array_equal(d.ws.download(np.uint32, len(d.guard))[-8:], d.guard[-8:])


@pytest.mark.parametrize("dtype", [nh.BF16, nh.F16])
def test_serving_behind_a_refused_request(ctx, dtype):  # noqa: F811
    """A loop of plan, append and decode in one graph, in which requests are
    refused, idle or end: every other one's result is of its own query and
    cache, by its own row."""
    rng, H, K, D, page, n, width, pages, rows = np.random.default_rng(87), 6, 2, 64, 16, 6, 5, 10, 120
    up = lambda a: ctx.to_device(np.asarray(a))
    cache = Cache8(ctx, rng, K, D, page, pages)
    lens, free = up(np.zeros(n, np.int32)), up(np.array([pages], np.int32))
    stack, table, new = up(rng.permutation(pages).astype(np.int32)), up(np.full((n, width), -1, np.int32)), up(np.zeros(n, np.int32))
    cu, status = up(np.zeros(n + 1, np.int32)), up(np.zeros(n, np.int32))
    req = ctx.kv_requests(page, pages, width, rows, lens, new, free, stack, table, lens, free, cu, status)
    qkv, q_ready, out = ctx.alloc(rows * (H + 2 * K) * D * 4), ctx.alloc(rows * H * D * 2), ctx.alloc(rows * H * D * 2)
    w = (H + 2 * K) * D
    desc = ctx.qkv_rows(qkv, qkv + H * D * 4, qkv + (H + K) * D * 4, nh.F32, H, K, D, w, D, w, D, w, D)
    size = ctx.attn8_decode_workspace(cache.desc, H, n, width * page)
    ws = ctx.alloc(size + 16)

    def step():
        ctx._check(ctx.kv_plan(req, n))
        ctx._check(ctx.kv8_append(cache.desc, desc, None, n, cu, rows, lens, table, width, None, q_ready, dtype))
        return ctx._check(ctx.attn8_decode_rows(cache.desc, q_ready, dtype, H, n, cu, rows, lens, table, width, width * page, D ** -0.5,
                                                out, None, ws, size))

    graph = Graph(hip(), ctx.stream, step)
    seen = set()
    #                10 pages: all taken; the last's page goes to the first, none is left for the second; ...
    for wish, want in (([32, 16, 17, 5, 40, 3], [0] * 6), ([1, 1, 1, 1, 0, -1], [0, 1, 0, 0, 0, 0]), ([1, 1, 1, 1, 1, 1], [0, 1, 0, 0, 0, 1]),
                       ([0, 1, -1, 1, 1, 1], [0] * 6), ([1, 1, 1, 1, 1, 1], [0, 0, 1, 0, 0, 0])):
        x = randn(rng, rows, H + 2 * K, D)
        qkv.upload(x)
        new.upload(np.array(wish, np.int32))
        out.upload(O.pack(np.full((rows, H, D), 9.0), dtype))
        ctx.sync()
        graph.launch()
        ctx.sync()
        got_status = status.download(np.int32, n).tolist()
        assert got_status == want, got_status
        seen |= set(got_status)
        at, got_lens, tab = cu.download(np.int32, n + 1), lens.download(np.int32, n), table.download(np.int32, (n, width))
        cache.codes, scales = cache.download()
        q, got = (O.value(t.download(O.NP[dtype], (rows, H, D)), dtype) for t in (q_ready, out))
        mine = np.zeros(rows, bool)
        for b in range(n):
            assert at[b + 1] - at[b] == (max(wish[b], 0) if got_status[b] == 0 else 0)
            if at[b + 1] == at[b]:
                continue
            m, t = int(got_lens[b]), at[b + 1] - 1
            mine[t] = True
            np.testing.assert_array_equal(q[t], O.value(O.pack(x[t, :H], dtype), dtype))
            values = [np.zeros((m, K, D)) for _ in range(2)]
            for j0 in range(0, m, 16):
                pg, blk, c = int(tab[b, j0 // page]), j0 % page // 16, min(16, m - j0)
                for which in (0, 1):
                    for h in range(K):
                        values[which][j0:j0 + c, h] = O8.CODES[cache.block(which, pg, blk, h)[:c]] * float(scales[which][pg, blk, h])
            for h in range(H):
                o, _, tol = O.attention(q[t, h][None], values[0][:, h * K // H], values[1][:, h * K // H], [m], D ** -0.5, dtype)
                within(got[t, h], o[0], tol[0], f"{wish} request {b} head {h}")
        assert (got[~mine] == 9.0).all()
    assert seen == {0, 1}
    graph.close()


# ------------------------------------------- searches for a row's sequence

def beside_the_window(a, token):
    """New rows (or, of blocks, units of new rows) whose sequence is not among
    the 64 looked at first; the kernels' arithmetic, on the host."""
    cu, n, ntok = a.cu.astype(np.int64), a.n, a.T + 3
    first = lambda row, b: row if token else row // 16 + 2 * b
    slots = ntok if token else ntok // 16 + 2 * n
    lane, missed = np.arange(64), 0
    for b in range(n):
        if a.new[b] == 0:
            continue
        begin = int(first(cu[b], b))
        blocks = (int(a.past[b]) % 16 + int(a.new[b]) + 15) // 16
        for slot in range(begin, begin + (int(a.new[b]) if token else blocks)):
            guess = min(max(int(np.float32(slot) / np.float32(slots) * np.float32(n)) - 31, 0), max(n - 63, 0))
            at = np.minimum(guess + lane, n)
            near = int(((guess + lane < n) & (first(np.clip(cu[at], 0, ntok), at) <= slot)).sum())
            missed += not (0 < near < 64 or n == 1)
    return missed


@pytest.mark.parametrize("new,token", [
    ([0] * 160 + [2] * 150, True), ([3] * 70 + [0] * 300 + [1] * 100, True), ([1] + [0] * 250 + [1, 1], True),
    ([300] * 20 + [1] * 280, False), ([1] * 280 + [300] * 20, False), ([0] * 200 + [40] * 90, False), ([20] * 150 + [0] * 5000, True), ([20] * 150 + [0] * 1000, False),
], ids=lambda v: f"{len(v)}x{sum(v)}" if isinstance(v, list) else None)
def test_append_sequences_looked_for(ctx, new, token):  # noqa: F811
    """Tokens that are a few sequences' of many: their sequence is not where it
    would be if all were alike."""
    past = np.random.default_rng(len(new)).integers(0, 40, len(new)) * (np.array(new) > 0)
    a = Append8(ctx, np.random.default_rng(1), nh.BF16, nh.BF16, 1, 1, 64, 16, "token", past, new)
    assert (a.T + 3 <= a.n) == token and beside_the_window(a, token) > 10 * (len(new) > 253)
    append_case(ctx, nh.BF16, nh.BF16, 1, 1, 64, 16, "token", 64, False, True, past, new, False)


def test_append_more_units_than_a_launch(ctx):  # noqa: F811
    """More pairs of block and heads than a launch has workgroups: they go on
    to further ones, with other sequences' angles."""
    rng, n, K, D, ntok = np.random.default_rng(88), 16400, 64, 64, 16500
    new = np.zeros(n, np.int64)
    new[:60], new[60:70], new[-79:] = 3, 17, rng.integers(1, 20, 79)
    past = rng.integers(0, 20, n) * (new > 0)
    a = Append8(ctx, rng, nh.BF16, nh.BF16, 0, K, D, 16, "token", past, new)
    assert (ntok // 16 + 2 * n) * (2 * K // 4) > 1 << 20 and ntok > n
    first = int(a.cu[n - 20]) // 16 + 2 * (n - 20)
    assert first * (2 * K // 4) > 1 << 20  # the last sequences' units are further ones
    x = ctx.alloc(ntok * a.width * 2)
    x.upload(a.x)
    at, w = (lambda head: x.ptr + head * (D + 8) * 2), a.width
    a.rows = ctx.qkv_rows(None, at(0), at(K), nh.BF16, 0, K, D, w, D + 8, w, D + 8, w, D + 8)
    inv = (1e6 ** (-np.arange(0, 32, 2) / 32)).astype(np.float32)
    prep = ctx.qk_prep(32, ctx.to_device(inv), False, False, None, None, 0, 1e-6)
    ctx._check(ctx.kv8_append(a.cache.desc, a.rows, prep, n, a.dcu, ntok, a.dlens, a.dtable, a.table.shape[1]))
    ctx.sync()
    codes, scales = a.cache.download()
    pos = np.zeros(a.T + 3, np.int64)
    for b in np.flatnonzero(new):
        pos[a.cu[b]:a.cu[b + 1]] = np.arange(past[b], past[b] + new[b])
    ready = O.prepared(a.values[:, :K], pos, inv, 32, False, False, None, False, 1e-6)
    blocks = list(a.blocks())
    there = [np.zeros(c.shape[:2], bool) for c in a.cache.codes]  # tokens that may change
    old = [c.copy() for c in a.cache.codes]
    for b, pg, blk, lo, row, m in blocks:
        for which in (0, 1):
            there[which][pg, 16 * blk:16 * blk + lo + m] = True
            for h in (0, 17, 63):
                a.cache.codes = codes
                got = a.cache.block(which, pg, blk, h)[lo:lo + m]
                value = ready[row:row + m, h] if which == 0 else a.values[row:row + m, K + h]
                e = float(scales[which][pg, blk, h])
                # half a step, half the smallest code; for keys 2^-15 of the largest for fp32 and the angles
                tol = np.maximum(2.0 ** -4 * np.abs(value), e * 2.0 ** -10) + (2.0 ** -15 * np.abs(value).max() if which == 0 else 0.0)
                within(O8.CODES[got] * e, value, tol, f"{b} {which} {h}")
    for which in (0, 1):
        assert (codes[which] == old[which])[~there[which]].all()


@pytest.mark.parametrize("n,page,longest,most,spare", [(5000, 16, 60, 9, 10), (4097, 32, 100, 20, -200), (65536, 16, 30, 2, 5)])
def test_plan_offsets_in_memory(ctx, n, page, longest, most, spare):  # noqa: F811
    """More requests than the rows' launch holds offsets of, and more rows than the first launch writes."""
    rng = np.random.default_rng(n)
    p = Plan(ctx, rng, page, *mixed(rng, n, longest, most), spare=spare)
    assert p.max_rows > 4096 and n > 4096
    p.run()
    ctx.sync()
    w = p.check()
    assert p.short == (w["status"] == 1).any()


# ------------------------------------------------------------- offsets that fall

class Guarded:
    """A device buffer of a host array, with words behind it that have to stay."""

    def __init__(self, ctx, host):  # noqa: F811
        self.host, self.bytes = host, np.frombuffer(np.ascontiguousarray(host).tobytes(), np.uint8)
        self.dev = ctx.to_device(np.concatenate([self.bytes, np.full(4096, 0xA5, np.uint8)]))

    def download(self):
        got = self.dev.download(np.uint8, len(self.bytes) + 4096)
        assert (got[len(self.bytes):] == 0xA5).all()
        return got[:len(self.bytes)].view(self.host.dtype).reshape(self.host.shape)


@pytest.mark.parametrize("cu,token", [([0, 20, 15, 31, 40], False), ([-100, 21, 10, 10 ** 9, 3], False), ([2 ** 31 - 1, -2 ** 31, 50, -1, 7], False),
                                      (None, True)])
def test_append_falling_offsets_stay_inside(ctx, cu, token):  # noqa: F811
    """Offsets outside the rows, or falling: nothing outside the buffers and
    the sequences' pages is touched, rows of no sequence neither, and a
    sequence beside them that shares no row is as it should be."""
    rng = np.random.default_rng(89)
    n = 64 if token else 4
    past, new = (rng.integers(0, 30, n), np.ones(n, np.int64)) if token else ([3, 20, 7, 9], [20, 11, 16, 9])
    a = Append8(ctx, rng, nh.BF16, nh.BF16, 2, 1, 64, 16, "token", past, new)
    ntok = 60 if token else a.T + 1  # two rows behind them, or more
    cu = np.array(rng.integers(-20, 90, n + 1) if cu is None else cu, np.int32)
    c, q = a.cache, O.pack(np.full((a.T + 3, 2, 64), 5.0), nh.BF16)
    parts = [Guarded(ctx, h) for h in (*c.codes, *c.scales, q)]
    desc = ctx.kv8_cache(*[p.dev for p in parts[:4]], 1, 64, 16, c.pages, 16 * c.row, c.row, 64)
    ctx._check(ctx.kv8_append(desc, a.rows, None, n, ctx.to_device(cu), ntok, a.dlens, a.dtable, a.table.shape[1], None, parts[4].dev, nh.BF16))
    ctx.sync()
    got = [p.download() for p in parts]
    spare = np.setdiff1d(np.arange(c.pages), a.table[a.table < c.pages])
    assert len(spare) == 2
    for g, p in zip(got[:4], parts):
        np.testing.assert_array_equal(g[spare], p.host[spare])
    np.testing.assert_array_equal(got[4][ntok:], q[ntok:])
    ends = np.clip(cu.astype(np.int64), 0, ntok)
    of_none = np.ones(a.T + 3, bool)
    for b in range(n):
        of_none[ends[b]:max(ends[b], ends[b + 1])] = False
    np.testing.assert_array_equal(got[4][of_none], q[of_none])
    if cu.tolist() == [0, 20, 15, 31, 40]:  # the last one: 9 rows behind 9 tokens
        np.testing.assert_array_equal(O.value(got[4][31:40], nh.BF16), a.values[31:40, :2])
        for blk, (lo, m, row) in enumerate(((9, 7, 31), (0, 2, 38))):
            pg = int(a.table[3, blk])
            for which in (0, 1):
                was = int(np.log2(c.scales[which][pg, 0, 0])) if lo else 0
                want, e = O8.append_block(a.values[row:row + m, 2 + which], lo, c.block(which, pg, 0, 0), was)
                np.testing.assert_array_equal(got[which][pg, :, :64], want)
                np.testing.assert_array_equal(got[which][pg, :, 64:], c.codes[which][pg, :, 64:])
                assert got[2 + which][pg, 0, 0] == 2.0 ** e


@pytest.mark.parametrize("max_len", [300, 30000])
@pytest.mark.parametrize("cu", [[5, 25, 12, 40, 47], [-100, 40, 10, 10 ** 9, 3], [2 ** 31 - 1, -2 ** 31, 50, -1, 60]], ids=str)
def test_prompt_falling_offsets_stay_inside(ctx, cu, max_len):  # noqa: F811
    """The same of the attention, whole and in parts."""
    d = Attend8(ctx, np.random.default_rng(90), nh.BF16, 4, 2, 128, 16, [50, 300, 20, 60], [10, 30, 20, 7])
    rows = d.nq - 2  # two rows behind those of the call
    q = np.random.default_rng(91).standard_normal(d.q.shape).astype(np.float32)
    d.q = O.pack(q, nh.BF16)
    d.dq.upload(d.q)
    d.cu = np.array(cu, np.int64)
    d.dcu.upload(np.array(cu, np.int32))
    out, lse = Guarded(ctx, O.pack(np.full((d.nq, 4, 128), 9.0), nh.BF16)), Guarded(ctx, np.full((d.nq, 4), 9.0, np.float32))
    d.out, d.lse = out.dev, lse.dev
    d.nq -= 2
    d.run(max_len=max_len, max_q=30)
    ctx.sync()
    d.nq += 2
    np.testing.assert_array_equal(d.ws.download(np.uint32, len(d.guard))[-8:], d.guard[-8:])
    got, got_lse, ends = O.value(out.download(), nh.BF16), lse.download(), np.clip(d.cu, 0, rows)
    of_none = np.ones(d.nq, bool)
    for b in range(4):
        of_none[ends[b]:max(ends[b], ends[b + 1])] = False
    assert (got[of_none] == 9.0).all() and (got_lse[of_none] == 9.0).all()
    if cu[0] == 5:  # the last one: 7 rows of 60
        for h in range(4):
            k, v, rows3 = d.k[3][:, h // 2], d.v[3][:, h // 2], np.arange(40, 47)
            o, ls, tol = O.attention(O.value(d.q, nh.BF16)[rows3, h], k, v, np.arange(54, 61), d.scale, nh.BF16)
            within(got[rows3, h], o, tol, f"head {h}")


@pytest.mark.parametrize("dtype", [nh.BF16, nh.F16])
def test_one_query_is_as_decode(ctx, dtype):  # noqa: F811
    """Decode, and prompts of one query: apart by no more than both may be off."""
    d = Attend8(ctx, np.random.default_rng(92), dtype, 16, 2, 256, 16, [900, 1, 40, 3000])
    p = Attend8(ctx, np.random.default_rng(92), dtype, 16, 2, 256, 16, [900, 1, 40, 3000], [1, 1, 1, 1])
    p.q[2:6] = d.q[:4]
    p.dq.upload(p.q)
    d.run()
    p.run()
    ctx.sync()
    one, other = d.read()[0][:4], p.read()[0][2:6]
    q = O.value(d.q, dtype)
    for b, n in enumerate(d.lens):
        for h in range(16):
            np.testing.assert_array_equal(d.k[b], p.k[b])
            _, _, tol = O.attention(q[b, h][None], d.k[b][:, h // 8], d.v[b][:, h // 8], [n], d.scale, dtype)
            within(one[b, h], other[b, h], 2 * tol[0], f"seq {b} head {h}")


@pytest.mark.parametrize("dtype,H,K,D", [(nh.BF16, 16, 2, 256), (nh.F16, 6, 2, 64)])
def test_step_in_two_calls(ctx, dtype, H, K, D):  # noqa: F811
    """One step's requests, pieces of prompts first and single tokens behind
    them: the pieces by one call, the tokens by another, on the same offsets,
    rows and outputs."""
    lens, lq = [200, 90, 1, 3000, 500, 17, 700], [70, 90, 1, 1, 0, 1, 1]
    d = Attend8(ctx, np.random.default_rng(93), dtype, H, K, D, 16, lens, lq)
    first, n, most = 2, len(lens), max(lens)
    size = max(ctx.attn8_prompt_workspace(d.cache.desc, H, first, d.nq, 90, 200), ctx.attn8_decode_workspace(d.cache.desc, H, n - first, most))
    ws = ctx.alloc(size + 16)
    ctx._check(ctx.attn8_prompt(d.cache.desc, d.dq, dtype, H, first, d.dcu, d.nq, d.dlens, d.dtable, d.max_pages, 90, 200, True, d.scale,
                                d.out, d.lse, ws, size))
    ctx._check(ctx.attn8_decode_rows(d.cache.desc, d.dq, dtype, H, n - first, d.dcu.ptr + 4 * first, d.nq, d.dlens.ptr + 4 * first,
                                     d.dtable.ptr + 4 * first * d.max_pages, d.max_pages, most, d.scale, d.out, d.lse, ws, size))
    ctx.sync()
    d.check()
