"""GPU: the operators on a cache in 8 bits against plain 64-bit forms
(kv8_oracle.py, context_oracle.py): a step's pages, the append, decode and
prompt attention; types, head layouts, page sizes and layouts, lengths of zero
and one, odd and long ones, rows, codes and scales that must stay as they
were, values that must not be read, replays of captured graphs, calls on two
streams, and all of them together as a program runs them."""
import ctypes

import numpy as np
import pytest

import context_oracle as O
import kv8_oracle as O8
import nmoe_hip as nh
from static_capture_client import hip
from test_gpu_context import ctx, randn, within  # noqa: F401 (ctx is a fixture)
from test_gpu_context_use import lse_tol
from test_gpu_graph import Graph

pytestmark = pytest.mark.gpu


# -------------------------------------------------------------------- plan

class Plan:
    """Requests with random pages, every array with a word behind its end."""

    def __init__(self, ctx, rng, page, lens, new, spare=5, max_rows=None, extra=2, rows=True):  # noqa: F811
        self.ctx, self.page, self.n = ctx, page, len(lens)
        self.lens, self.new = np.array(lens, np.int32), np.array(new, np.int32)
        fair = np.clip(self.lens, 0, 1 << 20)
        up = lambda v: -(-v // page)
        self.width = int(up(fair + np.maximum(self.new, 0)).max(initial=1)) + extra
        used = up(fair)
        need = np.where(self.new > 0, up(fair + np.maximum(self.new, 0)) - used, 0).sum()
        free = max(0, int(need) - int(used[self.new < 0].sum()) + spare)  # pages that come back counted
        self.short = int(need) > int(used[self.new < 0].sum()) + free
        self.pages = int(used.sum()) + free + 3
        order = rng.permutation(self.pages).astype(np.int32)
        self.table = np.full((self.n, self.width), -7, np.int32)
        held = np.arange(self.width)[None] < used[:, None]
        self.table[held] = order[:used.sum()]
        self.stack = order[used.sum():used.sum() + free]
        self.max_rows = int(np.maximum(self.new, 0).sum()) + 3 if max_rows is None else max_rows
        self.mem = mem = np.full(self.pages + 1, -9, np.int32)
        mem[:free] = self.stack
        up32 = lambda a, k: ctx.to_device(np.concatenate([np.asarray(a, np.int32).ravel(), np.full(k, -9, np.int32)]))
        self.d = dict(lens=up32(self.lens, 1), new=up32(self.new, 1), free=up32([free], 1), stack=ctx.to_device(mem),
                      table=up32(self.table, 1), lens_out=up32([], self.n + 1), free_out=up32([], 2), cu=up32([], self.n + 2),
                      status=up32([], self.n + 1), positions=up32([], self.max_rows + 1),
                      slots=ctx.to_device(np.full(self.max_rows + 1, -9, np.int64)))
        self.rows = rows

    def desc(self, **kw):
        d = dict(self.d, **kw)
        return self.ctx.kv_requests(self.page, self.pages, self.width, self.max_rows, d["lens"], d["new"], d["free"], d["stack"],
                                    d["table"], d["lens_out"], d["free_out"], d["cu"], d["status"],
                                    d["positions"] if self.rows else None, d["slots"] if self.rows else None)

    def run(self, stream=None, **kw):
        return self.ctx._check(self.ctx.kv_plan(self.desc(**kw), self.n, stream))

    def want(self):
        return O8.plan(self.lens, self.new, self.stack, self.table, self.page, self.pages, self.max_rows)

    def check(self, inplace=False):
        w = self.want()
        get = lambda name, k, t=np.int32: self.d[name].download(t, k)
        lens = get("lens" if inplace else "lens_out", self.n + 1)
        free = get("free" if inplace else "free_out", 2)
        np.testing.assert_array_equal(lens, [*w["lens"], -9])
        assert free.tolist()[0] == w["free"]
        np.testing.assert_array_equal(get("cu", self.n + 2), [*w["cu"], -9])
        np.testing.assert_array_equal(get("status", self.n + 1), [*w["status"], -9])
        np.testing.assert_array_equal(get("table", self.table.size + 1), [*w["table"].ravel(), -9])
        stack = get("stack", self.pages + 1)
        np.testing.assert_array_equal(stack[:len(w["stack"])], w["stack"])
        np.testing.assert_array_equal(stack[len(w["stack"]):], self.mem[len(w["stack"]):])
        rows = [w["positions"], w["slots"]] if self.rows else [np.full(self.max_rows, -9)] * 2
        np.testing.assert_array_equal(get("positions", self.max_rows + 1), [*rows[0], -9])
        np.testing.assert_array_equal(get("slots", self.max_rows + 1, np.int64), [*rows[1], -9])
        return w


def mixed(rng, n, longest, most):
    lens = (rng.integers(0, longest + 1, n) * (rng.random(n) < 0.8)).astype(np.int64)
    new = np.where(rng.random(n) < 0.6, 1, rng.integers(0, most + 1, n))
    new[rng.random(n) < 0.15] = -1
    return lens, new


@pytest.mark.parametrize("n,page,longest,most,spare,rows", [
    (1, 16, 100, 40, 0, True), (7, 48, 200, 300, 2, True), (64, 64, 900, 5, 4, False), (300, 16, 70, 33, -30, True),
    (1024, 32, 100, 3, 0, True), (1025, 16, 50, 3, -200, True), (3000, 16, 90, 20, 10, True), (257, 256, 3000, 200, 1, True),
    (40, 16, 0, 3000, -500, True), (2500, 16, 40, 1, -40, False),
])
def test_plan(ctx, n, page, longest, most, spare, rows):  # noqa: F811
    rng = np.random.default_rng(n + page)
    p = Plan(ctx, rng, page, *mixed(rng, n, longest, most), spare=spare, rows=rows)
    p.run()
    ctx.sync()
    w = p.check()
    assert p.short == (w["status"] == 1).any()


@pytest.mark.parametrize("lens,new,max_rows,extra", [
    ([0], [0], 0, 1), ([0], [1], 1, 0), ([16], [1], 1, 0), ([15, 16, 17], [1, 1, 1], 3, 0), ([5], [-1], 4, 0),
    ([40, 0, 3], [-1, -5, -2 ** 31], 2, 0), ([10, 20, 30], [5, 90, 5], 50, 0),  # rows for the first and, too late, the third
    ([10, 20, 30], [0, 90, 0], 50, 3), ([3, -1, 7, 10 ** 6, 9], [4, 4, -1, -1, 2], 100, 2),  # lengths that cannot be
    ([100, 7], [2 ** 31 - 1, 3], 9, 0),  # more than a row of the table holds
])
def test_plan_edges(ctx, lens, new, max_rows, extra):  # noqa: F811
    rng = np.random.default_rng(len(lens))
    p = Plan.__new__(Plan)
    fair = [v for v in lens if 0 <= v < 1000]
    Plan.__init__(p, ctx, rng, 16, [v if v in fair else 0 for v in lens], [min(v, 500) for v in new], max_rows=max_rows, extra=extra)
    p.lens, p.new = np.array(lens, np.int32), np.array(new, np.int32)
    p.d["lens"].upload(p.lens)
    p.d["new"].upload(p.new)
    p.run()
    ctx.sync()
    p.check()


def test_plan_none(ctx):  # noqa: F811
    """No requests: offsets, the stack's count and the padded rows are written."""
    p = Plan(ctx, np.random.default_rng(0), 16, [], [], max_rows=5)
    p.run()
    ctx.sync()
    p.check()


def test_plan_stack_count_out_of_range(ctx):  # noqa: F811
    """A count below zero is none; one above num_pages, and pages that come
    back beyond it, are as many as there can be."""
    rng = np.random.default_rng(3)
    for count in (-4, 10 ** 9):
        p = Plan(ctx, rng, 16, [33, 20], [-1, 100])
        p.d["free"].upload(np.array([count], np.int32))
        p.stack = np.zeros(0, np.int32) if count < 0 else p.d["stack"].download(np.int32, p.pages)
        p.run()
        ctx.sync()
        p.check()


def test_plan_in_place_and_replayed(ctx):  # noqa: F811
    """lens and the stack's count updated in place, step after step by one
    graph, with new wishes in between, until pages run out and come back."""
    rng, page = np.random.default_rng(9), 16
    p = Plan(ctx, rng, page, rng.integers(0, 60, 50), np.zeros(50, np.int64), spare=30, max_rows=500, extra=20)
    g = Graph(hip(), ctx.stream, lambda: p.run(lens_out=p.d["lens"], free_out=p.d["free"]))
    seen = set()
    for step in range(12):
        p.new = np.where(rng.random(50) < 0.1, -1, rng.integers(0, 25, 50)).astype(np.int32)
        p.d["new"].upload(p.new)
        for name in ("positions", "slots"):
            p.d[name].upload(np.full(p.max_rows + 1, -9, np.int64 if name == "slots" else np.int32))
        ctx.sync()
        g.launch()
        ctx.sync()
        w = O8.plan(p.lens, p.new, p.stack, p.table, page, p.pages, p.max_rows)
        np.testing.assert_array_equal(p.d["lens"].download(np.int32, 50), w["lens"])
        np.testing.assert_array_equal(p.d["table"].download(np.int32, p.table.shape), w["table"])
        np.testing.assert_array_equal(p.d["slots"].download(np.int64, p.max_rows), w["slots"])
        np.testing.assert_array_equal(p.d["positions"].download(np.int32, p.max_rows), w["positions"])
        np.testing.assert_array_equal(p.d["status"].download(np.int32, 50), w["status"])
        assert p.d["free"].download(np.int32, 1)[0] == w["free"]
        p.lens, p.table, p.stack = w["lens"], w["table"], w["stack"][:w["free"]]
        held = [int(v) for b in range(50) for v in p.table[b, :-(-int(p.lens[b]) // page)]]
        assert len(set(held)) == len(held) and not set(held) & set(p.stack.tolist())  # no page twice
        seen |= set(w["status"].tolist())
    assert seen == {0, 1}
    g.close()


# ------------------------------------------------------------------ append

class Cache8:
    """A paged cache in 8 bits, its pages dealt at random; codes and scales
    `fill` until they are put."""

    def __init__(self, ctx, rng, heads, dim, page, pages, layout="token", gap=0, fill=0x7F):  # noqa: F811
        self.ctx, self.heads, self.dim, self.page, self.pages, self.layout = ctx, heads, dim, page, pages, layout
        self.row = heads * dim + gap
        shape = (pages, page, self.row) if layout == "token" else (pages, heads, page, dim)
        self.codes = [np.full(shape, fill, np.uint8) for _ in range(2)]
        self.scales = [np.full((pages, page // 16, heads), np.nan, np.float32) for _ in range(2)]
        self.dev = [ctx.to_device(h) for h in self.codes + self.scales]
        st = (page * self.row, self.row, dim) if layout == "token" else (heads * page * dim, dim, page * dim)
        self.desc = ctx.kv8_cache(*self.dev, heads, dim, page, pages, *st)
        self.order = rng.permutation(pages).astype(np.int32)

    def block(self, which, page, blk, head):
        """View of a block's codes [16, dim]."""
        c, s = self.codes[which], slice(16 * blk, 16 * blk + 16)
        return c[page, s, head * self.dim:(head + 1) * self.dim] if self.layout == "token" else c[page, head, s]

    def upload(self):
        for h, d in zip(self.codes + self.scales, self.dev):
            d.upload(h)

    def download(self):
        got = [d.download(h.dtype, h.shape) for h, d in zip(self.codes + self.scales, self.dev)]
        return got[:2], got[2:]


class Append8:
    """Sequences with tokens before (random codes) and new rows, of a
    projection with a gap behind each head and token."""

    def __init__(self, ctx, rng, src, dst, H, K, D, page, layout, past, new, gap=8, spread=1.0, x=None):  # noqa: F811
        self.ctx, self.src, self.dst, self.H, self.K, self.D, self.page = ctx, src, dst, H, K, D, page
        self.past, self.new = np.array(past, np.int64), np.array(new, np.int64)
        self.n, self.T = len(new), int(np.sum(new))
        lens = self.past + self.new
        per = -(-lens // page)
        self.cache = c = Cache8(ctx, rng, K, D, page, int(per.sum()) + 2, layout, gap=16 if layout == "token" else 0, fill=0x55)
        self.table = np.full((self.n, int(per.max()) + 1), 0x3FFFFFFF, np.int32)
        at = 0
        for b, p in enumerate(per):
            self.table[b, :p] = c.order[at:at + p]
            at += p
        for b in range(self.n):
            for j0 in range(0, int(self.past[b]), 16):
                pg, blk = int(self.table[b, j0 // page]), j0 % page // 16
                for which in (0, 1):
                    for h in range(K):
                        c.block(which, pg, blk, h)[:] = rng.integers(0, 0x7F, (16, D)) | rng.integers(0, 2, (16, D)) << 7
                        c.scales[which][pg, blk, h] = 2.0 ** rng.integers(-9, -4)
        c.upload()
        self.cu = (np.cumsum([0, *self.new]) + 1).astype(np.int32)  # a row before the first
        rows = self.T + 3
        self.width = (H + 2 * K) * (D + gap) + 16
        if x is None:
            x = spread * randn(rng, rows, self.width) * np.exp(0.7 * randn(rng, 1, self.width))
        self.x = O.pack(x, src)
        dx, es = ctx.to_device(self.x), 4 if src == nh.F32 else 2
        at = lambda head: dx.ptr + head * (D + gap) * es
        w = self.width
        self.rows = ctx.qkv_rows(at(0) if H else None, at(H), at(H + K), src, H, K, D, w, D + gap, w, D + gap, w, D + gap)
        self.values = O.value(self.x, src)[:, :(H + 2 * K) * (D + gap)].reshape(rows, H + 2 * K, D + gap)[..., :D]
        self.q_out = ctx.to_device(O.pack(np.full((rows, max(H, 1), D), 5.0), dst))
        self.lens = lens.astype(np.int32)
        self.dcu, self.dlens, self.dtable = (ctx.to_device(a) for a in (self.cu, self.lens, self.table))

    def run(self, prep=None, positions=None, stream=None):
        return self.ctx._check(self.ctx.kv8_append(self.cache.desc, self.rows, prep, self.n, self.dcu, self.T + 3, self.dlens,
                                                   self.dtable, self.table.shape[1], positions, self.q_out if self.H else None,
                                                   self.dst, stream))

    def q(self):
        return O.value(self.q_out.download(O.NP[self.dst], (self.T + 3, max(self.H, 1), self.D)), self.dst)

    def blocks(self):
        """Each new block: sequence, page, block, first new place, first token's row, rows."""
        for b in range(self.n):
            begin, end = int(self.past[b]), int(self.lens[b])
            for j0 in range(begin // 16 * 16, end, 16):
                lo, hi = max(begin - j0, 0), min(end - j0, 16)
                if lo < hi:
                    yield b, int(self.table[b, j0 // self.page]), j0 % self.page // 16, lo, int(self.cu[b]) + j0 + lo - begin, hi - lo


SHAPES = [
    (nh.BF16, nh.BF16, 16, 2, 256, 16, "token", 64, False, True, [0], [1]),
    (nh.BF16, nh.BF16, 16, 2, 256, 64, "head", 64, False, True, [37, 0, 5, 16], [37, 0, 1, 130]),
    (nh.F32, nh.F16, 6, 2, 64, 48, "token", 64, True, True, [1, 47, 95, 200, 15], [19, 1, 1, 1, 1]),
    (nh.F32, nh.BF16, 5, 1, 128, 32, "head", 128, False, False, [3], [5]),
    (nh.F16, nh.F16, 8, 8, 64, 16, "token", 16, False, True, [0, 100], [70, 16]),
    (nh.F16, nh.BF16, 4, 4, 128, 16, "token", 32, True, False, [16, 17], [3, 15]),
    (nh.BF16, nh.F16, 0, 3, 256, 16, "head", 256, True, True, [7], [9]),
    (nh.F32, nh.BF16, 33, 11, 64, 16, "token", 0, False, False, [31], [2]),
    (nh.BF16, nh.BF16, 2, 1, 256, 16, "token", 240, False, True, [500], [600]),
    (nh.BF16, nh.BF16, 1, 1, 64, 16, "token", 64, False, True, [0] * 130, [1] * 130),
    (nh.F32, nh.F16, 20, 4, 256, 256, "head", 64, True, True, [250, 4], [290, 77]),
    # no more tokens than sequences: a token each, several of one block, several blocks of one, none
    (nh.F16, nh.F16, 7, 1, 64, 16, "token", 32, False, True, [5, 16, 31, 0, 100, 9, 3, 2], [1, 1, 0, 3, 1, 0, 1, 1]),
    (nh.F32, nh.BF16, 32, 8, 128, 48, "head", 128, True, True, [40] + [7] * 40, [41] + [0] * 40),
    (nh.BF16, nh.BF16, 16, 2, 256, 64, "token", 64, False, True, [3] * 69 + [700], [0] * 30 + [1] * 38 + [2, 0]),
    # a block a head, its steps shared by the wavefronts: older codes before the new ones, blocks of one row, none
    (nh.BF16, nh.BF16, 16, 2, 256, 16, "token", 64, False, True, [15, 3, 14, 0, 32, 5], [3, 30, 1, 0, 17, 10]),
    (nh.F16, nh.BF16, 4, 4, 128, 48, "head", 0, False, False, [1, 9, 47], [40, 5, 2]),
    (nh.F32, nh.F16, 0, 8, 64, 16, "token", 32, True, False, [9, 8, 30], [3, 8, 70]),
    # more blocks than run at once
    (nh.BF16, nh.BF16, 33, 11, 128, 16, "token", 64, False, True, [7, 100], [650, 3]),
]


@pytest.mark.parametrize("src,dst,H,K,D,page,layout,rot,inter,norm,past,new", SHAPES)
@pytest.mark.parametrize("given", [False, True])
def test_append(ctx, src, dst, H, K, D, page, layout, rot, inter, norm, past, new, given):  # noqa: F811
    rng = np.random.default_rng(sum(new) + D + given)
    a = Append8(ctx, rng, src, dst, H, K, D, page, layout, past, new, spread=3.0)
    inv = (1e6 ** (-np.arange(0, max(rot, 2), 2) / max(rot, 2))).astype(np.float32)
    weights = [O.pack(0.2 * randn(rng, D), nh.BF16) for _ in range(2)]
    prep = ctx.qk_prep(rot, ctx.to_device(inv), inter, norm, ctx.to_device(weights[0]), ctx.to_device(weights[1]), 1, 1e-6)
    pos = rng.integers(0, 1 << 21, a.T + 3).astype(np.int32)
    if not given:
        for b in range(a.n):
            pos[a.cu[b]:a.cu[b + 1]] = np.arange(past[b], past[b] + new[b])
    a.run(prep, ctx.to_device(pos) if given else None)
    ctx.sync()
    v = a.values
    ready = [O.prepared(v[:, lo:hi], pos, inv, rot, inter, norm, O.value(w, nh.BF16), True, 1e-6)
             for lo, hi, w in ((0, H, weights[0]), (H, H + K, weights[1]))]
    # fp32 before the one rounding: the sum of D squares and its root (2^-17), the weight, the products of the rotation,
    # an angle good to 2^-20 turns: 2^-16 of the row's largest value, 2^-16 * 2 pi for the angle
    slack = lambda w: 2.0 ** -15 * np.abs(w).max(axis=-1, keepdims=True)
    q, rows = a.q(), slice(a.cu[0], a.cu[-1])
    if H:
        within(q[rows], ready[0][rows], O.HALF[dst] * np.abs(ready[0][rows]) + slack(ready[0][rows]) + O.TINY[dst], "q")
    assert (q[:rows.start] == 5.0).all() and (q[rows.stop:] == 5.0).all()
    codes, scales = a.cache.download()
    want_codes, want_scales = [c.copy() for c in a.cache.codes], [s.copy() for s in a.cache.scales]
    for b, pg, blk, lo, row, m in a.blocks():
        for which in (0, 1):
            for h in range(K):
                x = (ready[1][row:row + m, h] if which == 0 else v[row:row + m, H + K + h])
                t = slack(x) if which == 0 else np.zeros((m, 1))
                was = np.log2(a.cache.scales[which][pg, blk, h]) if lo else O8.LOW
                fresh = {max(O8.power_of(x * f), was) for f in ((1 - 2.0 ** -14, 1.0, 1 + 2.0 ** -14) if which == 0 else (1.0,))}
                e = np.log2(float(scales[which][pg, blk, h]))
                assert e in fresh, (b, pg, blk, h, e, fresh)
                want_scales[which][pg, blk, h] = 2.0 ** e
                wc = a.cache.block(which, pg, blk, h).copy()
                if lo and e > was:
                    wc[:lo] = O8.codes_of(O8.CODES[wc[:lo]] * 2.0 ** (was - e))
                a.cache.codes, save = codes, a.cache.codes
                got = a.cache.block(which, pg, blk, h)
                a.cache.codes = save
                value = O8.CODES[got[lo:lo + m]] * 2.0 ** e
                # half a step: 2^-4 of the value, and half the smallest code
                within(value, x, np.maximum(2.0 ** -4 * np.abs(x), 2.0 ** (e - 10)) + t, "kv"[which])
                if which == 1:
                    np.testing.assert_array_equal(got[lo:lo + m], O8.codes_of(x * 2.0 ** -e))
                assert (got[:lo] == wc[:lo]).all() and (got[lo + m:] == wc[lo + m:]).all()
                a.cache.codes = want_codes
                a.cache.block(which, pg, blk, h)[:] = got
                a.cache.codes = save
    for which in (0, 1):  # nothing else was written
        np.testing.assert_array_equal(codes[which], want_codes[which])
        np.testing.assert_array_equal(scales[which], want_scales[which])


def plain_rows(ctx, rng, x, past, new, H=1, K=1, D=64, page=16, src=nh.F32):  # noqa: F811
    """An append without norm and rotation of given k and v rows [T, 2 K, D] (v behind k)."""
    T = x.shape[0]
    wide = np.zeros((T + 3, (H + 2 * K) * D + 16), np.float32)
    wide[1:T + 1, H * D:(H + 2 * K) * D] = x.reshape(T, -1)
    return Append8(ctx, rng, src, nh.BF16, H, K, D, page, "token", past, new, gap=0, x=wide)


def test_append_values(ctx):  # noqa: F811
    """What no norm or rotation has touched: bit for bit the definition's, with
    infinities, NaN, zeros, the largest and the smallest numbers among it."""
    rng = np.random.default_rng(1)
    x = (randn(rng, 96, 2, 64) * 2.0 ** rng.integers(-12, 12, (96, 2, 64))).astype(np.float32)
    x[0:16] = 0.0
    x[3, :, 5], x[20, :, 7], x[21, :, 8], x[22, 0, 9] = -0.0, np.inf, -np.inf, np.nan
    x[32:48] *= np.float32(2.0 ** 100)
    x[33, :, 1] = 3.4e38
    x[48:64] = (x[48:64] * 2.0 ** -100 * 2.0 ** -30).astype(np.float32)
    x[64, :, :] = 448.0
    x[65:80] = np.clip(x[65:80], -447, 447)
    x[80, :, 3] = np.nextafter(np.float32(448.0), np.float32(500))
    x[81:] = np.clip(x[81:], -447, 447)
    a = plain_rows(ctx, rng, x, [0], [96])
    a.run()
    ctx.sync()
    codes, scales = a.cache.download()
    a.cache.codes = codes
    for _, pg, blk, lo, row, m in a.blocks():
        for which in (0, 1):
            want, e = O8.append_block(x[row - 1:row - 1 + m, which].astype(np.float64), 0, np.zeros((16, 64), np.uint8), 0)
            assert scales[which][pg, blk, 0] == 2.0 ** e, (pg, blk, which)
            assert O8.same_codes(a.cache.block(which, pg, blk, 0)[:m], want[:m]).all()


def test_append_token_by_token(ctx):  # noqa: F811
    """Blocks that grow, by one token and by several, from small rows to large
    ones and back: codes and scales as the definition has them, every step; an
    earlier use of the pages leaves no trace."""
    rng = np.random.default_rng(2)
    pieces = [1, 1, 1, 4, 1, 9, 1, 1, 14, 1, 1, 1, 3, 1]
    x = randn(rng, sum(pieces), 2, 64) * (4.0 ** rng.integers(-4, 5, sum(pieces)))[:, None, None]
    x[5, 1, 3] = np.nan
    first = plain_rows(ctx, rng, 1e6 * randn(rng, 48, 2, 64), [0], [48])
    first.run()
    ctx.sync()
    codes, scales = first.cache.download()
    held = {w: [codes[w].copy(), scales[w].copy()] for w in (0, 1)}
    at = 0
    for m in pieces:
        a = plain_rows(ctx, rng, x[at:at + m].astype(np.float32), [0], [m])
        a.cache, a.past[:], a.table = first.cache, at, first.table
        a.lens = np.array([at + m], np.int32)
        a.dlens, a.dtable = ctx.to_device(a.lens), ctx.to_device(a.table)
        a.run()
        ctx.sync()
        codes, scales = first.cache.download()
        for _, pg, blk, lo, row, k in a.blocks():
            for w in (0, 1):
                first.cache.codes = [held[0][0], held[1][0]]
                mine = first.cache.block(w, pg, blk, 0)
                was = int(np.log2(held[w][1][pg, blk, 0])) if lo else 0
                rows = x[at + row - 1:at + row - 1 + k, w].astype(np.float32).astype(np.float64)
                mine[:], e = O8.append_block(rows, lo, mine, was)
                held[w][1][pg, blk, 0] = 2.0 ** e
        for w in (0, 1):
            assert O8.same_codes(codes[w], held[w][0]).all(), (at, w)
            np.testing.assert_array_equal(scales[w], held[w][1])
        at += m


def test_append_bad_sequences(ctx):  # noqa: F811
    """A length below its rows, or past the table's row: NaN in q_out, nothing
    written; a page outside the cache: its tokens are not; the others are."""
    rng = np.random.default_rng(4)
    a = Append8(ctx, rng, nh.BF16, nh.BF16, 4, 2, 64, 16, "token", [20, 5, 33, 40, 0], [30, 6, 20, 30, 3])
    lens, table = a.lens.copy(), a.table.copy()
    lens[1] = 5
    lens[2] = table.shape[1] * 16 + 1
    table[3, 3], table[3, 4] = a.cache.pages, -1
    a.dlens.upload(lens)
    a.dtable.upload(table)
    a.run()
    ctx.sync()
    q, (codes, scales) = a.q(), a.cache.download()
    for b in range(a.n):
        rows = slice(a.cu[b], a.cu[b + 1])
        if b in (1, 2):
            assert np.isnan(q[rows]).all()
        else:
            np.testing.assert_array_equal(q[rows], a.values[rows, :4])
    written = {(pg, blk) for b, pg, blk, *_ in a.blocks() if b in (0, 4)} | {(int(a.table[3, 2]), 0)}
    changed = {(int(p), 0) for w in (0, 1) for p in np.argwhere((codes[w] != a.cache.codes[w]).any(axis=(1, 2)))[:, 0]}
    assert changed == written
    assert (q[:a.cu[0]] == 5.0).all() and (q[a.cu[-1]:] == 5.0).all()


def test_append_offsets_that_fall(ctx):  # noqa: F811
    """Offsets outside the rows, or falling: nothing outside the buffers is
    touched, and sequences beside them are as they should be."""
    rng = np.random.default_rng(5)
    a = Append8(ctx, rng, nh.BF16, nh.BF16, 2, 1, 64, 16, "token", [3, 20, 7], [20, 11, 9])
    a.dcu.upload(np.array([-100, 21, 10, 10 ** 9], np.int32))
    a.run()
    ctx.sync()
    a.dcu.upload(np.array([2 ** 31 - 1, -2 ** 31, 50, -1], np.int32))
    a.run()
    ctx.sync()


def test_append_far_apart(ctx):  # noqa: F811
    """Pages 3 * 2^30 bytes apart, the second past 2^32."""
    rng, stride = np.random.default_rng(6), 3 << 30
    x = randn(rng, 40, 2, 64)
    a = plain_rows(ctx, rng, x, [0], [40])
    big = ctx.alloc(2 * stride + (1 << 16))
    scales = [ctx.to_device(np.zeros((3, 1, 1), np.float32)) for _ in range(2)]
    a.cache.desc = ctx.kv8_cache(big, big + 4096, *scales, 1, 64, 16, 3, stride, 64, 64)
    table = np.array([[2, 0, 1]], np.int32)
    a.dtable = ctx.to_device(table)
    a.table = table
    a.run()
    q = O.pack(randn(rng, 1, 2, 64), nh.BF16)
    out, ws = ctx.alloc(256), ctx.alloc(1 << 20)
    ctx._check(ctx.attn8_decode(a.cache.desc, ctx.to_device(q), nh.BF16, 2, 1, a.dlens, a.dtable, 3, 40, 0.125, out, None, ws, 1 << 20))
    ctx.sync()
    k, v = [], []
    for j0, pg in ((0, 2), (16, 0), (32, 1)):
        for which, to in ((0, k), (1, v)):
            want, e = O8.append_block(x[j0:j0 + 16, which].astype(np.float64), 0, np.zeros((16, 64), np.uint8), 0)
            m = min(16, 40 - j0)
            got = big.download(np.uint8, (16, 64), pg * stride + 4096 * which)
            np.testing.assert_array_equal(got[:m], want[:m])
            assert scales[which].download(np.float32, 3)[pg] == 2.0 ** e
            to.append(O8.CODES[want[:m]] * 2.0 ** e)
    for h in range(2):
        o, _, tol = O.attention(O.value(q, nh.BF16)[0, h][None], np.concatenate(k), np.concatenate(v), [40], 0.125, nh.BF16)
        within(O.value(out.download(np.uint16, (2, 64)), nh.BF16)[h], o[0], tol[0], f"head {h}")


# --------------------------------------------------------------- attention

class Attend8:
    """Decode (lq None) or prompt attention over random codes and scales; NaN
    codes and scales wherever no sequence has a token."""

    def __init__(self, ctx, rng, dtype, H, K, D, page, lens, lq=None, causal=True, layout="token", gap=0, spread=1.0):  # noqa: F811
        self.ctx, self.dtype, self.H, self.K, self.D, self.page, self.causal = ctx, dtype, H, K, D, page, causal
        self.lens, self.lq = np.array(lens, np.int32), lq
        per = -(-np.maximum(self.lens, 0) // page)
        self.cache = c = Cache8(ctx, rng, K, D, page, int(per.sum()) + 2, layout, gap)
        self.max_pages = int(per.max(initial=0)) + 1
        self.table = np.full((len(lens), self.max_pages), 0x3FFFFFFF, np.int32)
        at = 0
        for b, p in enumerate(per):
            self.table[b, :p] = c.order[at:at + p]
            at += p
        self.k, self.v = [], []
        for b, n in enumerate(self.lens):
            rows = [np.zeros((max(n, 0), K, D)) for _ in range(2)]
            for j0 in range(0, n, 16):
                pg, blk, m = int(self.table[b, j0 // page]), j0 % page // 16, min(16, n - j0)
                for which in (0, 1):
                    # as a block of 16 has them: magnitudes up to 448, scales of all sorts
                    x = np.clip(120.0 * rng.standard_normal((m, K, D)), -448, 448) * np.exp(-1.5 * rng.random((m, 1, 1)))
                    codes, e = O8.codes_of(x), rng.integers(-9, -5, K)
                    for h in range(K):
                        c.block(which, pg, blk, h)[:m] = codes[:, h]
                    c.scales[which][pg, blk] = 2.0 ** e
                    rows[which][j0:j0 + m] = O8.CODES[codes] * (2.0 ** e)[None, :, None]
            self.k.append(rows[0])
            self.v.append(rows[1])
        c.upload()
        self.cu = (np.cumsum([0, *(lq if lq is not None else [1] * len(lens))]) + (2 if lq is not None else 0)).astype(np.int32)
        self.nq = int(self.cu[-1]) + (3 if lq is not None else 1)
        q = np.full((self.nq, H, D), np.nan, np.float32)
        q[self.cu[0]:self.cu[-1]] = spread * rng.standard_normal((self.cu[-1] - self.cu[0], H, D))
        self.q, self.scale = O.pack(q, dtype), D ** -0.5
        self.dq, self.dlens, self.dtable, self.dcu = (ctx.to_device(t) for t in (self.q, self.lens, self.table, self.cu))
        self.out = ctx.to_device(O.pack(np.full((self.nq, H, D), 9.0), dtype))
        self.lse = ctx.to_device(np.full(self.nq * H, 9.0, np.float32))
        self.ws = None

    def size(self, max_len=None, max_q=None):
        n, most = len(self.lens), int(max(self.lens.max(initial=0), 0)) if max_len is None else max_len
        if self.lq is None:
            return self.ctx.attn8_decode_workspace(self.cache.desc, self.H, n, most)
        return self.ctx.attn8_prompt_workspace(self.cache.desc, self.H, n, self.nq, max(self.lq) if max_q is None else max_q, most)

    def run(self, max_len=None, max_q=None, stream=None, ws=None, lse=True):
        c, n, most = self.ctx, len(self.lens), int(max(self.lens.max(initial=0), 0)) if max_len is None else max_len
        size = self.size(max_len, max_q)
        if ws is None:
            self.guard = np.full(size // 4 + 8, 0x7FC12345, np.uint32)
            ws = self.ws = c.to_device(self.guard)
        lse = self.lse if lse else None
        if self.lq is None:
            return c._check(c.attn8_decode(self.cache.desc, self.dq, self.dtype, self.H, n, self.dlens, self.dtable, self.max_pages,
                                           most, self.scale, self.out, lse, ws, size, stream))
        return c._check(c.attn8_prompt(self.cache.desc, self.dq, self.dtype, self.H, n, self.dcu, self.nq, self.dlens, self.dtable,
                                       self.max_pages, max(self.lq) if max_q is None else max_q, most, self.causal, self.scale,
                                       self.out, lse, ws, size, stream))

    def read(self):
        return (O.value(self.out.download(O.NP[self.dtype], (self.nq, self.H, self.D)), self.dtype),
                self.lse.download(np.float32, (self.nq, self.H)))

    def check(self, heads=None, skip=(), lse=True, rows=None):
        got, got_lse = self.read()
        q, G = O.value(self.q, self.dtype), self.H // self.K
        inside = np.zeros(self.nq, bool)
        if self.ws is not None:  # nothing behind the workspace's end
            np.testing.assert_array_equal(self.ws.download(np.uint32, len(self.guard))[-8:], self.guard[-8:])
        for b, n in enumerate(self.lens):
            q0, q1 = self.cu[b], self.cu[b + 1]
            inside[q0:q1] = True
            if b in skip:
                continue
            i = np.arange(q1 - q0)
            see = np.clip(i + 1 + n - (q1 - q0), 0, n) if self.causal and self.lq is not None else np.full(q1 - q0, max(n, 0))
            pick = i if rows is None or len(i) <= rows else np.unique(np.concatenate([i[:3], i[-3:], i[::len(i) // rows]]))
            for h in range(self.H) if heads is None else heads:
                k, v = self.k[b][:, h // G], self.v[b][:, h // G]
                o, ls, tol = O.attention(q[q0 + pick, h], k, v, see[pick], self.scale, self.dtype)
                within(got[q0 + pick, h], o, tol, f"seq {b} head {h}")
                if lse:
                    for r, w in zip(pick, ls):
                        g = got_lse[q0 + r, h]
                        assert g == w if np.isneginf(w) else abs(g - w) <= lse_tol(q[q0 + r, h], k[:see[r]], self.scale, w), (b, h, r, g, w)
        assert (got[~inside] == 9.0).all() and (not lse or (got_lse[~inside] == 9.0).all())


@pytest.mark.parametrize("dtype,H,K,D,page,layout,lens,gap", [
    (nh.BF16, 16, 2, 256, 16, "token", [777, 1, 0, 33, 16, 17], 0),
    (nh.F16, 8, 8, 64, 48, "token", [100, 0, 5, 47, 48, 49, 95], 16),
    (nh.BF16, 32, 8, 128, 64, "head", [300, 1, 64, 65], 0),
    (nh.F16, 7, 1, 64, 16, "head", [3000, 2], 0),
    (nh.BF16, 12, 4, 128, 32, "token", [15, 500], 32),
    (nh.F16, 33, 11, 256, 16, "token", [70, 31], 0),
    (nh.BF16, 40, 2, 128, 256, "token", [1000, 255, 257], 0),
    (nh.F16, 2, 2, 128, 16, "token", [5000], 0),
    (nh.BF16, 1, 1, 256, 16, "token", [9000, 128, 129], 0),
])
def test_decode(ctx, dtype, H, K, D, page, layout, lens, gap):  # noqa: F811
    d = Attend8(ctx, np.random.default_rng(H + D), dtype, H, K, D, page, lens, layout=layout, gap=gap)
    d.run()
    ctx.sync()
    d.check(heads=range(0, H, 1 if H <= 16 else 5))


@pytest.mark.parametrize("max_len", [0, 1, 100, 5000, 2 ** 31 - 1])
def test_decode_max_len_is_a_hint(ctx, max_len):  # noqa: F811
    d = Attend8(ctx, np.random.default_rng(5), nh.BF16, 4, 2, 128, 32, [700, 3, 0, 4099])
    d.run(max_len)
    ctx.sync()
    d.check()


def test_decode_many_sequences(ctx):  # noqa: F811
    rng = np.random.default_rng(8)
    d = Attend8(ctx, rng, nh.F16, 4, 1, 64, 16, rng.integers(0, 40, 700).tolist())
    d.run()
    ctx.sync()
    d.check(skip=set(range(700)) - set(range(0, 700, 37)))


@pytest.mark.parametrize("lq", [None, [1, 1, 1], [9, 40, 3]])
def test_far_scores(ctx, lq):  # noqa: F811
    """Scores far apart: one key takes all; then all equal; then a scale of 0 and one below it."""
    d = Attend8(ctx, np.random.default_rng(6), nh.BF16, 4, 2, 64, 16, [301, 64, 3], lq=lq, spread=60.0)
    d.run()
    ctx.sync()
    d.check()
    d.scale = -d.scale
    d.run()
    ctx.sync()
    d.check()
    d.scale = 0.0
    d.run()
    ctx.sync()
    d.check()


@pytest.mark.parametrize("lq", [None, [4, 20, 33, 1, 70]])
def test_bad_pages(ctx, lq):  # noqa: F811
    """A length past the table's row, a page number outside the cache among
    those that are seen: NaN there; the others are as they were."""
    d = Attend8(ctx, np.random.default_rng(7), nh.BF16, 16, 2, 128, 16, [100, 60, 33, 200, 5000], lq=lq)
    d.table[1, 2] = d.cache.pages
    d.table[3, 0] = -1
    d.table[4, 300] = 0x7FFFFFFF
    d.table[2, 3:] = 0x40000000
    d.dtable.upload(d.table)
    lens = d.lens.copy()
    lens[0] = d.max_pages * 16 + 1
    d.dlens.upload(lens)
    d.run()
    ctx.sync()
    got, lse = d.read()
    for b in (0, 1, 3, 4):
        i = np.arange(d.cu[b + 1] - d.cu[b])
        first = {0: -1, 1: 32, 3: 0, 4: 4800}[b]  # the first token on a bad page
        sees = np.ones(len(i), bool) if lq is None else i + lens[b] - len(i) >= first
        assert np.isnan(got[d.cu[b] + i[sees]]).all() and np.isnan(lse[d.cu[b] + i[sees]]).all(), b
    d.check(skip=(0, 1, 3, 4))


def test_values_of_no_number(ctx):  # noqa: F811
    """A NaN among a sequence's own codes reaches its rows and no other's."""
    d = Attend8(ctx, np.random.default_rng(17), nh.BF16, 4, 2, 128, 16, [100, 60, 90])
    d.cache.block(1, int(d.table[1, 1]), 0, 0)[3, 5] = 0x7F
    d.cache.block(0, int(d.table[2, 0]), 0, 1)[2, 9] = 0xFF
    d.cache.upload()
    d.run()
    ctx.sync()
    got, _ = d.read()
    assert np.isnan(got[1, :2, 5]).all() and np.isfinite(got[1, 2:]).all()
    assert np.isnan(got[2, 2:]).all() and np.isfinite(got[2, :2]).all()
    d.check(skip=(1, 2))


def test_scales_behind_a_query(ctx):  # noqa: F811
    """A block of great scale that only later queries see costs earlier ones no bit."""
    p = Attend8(ctx, np.random.default_rng(62), nh.F16, 4, 2, 64, 16, [128, 40], [128, 40])
    for b, j0 in ((0, 32), (0, 112), (1, 32)):
        pg = int(p.table[b, j0 // 16])
        p.cache.block(1, pg, 0, 0)[:] = 1  # the least code: 2^-9
        p.cache.scales[1][pg, 0, 0] = 2.0 ** 20
        p.v[b][j0:j0 + 16, 0] = 2.0 ** 11
    p.cache.upload()
    p.run()
    ctx.sync()
    p.check()


def test_decode_in_place(ctx):  # noqa: F811
    """out over q, no lse."""
    d = Attend8(ctx, np.random.default_rng(9), nh.BF16, 6, 3, 128, 16, [90, 17, 1], gap=48)
    d.out = ctx.to_device(np.concatenate([d.q[:3], O.pack(np.full((1, 6, 128), 9.0), nh.BF16)]))
    d.dq = d.out
    d.run(lse=False)
    ctx.sync()
    d.check(lse=False)


@pytest.mark.parametrize("dtype,D", [(nh.BF16, 128), (nh.F16, 64)])
@pytest.mark.parametrize("lq", [None, [2, 30]])
def test_scales_of_all_sizes(ctx, dtype, D, lq):  # noqa: F811
    """Blocks whose scales are 2^60 apart, and zeros with the least scale:
    each counts by its values."""
    rng = np.random.default_rng(21)
    d = Attend8(ctx, rng, dtype, 4, 2, D, 16, [77, 160], lq=lq)
    for b, n in enumerate(d.lens):
        for j0 in range(0, n, 16):
            pg, m = int(d.table[b, j0 // 16]), min(16, n - j0)
            e = rng.choice([-117, -60, -20, -8, -6], 2) if dtype == nh.BF16 else rng.choice([-117, -30, -8, -6], 2)
            d.cache.scales[1][pg, 0] = 2.0 ** e
            for h in range(2):
                if e[h] == -117:
                    d.cache.block(1, pg, 0, h)[:m] = 0
                d.v[b][j0:j0 + m, h] = O8.CODES[d.cache.block(1, pg, 0, h)[:m]] * 2.0 ** e[h]
    d.cache.upload()
    d.run()
    ctx.sync()
    d.check()


@pytest.mark.parametrize("dtype,H,K,D,page,layout,lens,lq,causal", [
    (nh.BF16, 4, 2, 128, 16, "token", [1], [1], True),
    (nh.BF16, 16, 2, 256, 64, "token", [5, 64, 1, 130], [5, 64, 1, 130], True),
    (nh.F16, 8, 8, 64, 48, "head", [63, 65, 129, 7, 200], [63, 65, 129, 7, 200], True),
    (nh.F16, 7, 1, 64, 16, "token", [33, 257], [33, 257], True),
    (nh.BF16, 12, 4, 128, 32, "token", [140, 1000], [100, 31], True),
    (nh.F16, 6, 2, 256, 16, "head", [100, 260], [70, 20], True),
    (nh.BF16, 4, 4, 128, 16, "token", [70, 0, 31], [130, 9, 0], True),  # queries that see nothing, and none
    (nh.BF16, 4, 2, 64, 16, "token", [77, 500, 128], [50, 3, 129], False),
    (nh.F16, 4, 2, 128, 256, "token", [64, 30, 0], [40, 0, 129], False),
    (nh.BF16, 2, 1, 256, 16, "head", [300], [300], False),
    (nh.BF16, 33, 11, 64, 16, "token", [50, 40], [20, 40], True),
    (nh.BF16, 16, 2, 256, 16, "token", [5000, 9], [3, 1], True),  # few rows, many keys
    (nh.F16, 32, 8, 128, 64, "token", [3000], [17], True),
    (nh.BF16, 40, 1, 64, 16, "token", [700, 2000, 1], [1, 1, 1], True),
    (nh.BF16, 8, 1, 128, 16, "token", [0, 0], [3, 5], False),
])
def test_prompt(ctx, dtype, H, K, D, page, layout, lens, lq, causal):  # noqa: F811
    p = Attend8(ctx, np.random.default_rng(H + D + sum(lq)), dtype, H, K, D, page, lens, lq, causal, layout)
    p.run()
    ctx.sync()
    p.check(heads=range(0, H, 1 if H <= 16 else 7))


@pytest.mark.parametrize("dtype,H,K,D,lens,lq", [
    (nh.BF16, 32, 4, 64, [2100, 900], [2100, 900]), (nh.BF16, 16, 2, 256, [1500, 700], [1500, 700]),
    (nh.F16, 32, 8, 128, [1000, 1400, 20], [1000, 600, 20]), (nh.F16, 16, 2, 256, [1100], [1100]),
    (nh.BF16, 32, 2, 128, [333, 900, 280], [333, 280, 280]), (nh.BF16, 8, 8, 64, [601, 9], [601, 9]),
])
@pytest.mark.parametrize("hint", [None, 1, 2 ** 31 - 1])
def test_prompt_long(ctx, dtype, H, K, D, lens, lq, hint):  # noqa: F811
    """Whatever max_q and max_len say, what is computed goes by the lengths."""
    p = Attend8(ctx, np.random.default_rng(D), dtype, H, K, D, 64, lens, lq)
    p.run(max_len=hint, max_q=hint)
    ctx.sync()
    p.check(heads=[0, H - 1], rows=40)


def test_prompt_offsets_that_fall(ctx):  # noqa: F811
    """Offsets outside the rows, or falling: nothing outside the buffers is touched."""
    p = Attend8(ctx, np.random.default_rng(31), nh.BF16, 4, 2, 128, 16, [50, 300, 20], [50, 30, 20])
    for cu in ([-100, 40, 10, 10 ** 9], [2 ** 31 - 1, -2 ** 31, 50, -1]):
        p.dcu.upload(np.array(cu, np.int32))
        p.run()
        ctx.sync()


def test_one_query_as_decode(ctx):  # noqa: F811
    """Decode, and prompts of one query: the same up to the roundings of both."""
    rng = np.random.default_rng(33)
    d = Attend8(ctx, rng, nh.BF16, 16, 2, 256, 16, [900, 1, 40])
    d.run()
    ctx.sync()
    want, _ = d.read()
    p = Attend8(ctx, np.random.default_rng(33), nh.BF16, 16, 2, 256, 16, [900, 1, 40], [1, 1, 1])
    p.q[2:5] = d.q[:3]
    p.dq.upload(p.q)
    p.run()
    ctx.sync()
    p.check()
    d.check()


# ------------------------------------------------------ graphs and streams

@pytest.mark.parametrize("lq", [None, [60, 33, 8]])
def test_attention_replays(ctx, lq):  # noqa: F811
    """A captured call follows new lengths, pages and queries; eager calls and
    synchronizations between; the same bits as an eager call."""
    rng = np.random.default_rng(14)
    d = Attend8(ctx, rng, nh.BF16, 16, 2, 256, 16, [2000, 700, 90], lq=lq)
    d.run()
    ctx.sync()
    ws = ctx.alloc(d.size(2000) + 16)
    g = Graph(hip(), ctx.stream, lambda: d.run(2000, ws=ws))
    for step in range(4):
        d.lens[:] = [2000 - 300 * step, 700 - 13 * step, 90 - 30 * step]
        for b in range(3):
            d.k[b], d.v[b] = d.k[b][:d.lens[b]], d.v[b][:d.lens[b]]
        q = rng.standard_normal(d.q.shape).astype(np.float32)
        d.q = O.pack(q, nh.BF16)
        d.dq.upload(d.q)
        d.dlens.upload(d.lens)
        d.run(2000)
        ctx.sync()
        eager = [t.tobytes() for t in d.read()]
        d.out.upload(O.pack(np.full((d.nq, 16, 256), 9.0), nh.BF16))
        g.launch()
        ctx.sync()
        assert [t.tobytes() for t in d.read()] == eager
        d.check(heads=[0, 15])
    g.close()


def test_two_streams(ctx):  # noqa: F811
    """Calls of one context on two streams at once, a workspace and outputs
    each: the bits of the same calls alone, every time."""
    hp, rng = hip(), np.random.default_rng(44)
    streams = [ctypes.c_void_p(), ctypes.c_void_p()]
    for s in streams:
        assert hp.hipStreamCreate(ctypes.byref(s)) == 0
    jobs = []
    for i in range(2):
        d = Attend8(ctx, rng, nh.BF16, 16, 2, 256, 16, [3000, 5, 800 + i])
        p = Attend8(ctx, rng, nh.F16, 4, 2, 128, 16, [2500, 100 + i], [40, 100 + i])
        a = Append8(ctx, rng, nh.BF16, nh.BF16, 4, 2, 128, 16, "token", [40, 3], [70, 1 + i])
        n = Plan(ctx, rng, 16, *mixed(rng, 200, 100, 30 + i))
        jobs.append((d, p, a, n, ctx.alloc(d.size() + 16), ctx.alloc(p.size() + 16)))

    def go(job, stream):
        d, p, a, n, wd, wp = job
        d.run(ws=wd, stream=stream)
        p.run(ws=wp, stream=stream)
        a.run(stream=stream)
        n.run(stream=stream)

    def bits(job):
        d, p, a, n = job[:4]
        codes, scales = a.cache.download()
        return [x.tobytes() for x in (*d.read(), *p.read(), *codes, *scales, n.d["slots"].download(np.int64, n.max_rows))]

    try:
        alone = []
        for job in jobs:
            go(job, None)
            ctx.sync()
            alone.append(bits(job))
        for _ in range(4):
            for job, s in zip(jobs, streams):
                go(job, s.value)
            for s in streams:
                assert hp.hipStreamSynchronize(s) == 0
            assert [bits(job) for job in jobs] == alone
        for d, p, _, n, _, _ in jobs:
            d.check()
            p.check()
            n.check()
    finally:
        for s in streams:
            assert hp.hipStreamDestroy(s) == 0


# --------------------------------------------------------------- all of it

@pytest.mark.parametrize("dtype,H,K,D,page", [(nh.BF16, 16, 2, 256, 16), (nh.F16, 6, 2, 64, 48)])
def test_serving_steps(ctx, dtype, H, K, D, page):  # noqa: F811
    """Requests that come in pieces, go on token by token and end: pages from
    the plan, rows appended, attention of the pieces and of the tokens, against
    attention over the values that the cache holds, step after step."""
    rng, n, width, pages, rows = np.random.default_rng(50), 5, 12, 30, 160
    up = lambda a: ctx.to_device(np.asarray(a))
    cache = Cache8(ctx, rng, K, D, page, pages)
    lens, free = up(np.zeros(n, np.int32)), up(np.array([pages], np.int32))
    stack, table, new = up(rng.permutation(pages).astype(np.int32)), up(np.full((n, width), -1, np.int32)), up(np.zeros(n, np.int32))
    cu, status = up(np.zeros(n + 1, np.int32)), up(np.zeros(n, np.int32))
    req = ctx.kv_requests(page, pages, width, rows, lens, new, free, stack, table, lens, free, cu, status)
    inv = (1e6 ** (-np.arange(0, 32, 2) / 32)).astype(np.float32)
    prep = ctx.qk_prep(32, up(inv), False, True, None, None, 0, 1e-6)
    qkv, q_ready, out = ctx.alloc(rows * (H + 2 * K) * D * 4), ctx.alloc(rows * H * D * 2), ctx.alloc(rows * H * D * 2)
    w = (H + 2 * K) * D
    desc = ctx.qkv_rows(qkv, qkv + H * D * 4, qkv + (H + K) * D * 4, nh.F32, H, K, D, w, D, w, D, w, D)
    size = max(ctx.attn8_prompt_workspace(cache.desc, H, n, rows, rows, width * page),
               ctx.attn8_decode_workspace(cache.desc, H, n, width * page))
    ws = ctx.alloc(size + 16)
    past = [[] for _ in range(n)]  # raw rows that a request has had
    for step, wish in enumerate([[40, 7, 0, 33, 1], [50, 1, 20, 1, 1], [1, 1, 1, 1, 1], [1, -1, 1, 30, 1], [1, 5, 1, 1, -1],
                                 [1, 1, 1, 1, 1], [0, 1, 0, 1, 3]]):
        new.upload(np.array(wish, np.int32))
        ctx._check(ctx.kv_plan(req, n))
        x = randn(rng, rows, H + 2 * K, D) * np.exp(0.5 * randn(rng, 1, H + 2 * K, 1))
        qkv.upload(x)
        ctx._check(ctx.kv8_append(cache.desc, desc, prep, n, cu, rows, lens, table, width, None, q_ready, dtype))
        one = all(v == 1 for v in wish)
        if one:  # a token each: row b is sequence b's
            ctx._check(ctx.attn8_decode(cache.desc, q_ready, dtype, H, n, lens, table, width, width * page, D ** -0.5, out, None, ws, size))
        else:
            ctx._check(ctx.attn8_prompt(cache.desc, q_ready, dtype, H, n, cu, rows, lens, table, width, max(wish), width * page,
                                        True, D ** -0.5, out, None, ws, size))
        ctx.sync()
        assert (status.download(np.int32, n) == 0).all()
        at, got_lens, tab = cu.download(np.int32, n + 1), lens.download(np.int32, n), table.download(np.int32, (n, width))
        codes, scales = cache.download()
        cache.codes, q, got = codes, O.value(q_ready.download(O.NP[dtype], (rows, H, D)), dtype), O.value(out.download(O.NP[dtype], (rows, H, D)), dtype)
        for b in range(n):
            if wish[b] < 0:
                past[b] = []
            past[b] += list(x[at[b]:at[b + 1]].astype(np.float64))
            m = len(past[b])
            assert m == got_lens[b] and at[b + 1] - at[b] == max(wish[b], 0)
            if m == 0:
                continue
            ready = O.prepared(np.array(past[b])[:, H:H + K], np.arange(m), inv, 32, False, True, None, False, 1e-6)
            values = [np.zeros((m, K, D)) for _ in range(2)]
            for j0 in range(0, m, 16):
                pg, blk, c = int(tab[b, j0 // page]), j0 % page // 16, min(16, m - j0)
                for which in (0, 1):
                    for h in range(K):
                        sc = float(scales[which][pg, blk, h])
                        values[which][j0:j0 + c, h] = O8.CODES[cache.block(which, pg, blk, h)[:c]] * sc
                        true = (ready if which == 0 else np.array(past[b])[:, H + K:])[j0:j0 + c, h]
                        # half a step; a code below 2^-6 was rounded more than once, by half the smallest step each,
                        # for scales that at least double: once and a half more in all
                        t = np.maximum(2.0 ** -4 * np.abs(true), 2.0 * 2.0 ** -10 * sc) + 2.0 ** -14 * np.abs(true).max()
                        within(values[which][j0:j0 + c, h], true, t, "kv"[which])
            for h in range(H):
                r = np.arange(at[b], at[b + 1])
                o, _, tol = O.attention(q[r, h], values[0][:, h // (H // K)], values[1][:, h // (H // K)], np.arange(len(r)) + 1 + m - len(r),
                                        D ** -0.5, dtype)
                within(got[r, h], o, tol, f"step {step} request {b} head {h}")
