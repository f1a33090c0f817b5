"""GPU: the context operators against plain 64-bit forms (context_oracle.py):
types, head layouts, page sizes and layouts, lengths of zero and one, odd and
long ones, strided rows, rows and pages that must stay as they were, values
that must not be read, replays of captured graphs, calls on two streams."""


import numpy as np
import pytest

import context_oracle as O
import nmoe_hip as nh
from test_gpu_graph import Graph
from static_capture_client import hip

pytestmark = pytest.mark.gpu


@pytest.fixture()
def ctx():
    c = nh.Context(0, max_tokens=1)
    yield c
    c.close()


def within(got, want, tol, what):
    err = np.abs(got.astype(np.float64) - want)
    bad = ~(err <= tol)
    assert not bad.any(), (what, int(bad.sum()), float(np.nanmax(err / np.maximum(tol, 1e-300))), np.argwhere(bad)[:3])


def randn(rng, *shape):
    return rng.standard_normal(shape).astype(np.float32)


class Cache:
    """A paged cache, filled with `fill`, its pages dealt at random."""

    def __init__(self, ctx, rng, dtype, heads, dim, page, pages, layout="token", fill=np.nan, gap=0):
        self.ctx, self.dtype, self.heads, self.dim, self.page, self.pages, self.layout = ctx, dtype, heads, dim, page, pages, layout
        self.row = heads * dim + gap
        shape = (pages, page, self.row) if layout == "token" else (pages, heads, page, dim)
        self.host = [O.pack(np.full(shape, fill, np.float32), dtype) for _ in range(2)]
        self.dev = [ctx.to_device(h) for h in self.host]
        st = (page * self.row, self.row, dim) if layout == "token" else (heads * page * dim, dim, page * dim)
        self.desc = ctx.kv_cache(self.dev[0], self.dev[1], dtype, heads, dim, page, pages, *st)
        self.order = rng.permutation(pages).astype(np.int32)

    def rows(self, which, host=None):
        """[slots, heads, dim] view of k (0) or v (1)."""
        h = self.host[which] if host is None else host
        if self.layout == "token":
            return h[:, :, :self.heads * self.dim].reshape(-1, self.heads, self.dim)
        return np.ascontiguousarray(h.transpose(0, 2, 1, 3)).reshape(-1, self.heads, self.dim)

    def put(self, which, slots, rows):
        h = self.host[which]
        for s, r in zip(slots, rows):
            p, o = divmod(int(s), self.page)
            if self.layout == "token":
                h[p, o, :self.heads * self.dim] = r.ravel()
            else:
                h[p, :, o] = r

    def upload(self):
        for h, d in zip(self.host, self.dev):
            d.upload(h)

    def download(self, which):
        return self.dev[which].download(self.host[which].dtype, self.host[which].shape)


# ------------------------------------------------------------------ append

@pytest.mark.parametrize("src,dst,H,K,D,page,layout,rot,inter,norm,T", [
    (nh.BF16, nh.BF16, 16, 2, 256, 16, "token", 64, False, True, 1),
    (nh.BF16, nh.BF16, 16, 2, 256, 64, "head", 64, False, True, 37),
    (nh.F32, nh.F16, 6, 2, 64, 48, "token", 64, True, True, 19),
    (nh.F32, nh.BF16, 5, 1, 128, 32, "head", 128, False, False, 5),
    (nh.F16, nh.F16, 8, 8, 64, 16, "token", 16, False, True, 70),
    (nh.F16, nh.BF16, 4, 4, 128, 16, "token", 32, True, False, 3),
    (nh.BF16, nh.F16, 0, 3, 256, 16, "head", 256, True, True, 9),
    (nh.F32, nh.BF16, 33, 11, 64, 16, "token", 0, False, False, 2),
    (nh.BF16, nh.BF16, 2, 1, 256, 16, "token", 240, False, True, 600),
    # more tokens than blocks: several in turn, of one set of rows and of two
    (nh.BF16, nh.BF16, 1, 1, 64, 16, "token", 64, False, True, 2600),
    (nh.F32, nh.F16, 20, 4, 256, 16, "head", 64, True, True, 1100),
    (nh.F16, nh.BF16, 2, 1, 128, 16, "token", 0, False, True, 1030),
])
def test_append(ctx, src, dst, H, K, D, page, layout, rot, inter, norm, T):
    rng = np.random.default_rng(T + D)
    pages = -(-T // page) + 2
    c = Cache(ctx, rng, dst, K, D, page, pages, layout, fill=7.0)
    gap = 8  # rows of one projection side by side, a gap behind each head and each token
    width = (H + 2 * K) * (D + gap) + 16
    x = O.pack(3.0 * randn(rng, T, width), src)
    dx, es = ctx.to_device(x), 4 if src == nh.F32 else 2
    at = lambda head: dx.ptr + head * (D + gap) * es
    rows = ctx.qkv_rows(at(0) if H else None, at(H), at(H + K), src, H, K, D, width, D + gap, width, D + gap, width, D + gap)
    pos = rng.integers(0, 1 << 21, T).astype(np.int32)
    pos[0] = 2 ** 31 - 1 if T > 2 else 0
    slots = c.order[np.arange(T) // page].astype(np.int64) * page + np.arange(T) % page
    slots = np.where(np.arange(T) % 7 == 5, np.array([-1, pages * page, -2 ** 40, 2 ** 33])[np.arange(T) % 4], slots)
    inv = (1e6 ** (-np.arange(0, max(rot, 2), 2) / max(rot, 2))).astype(np.float32)
    qw, kw = (0.2 * randn(rng, D) for _ in range(2))
    qwd, kwd = (O.pack(w, nh.BF16) for w in (qw, kw))
    prep = ctx.qk_prep(rot, ctx.to_device(inv), inter, norm, ctx.to_device(qwd), ctx.to_device(kwd), 1, 1e-6)
    q_out = ctx.to_device(O.pack(np.full((T + 1, max(H, 1), D), 5.0), dst))
    ctx._check(ctx.kv_append(c.desc, rows, prep, T, ctx.to_device(pos), ctx.to_device(slots), q_out if H else None))
    ctx.sync()
    v = O.value(x, src)[:, :(H + 2 * K) * (D + gap)].reshape(T, H + 2 * K, D + gap)[..., :D]
    want_q = O.prepared(v[:, :H], pos, inv, rot, inter, norm, O.value(qwd, nh.BF16), True, 1e-6)
    want_k = O.prepared(v[:, H:H + K], pos, inv, rot, inter, norm, O.value(kwd, nh.BF16), True, 1e-6)

    def tol(w):
        # fp32 before the one rounding: the sum of D squares and its root (2^-17), the weight, the products of
        # the rotation, an angle good to 2^-20 turns: 2^-16 of the row's largest value, 2^-16 * 2 pi for the angle
        big = np.abs(w).max(axis=-1, keepdims=True)
        return O.HALF[dst] * np.abs(w) + 2.0 ** -15 * big + O.TINY[dst]

    got_q = O.value(q_out.download(O.NP[dst], (T + 1, max(H, 1), D)), dst)
    if H:
        within(got_q[:T], want_q, tol(want_q), "q")
    assert (got_q[T] == 5.0).all()
    keep = (slots >= 0) & (slots < pages * page)
    for which, want in ((0, want_k), (1, v[:, H + K:])):
        want_all = O.value(c.rows(which), dst)
        t = np.zeros_like(want_all)
        want_all[slots[keep]] = want[keep]
        t[slots[keep]] = (tol(want) if which == 0 else O.HALF[dst] * np.abs(want) + O.TINY[dst])[keep]
        within(O.value(c.rows(which, c.download(which)), dst), want_all, t, "kv"[which])


def test_append_without_prep(ctx):
    """No prep: q, k and v arrive as they are, bit for bit."""
    rng = np.random.default_rng(3)
    c = Cache(ctx, rng, nh.BF16, 2, 128, 16, 3, fill=0.0)
    x = O.pack(randn(rng, 5, 6, 128), nh.BF16)
    x[0, 0, 0], x[1, 2, 5], x[2, 4, 7] = 0x7F80, 0xFF80, 0x7F80  # infinities pass
    d = ctx.to_device(x)
    rows = ctx.qkv_rows(d, d + 2 * 256, d + 4 * 256, nh.BF16, 2, 2, 128, 768, 128, 768, 128, 768, 128)
    slots = np.array([47, 0, 16, 15, 33], np.int64)
    q_out = ctx.alloc(5 * 2 * 256)
    ctx._check(ctx.kv_append(c.desc, rows, None, 5, ctx.to_device(np.zeros(5, np.int32)), ctx.to_device(slots), q_out))
    ctx.sync()
    np.testing.assert_array_equal(q_out.download(np.uint16, (5, 2, 128)), x[:, :2])
    for which in (0, 1):
        np.testing.assert_array_equal(c.rows(which, c.download(which))[slots], x[:, 2 + 2 * which:4 + 2 * which])


# ------------------------------------------------------------------ decode

class Decode:
    def __init__(self, ctx, rng, dtype, H, K, D, page, lens, layout="token", spread=1.5, extra_pages=3, gap=0):
        self.ctx, self.dtype, self.H, self.D, self.lens = ctx, dtype, H, D, np.array(lens, np.int32)
        need = [-(-max(n, 0) // page) for n in lens]
        c = self.cache = Cache(ctx, rng, dtype, K, D, page, sum(need) + extra_pages, layout, fill=np.nan, gap=gap)
        self.max_pages = max(max(need), 1) + 1
        self.table = np.full((len(lens), self.max_pages), -5, np.int32)
        self.k, self.v, at = [], [], 0
        for b, n in enumerate(lens):
            self.table[b, :need[b]] = c.order[at:at + need[b]]
            at += need[b]
            kv = [O.pack(randn(rng, max(n, 0), K, D), dtype) for _ in range(2)]
            if n > 0:
                j = np.arange(n)
                slots = self.table[b, j // page].astype(np.int64) * page + j % page
                c.put(0, slots, kv[0])
                c.put(1, slots, kv[1])
            self.k.append(O.value(kv[0], dtype))
            self.v.append(O.value(kv[1], dtype))
        c.upload()
        n = len(lens)
        self.q = O.pack(spread * randn(rng, n, H, D), dtype)
        self.dq, self.dlens, self.dtable = ctx.to_device(self.q), ctx.to_device(self.lens), ctx.to_device(self.table)
        self.out = ctx.to_device(O.pack(np.full((n + 1, H, D), 9.0), dtype))
        self.lse = ctx.to_device(np.full((n + 1) * H, 9.0, np.float32))
        self.scale = D ** -0.5

    def run(self, max_len=None, stream=None, lse=True, ws=None):
        c, n = self.ctx, len(self.lens)
        max_len = max(1, int(self.lens.max())) if max_len is None else max_len
        size = c.attn_decode_workspace(self.cache.desc, self.H, n, max_len)
        ws = c.to_device(np.full(max(size, 16), 0xFF, np.uint8)) if ws is None else ws  # what it holds does not matter
        return c._check(c.attn_decode(self.cache.desc, self.dq, self.H, n, self.dlens, self.dtable, self.max_pages,
                                      max_len, self.scale, self.out, self.lse if lse else None, ws, size, stream))

    def read(self):
        n = len(self.lens)
        return (O.value(self.out.download(O.NP[self.dtype], (n + 1, self.H, self.D)), self.dtype),
                self.lse.download(np.float32, (n + 1, self.H)))

    def check(self, skip=(), lse=True):
        got, got_lse = self.read()
        assert (got[-1] == 9.0).all() and (got_lse[-1] == 9.0).all()
        q, G = O.value(self.q, self.dtype), self.H // self.cache.heads
        for b, n in enumerate(self.lens):
            if b in skip:
                continue
            for h in range(self.H):
                o, ls, tol = O.attention(q[b, h][None], self.k[b][:, h // G], self.v[b][:, h // G], [n], self.scale,
                                         self.dtype)
                within(got[b, h], o[0], tol[0], f"seq {b} (len {n}) head {h}")
                if lse:
                    assert got_lse[b, h] == ls[0] or abs(got_lse[b, h] - ls[0]) < 1e-4 * max(1.0, abs(ls[0])), (b, h)


@pytest.mark.parametrize("dtype,H,K,D,page,layout,lens", [
    (nh.BF16, 16, 2, 256, 16, "token", [1, 0, 15, 16, 17, 31, 33, 777]),
    (nh.F16, 16, 2, 256, 48, "head", [47, 48, 49, 1000, -3]),
    (nh.BF16, 8, 8, 64, 16, "token", [5, 64, 130]),
    (nh.F16, 7, 1, 64, 32, "token", [100, 1, 0, 333]),
    (nh.BF16, 12, 4, 128, 256, "head", [255, 257, 513]),
    (nh.F16, 32, 8, 128, 64, "token", [2049]),
    (nh.BF16, 40, 2, 128, 16, "token", [65, 300]),  # more heads a key than one tile holds
    (nh.F16, 17, 1, 256, 16, "head", [129]),
    (nh.BF16, 1, 1, 128, 16, "token", [40000]),
    (nh.BF16, 16, 16, 256, 16, "token", [70, 3]),
])
def test_decode(ctx, dtype, H, K, D, page, layout, lens):
    d = Decode(ctx, np.random.default_rng(H * 1000 + D + len(lens)), dtype, H, K, D, page, lens, layout)
    d.run()
    ctx.sync()
    d.check()


@pytest.mark.parametrize("max_len", [0, 1, 100, 5000, 2 ** 31 - 1])
def test_decode_max_len_is_a_hint(ctx, max_len):
    """Whatever max_len says, what is read goes by the lengths."""
    d = Decode(ctx, np.random.default_rng(5), nh.BF16, 4, 2, 128, 32, [700, 3, 0, 4099])
    d.run(max_len)
    ctx.sync()
    d.check()


def test_decode_many_sequences(ctx):
    rng = np.random.default_rng(8)
    d = Decode(ctx, rng, nh.F16, 4, 1, 64, 16, rng.integers(0, 40, 700).tolist())
    d.run()
    ctx.sync()
    d.check(skip=set(range(700)) - set(range(0, 700, 37)))


def test_decode_far_scores(ctx):
    """Scores far apart: one key takes all, the rest underflow; then scores all equal."""
    d = Decode(ctx, np.random.default_rng(6), nh.BF16, 4, 2, 64, 16, [301, 64], spread=60.0)
    d.run()
    ctx.sync()
    d.check()
    d.q[:] = 0
    d.dq.upload(d.q)
    d.run()
    ctx.sync()
    d.check()
    d.scale = 0.0
    d.run()
    ctx.sync()
    d.check()


def test_decode_bad_pages(ctx):
    """A page number outside the cache, or a length past the table's row:
    that sequence is NaN, the others are as they were.  Numbers behind a
    length are not looked at."""
    d = Decode(ctx, np.random.default_rng(7), nh.BF16, 16, 2, 128, 16, [100, 60, 33, 200, 5000])
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
        assert np.isnan(got[b]).all() and np.isnan(lse[b]).all(), b
    d.check(skip=(0, 1, 3, 4))


def test_decode_in_place_and_strided(ctx):
    """out over q, no lse, rows of the cache with a gap between tokens."""
    d = Decode(ctx, np.random.default_rng(9), nh.BF16, 6, 3, 128, 16, [90, 17, 1], gap=40)
    d.out = ctx.to_device(np.concatenate([d.q, O.pack(np.full((1, 6, 128), 9.0), nh.BF16)]))
    d.dq = d.out
    d.run(lse=False)
    ctx.sync()
    d.check(lse=False)


def test_decode_long_offsets(ctx):
    """Element offsets past 2^32: pages 3 * 2^30 elements apart."""
    H, K, D, page, stride = 4, 2, 64, 16, 3 << 30
    rng = np.random.default_rng(11)
    k, v = (O.pack(randn(rng, 2, page, K, D), nh.F16) for _ in range(2))
    big = ctx.alloc((stride + page * K * D) * 2 + (1 << 20))
    half = page * K * D * 2  # v lies behind k
    desc = ctx.kv_cache(big, big + half, nh.F16, K, D, page, 2, stride, K * D, D)
    for p in range(2):
        big.upload(k[p], p * stride * 2)
        big.upload(v[p], p * stride * 2 + half)
    q = O.pack(randn(rng, 1, H, D), nh.F16)
    out = ctx.alloc(H * D * 2)
    size = ctx.attn_decode_workspace(desc, H, 1, 30)
    ws = ctx.alloc(max(size, 16))
    ctx._check(ctx.attn_decode(desc, ctx.to_device(q), H, 1, ctx.to_device(np.array([30], np.int32)),
                               ctx.to_device(np.array([[1, 0]], np.int32)), 2, 30, 0.125, out, None, ws, size))
    ctx.sync()
    got = O.value(out.download(np.float16, (H, D)), nh.F16)
    kk, vv = (O.value(np.concatenate([t[1], t[0]]), nh.F16) for t in (k, v))
    for h in range(H):
        o, _, tol = O.attention(O.value(q, nh.F16)[0, h][None], kk[:, h // 2], vv[:, h // 2], [30], 0.125, nh.F16)
        within(got[h], o[0], tol[0], f"head {h}")


# ------------------------------------------------------------------ prompt

class Prompt:
    def __init__(self, ctx, rng, dtype, H, K, D, lq, lk=None, causal=True, before=0, behind=3, gap=0, fill=np.nan):
        self.ctx, self.dtype, self.H, self.K, self.D, self.causal = ctx, dtype, H, K, D, causal
        lk = lq if lk is None else lk
        self.cq = (np.cumsum([0] + list(lq)) + before).astype(np.int32)
        self.ck = (np.cumsum([0] + list(lk)) + before).astype(np.int32)
        self.nq, self.nk = int(self.cq[-1]) + behind, int(self.ck[-1]) + behind
        self.w = [h * (D + gap) + 2 * gap for h in (H, K, K)]

        def rows(n, heads, w, lo, hi):
            x = np.full((n, w), fill, np.float32)
            x[lo:hi, :heads * (D + gap)] = (1.3 * rng.standard_normal((hi - lo, heads * (D + gap)))).astype(np.float32)
            return O.pack(x, dtype)

        self.q = rows(self.nq, H, self.w[0], self.cq[0], self.cq[-1])
        self.k = rows(self.nk, K, self.w[1], self.ck[0], self.ck[-1])
        self.v = rows(self.nk, K, self.w[2], self.ck[0], self.ck[-1])
        self.gap, self.scale, self.lq, self.lk = gap, D ** -0.5, lq, lk
        self.dev = [ctx.to_device(t) for t in (self.q, self.k, self.v)]
        self.desc = ctx.qkv_rows(*self.dev, dtype, H, K, D, self.w[0], D + gap, self.w[1], D + gap, self.w[2], D + gap)
        self.out = ctx.to_device(O.pack(np.full((self.nq, H, D), 9.0), dtype))
        self.lse = ctx.to_device(np.full(self.nq * H, 9.0, np.float32))
        self.dcq, self.dck = ctx.to_device(self.cq), ctx.to_device(self.ck)

    def heads(self, t, heads):
        return O.value(t, self.dtype)[:, :heads * (self.D + self.gap)].reshape(-1, heads, self.D + self.gap)[..., :self.D]

    def run(self, max_q=None, max_k=None, stream=None, same=False):
        c = self.ctx
        return c._check(c.attn_prompt(self.desc, len(self.lq), self.dcq, None if same else self.dck, self.nq, self.nk,
                                      max(self.lq) if max_q is None else max_q, max(self.lk) if max_k is None else max_k,
                                      self.causal, self.scale, self.out, self.lse, stream))

    def read(self):
        return (O.value(self.out.download(O.NP[self.dtype], (self.nq, self.H, self.D)), self.dtype),
                self.lse.download(np.float32, (self.nq, self.H)))

    def check(self, heads=None, skip=()):
        got, got_lse = self.read()
        q, k, v, G = self.heads(self.q, self.H), self.heads(self.k, self.K), self.heads(self.v, self.K), self.H // self.K
        inside = np.zeros(self.nq, bool)
        for b in range(len(self.lq)):
            q0, q1, k0, k1 = self.cq[b], self.cq[b + 1], self.ck[b], self.ck[b + 1]
            inside[q0:q1] = True
            if b in skip:
                continue
            i = np.arange(q1 - q0)
            see = i + 1 + (k1 - k0) - (q1 - q0) if self.causal else np.full(q1 - q0, k1 - k0)
            for h in range(self.H) if heads is None else heads:
                o, ls, tol = O.attention(q[q0:q1, h], k[k0:k1, h // G], v[k0:k1, h // G], see, self.scale, self.dtype)
                within(got[q0:q1, h], o, tol, f"seq {b} head {h}")
                gl = got_lse[q0:q1, h]
                none = np.isneginf(ls)
                assert np.isneginf(gl[none]).all(), (b, h)
                assert (np.abs(gl[~none] - ls[~none]) < 1e-4 * np.maximum(1.0, np.abs(ls[~none]))).all(), (b, h)
        assert (got[~inside] == 9.0).all() and (got_lse[~inside] == 9.0).all()


@pytest.mark.parametrize("dtype,H,K,D,lq,lk,causal,gap", [
    (nh.BF16, 4, 2, 128, [1], None, True, 0),
    (nh.BF16, 16, 2, 256, [5, 64, 1, 130], None, True, 0),
    (nh.F16, 8, 8, 64, [63, 65, 129, 7, 200], None, True, 8),
    (nh.F16, 7, 1, 64, [33, 257], None, True, 0),
    (nh.BF16, 12, 4, 128, [100, 31], [140, 1000], True, 16),
    (nh.F16, 6, 2, 256, [70, 20], [100, 260], True, 0),
    (nh.BF16, 4, 4, 128, [130, 9], [70, 0], True, 0),  # queries that see nothing
    (nh.BF16, 4, 2, 64, [50, 3, 129], [77, 500, 128], False, 0),
    (nh.F16, 4, 2, 128, [40, 0, 129], [64, 30, 0], False, 0),
    (nh.BF16, 2, 1, 256, [300], [300], False, 0),
])
def test_prompt(ctx, dtype, H, K, D, lq, lk, causal, gap):
    """Rows before and behind the sequences hold NaN and stay as they were."""
    p = Prompt(ctx, np.random.default_rng(H + D + sum(lq)), dtype, H, K, D, lq, lk, causal, before=2, gap=gap)
    p.run()
    ctx.sync()
    p.check()


@pytest.mark.parametrize("D,H,K", [(64, 2, 1), (128, 2, 2), (256, 2, 1)])
def test_prompt_long(ctx, D, H, K):
    p = Prompt(ctx, np.random.default_rng(D), nh.BF16, H, K, D, [1500, 700])
    p.run(same=True)
    ctx.sync()
    p.check(heads=[0, H - 1])


@pytest.mark.parametrize("dtype,D,H,K,lq,lk", [
    (nh.BF16, 256, 32, 2, [600], [600]),  # keys shared by two groups of a block, blocks in more than one round
    (nh.F16, 64, 64, 8, [601], [601]),
    (nh.BF16, 128, 32, 2, [333, 280], [900, 280]),
    (nh.F16, 128, 2, 2, [40, 31], [2000, 65]),  # the same with all blocks at once
    (nh.BF16, 256, 4, 1, [3], [700]),
    (nh.BF16, 64, 32, 4, [2100, 900], [2100, 900]),  # blocks enough to go without
    (nh.F16, 256, 32, 2, [1100], [1100]),  # two groups of four pieces
    (nh.BF16, 256, 64, 8, [600, 500], [600, 500]),  # without, wider heads
    (nh.F16, 128, 64, 8, [500, 600], [500, 600]),
])
def test_prompt_forms(ctx, dtype, D, H, K, lq, lk):
    p = Prompt(ctx, np.random.default_rng(D + H), dtype, H, K, D, lq, lk)
    p.run()
    ctx.sync()
    p.check(heads=[0, H // 2, H - 1])


@pytest.mark.parametrize("max_q,max_k", [(0, 0), (1, 1), (64, 2 ** 31 - 1), (2 ** 31 - 1, 3)])
def test_prompt_sizes_are_hints(ctx, max_q, max_k):
    p = Prompt(ctx, np.random.default_rng(2), nh.F16, 4, 2, 128, [300, 2, 140], [300, 90, 400])
    p.run(max_q, max_k)
    ctx.sync()
    p.check()


def test_prompt_offsets_are_held(ctx):
    """Offsets past the rows there are, negative or falling: rows are never
    touched outside 0 .. ntok, and the sequences in order are right."""
    p = Prompt(ctx, np.random.default_rng(4), nh.BF16, 2, 1, 64, [40, 30, 50], behind=0)
    p.dcq.upload(np.array([-7, 40, 70, 1 << 30], np.int32))
    p.dck.upload(np.array([-(1 << 31), 40, 70, (1 << 31) - 1], np.int32))
    p.run()
    ctx.sync()
    p.check()
    p.dcq.upload(np.array([0, 40, 10, 5], np.int32))  # falling: no rows of their own
    p.run()
    ctx.sync()
    p.check(skip=(1, 2))


def test_prompt_other_sequence_not_finite(ctx):
    """NaN and infinities in one sequence stay there."""
    p = Prompt(ctx, np.random.default_rng(12), nh.BF16, 4, 2, 128, [50, 61, 40])
    p.k[50:111] = O.pack(np.full(1, np.inf), nh.BF16)[0]
    p.v[50:111] = O.pack(np.full(1, np.nan), nh.BF16)[0]
    for t, d in ((p.k, p.dev[1]), (p.v, p.dev[2])):
        d.upload(t)
    p.run()
    ctx.sync()
    p.check(skip=(1,))


def test_prompt_far_scores(ctx):
    p = Prompt(ctx, np.random.default_rng(13), nh.F16, 2, 2, 64, [200])
    p.scale = 5.0
    p.run()
    ctx.sync()
    p.check()
    p.scale = 0.0
    p.run()
    ctx.sync()
    p.check()
    p.scale = -0.3
    p.run()
    ctx.sync()
    p.check()


# -------------------------------------------------------------- delta rule

class Delta:
    def __init__(self, ctx, rng, dtype, Hk, Hv, Dk, Dv, lens, l2=True, index=None, states=None, zero=False, gap=0,
                 before=0, behind=2, strong=1.0):
        self.ctx, self.dtype, self.Hk, self.Hv, self.Dk, self.Dv, self.lens, self.l2 = ctx, dtype, Hk, Hv, Dk, Dv, lens, l2
        n, T = len(lens), sum(lens) + before + behind
        self.T, self.cu = T, (np.cumsum([0] + list(lens)) + before).astype(np.int32)
        w = [Hk * Dk + gap, Hk * Dk + gap, Hv * Dv + gap]
        q, k, v = (randn(rng, T, x) for x in w)
        k += 0.5 * randn(rng, 1, w[1])
        if not l2:
            q, k = q / np.sqrt(Dk), k / np.sqrt(1.3 * Dk)
        self.q, self.k, self.v = (O.pack(t, dtype) for t in (q, k, v))
        self.g = (-strong * np.exp(1.5 * randn(rng, T, Hv) - 2.0)).astype(np.float32)
        self.beta = (1 / (1 + np.exp(-randn(rng, T, Hv)))).astype(np.float32)
        self.num = n if states is None else states
        self.s0 = 0.2 * randn(rng, self.num, Hv, Dk, Dv)
        self.index = None if index is None else np.array(index, np.int32)
        self.zero, self.scale, self.eps = zero, Dk ** -0.5, 1e-6
        self.dev = [ctx.to_device(t) for t in (self.q, self.k, self.v, self.g, self.beta, self.s0)]
        self.ds_out = ctx.to_device(np.full(self.s0.shape, 4.0, np.float32))
        self.out = ctx.to_device(O.pack(np.full((T, Hv, Dv), 9.0), dtype))
        self.w = w
        self.dindex = None if index is None else ctx.to_device(self.index)
        self.dcu = ctx.to_device(self.cu)
        self.bind(self.dev[5], self.ds_out)

    def bind(self, s_in, s_out):
        self.desc = self.ctx.delta_rule(*self.dev[:3], self.dtype, self.Hk, self.Hv, self.Dk, self.Dv, *self.w,
                                        *self.dev[3:5], self.scale, self.l2, self.eps, None if self.zero else s_in, s_out,
                                        self.dindex, self.num, self.out)

    def step(self, stream=None):
        return self.ctx._check(self.ctx.delta_step(self.desc, len(self.lens), stream))

    def run(self, max_len=None, stream=None, ws=None):
        c, n = self.ctx, len(self.lens)
        size = c.delta_prompt_workspace(self.desc, n, self.T)
        ws = c.to_device(np.full(max(size, 16), 0xFF, np.uint8)) if ws is None else ws
        return c._check(c.delta_prompt(self.desc, n, self.dcu, self.T, max(self.lens) if max_len is None else max_len,
                                       ws, size, stream))

    def state(self, buf=None):
        return (buf or self.ds_out).download(np.float32, self.s0.shape)

    def check(self, state=None, first=None, untouched=4.0, skip=()):
        T, Hv = self.T, self.Hv
        got = O.value(self.out.download(O.NP[self.dtype], (T, Hv, self.Dv)), self.dtype)
        S = self.state() if state is None else state
        q, k = (O.value(t, self.dtype)[:, :self.Hk * self.Dk].reshape(T, self.Hk, self.Dk) for t in (self.q, self.k))
        v = O.value(self.v, self.dtype)[:, :Hv * self.Dv].reshape(T, Hv, self.Dv)
        inside, used = np.zeros(T, bool), np.zeros(self.num, bool)
        first = self.s0 if first is None else first
        for b, n in enumerate(self.lens):
            t0, t1 = self.cu[b], self.cu[b + 1]
            inside[t0:t1] = True
            i = b if self.index is None else self.index[b]
            if i < 0 or i >= self.num:
                assert (got[t0:t1] == 0).all() if i < 0 else np.isnan(got[t0:t1]).all()
                continue
            used[i] = True
            if b in skip:
                continue
            want, Sw = O.delta_rule(q[t0:t1], k[t0:t1], v[t0:t1], self.g[t0:t1], self.beta[t0:t1], self.scale, self.l2,
                                    self.eps, np.zeros_like(first[i]) if self.zero else first[i])
            # every token changes the state by fp32 sums of Dk products (their half steps add up as sqrt(Dk), taken
            # as 128 once) and by its decay and its update (a half step of the state each, twice over for the
            # chunked form's own sums)
            rel = 2.0 ** -24 * (128 + 4 * n)
            for h in range(Hv):
                e, size = np.linalg.norm(S[i, h] - Sw[h]), np.linalg.norm(Sw[h])
                assert e <= rel * size, (b, h, e, rel * size)
                if n:
                    size = np.linalg.norm(want[:, h], axis=-1, keepdims=True) + 0.05 * np.linalg.norm(want[:, h]) / n ** 0.5
                    within(got[t0:t1, h], want[:, h], O.HALF[self.dtype] * np.abs(want[:, h]) + 4 * rel * size +
                           O.TINY[self.dtype], f"seq {b} head {h}")
        assert (got[~inside] == 9.0).all()
        if untouched is not None:
            assert (S[~used] == untouched).all()


@pytest.mark.parametrize("dtype,Hk,Hv,Dk,Dv,n,l2", [
    (nh.BF16, 16, 32, 128, 128, 1, True), (nh.BF16, 2, 4, 128, 128, 7, True), (nh.F32, 2, 6, 64, 128, 3, True),
    (nh.F16, 3, 3, 128, 64, 5, False), (nh.F32, 1, 1, 64, 64, 70, False), (nh.F16, 1, 8, 64, 64, 2, True)])
def test_delta_step(ctx, dtype, Hk, Hv, Dk, Dv, n, l2):
    d = Delta(ctx, np.random.default_rng(Hv + n), dtype, Hk, Hv, Dk, Dv, [1] * n, l2, gap=16)
    d.step()
    ctx.sync()
    d.check()


def test_delta_step_indexed_in_place(ctx):
    """States of a pool, in place; a padded row; an index past the pool."""
    d = Delta(ctx, np.random.default_rng(1), nh.BF16, 2, 4, 128, 128, [1] * 5, index=[7, -1, 0, 9, 3], states=9)
    d.bind(d.dev[5], d.dev[5])
    d.step()
    ctx.sync()
    S = d.state(d.dev[5])
    d.check(state=S, untouched=None)
    rest = [i for i in range(9) if i not in (7, 0, 3)]
    np.testing.assert_array_equal(S[rest], d.s0[rest])


@pytest.mark.parametrize("dtype,Hk,Hv,Dk,Dv,lens,l2", [
    (nh.BF16, 2, 4, 128, 128, [1, 63, 64, 65, 200], True),
    (nh.F32, 1, 3, 128, 128, [129, 2], True),
    (nh.F16, 2, 2, 64, 128, [31, 0, 100], False),
    (nh.BF16, 1, 2, 128, 64, [300], True),
    (nh.F32, 2, 2, 64, 64, [17, 16, 15, 48], False),
    (nh.F16, 1, 4, 128, 128, [90, 128], True),
    (nh.BF16, 16, 32, 128, 128, [70], True),
])
def test_delta_prompt(ctx, dtype, Hk, Hv, Dk, Dv, lens, l2):
    d = Delta(ctx, np.random.default_rng(Hv + sum(lens)), dtype, Hk, Hv, Dk, Dv, lens, l2, gap=16, before=3)
    d.run()
    ctx.sync()
    d.check()


@pytest.mark.parametrize("dtype,Dk,lens", [(nh.BF16, 128, [3] * 39 + [65]), (nh.F32, 64, [2] * 19 + [70])])
def test_delta_prompt_many(ctx, dtype, Dk, lens):
    """More blocks than run at once: a block then has all heads on a head of k."""
    d = Delta(ctx, np.random.default_rng(27), dtype, 16, 32, Dk, 64, lens)
    d.run()
    ctx.sync()
    d.check()


@pytest.mark.parametrize("max_len", [0, 1, 64, 2 ** 31 - 1])
def test_delta_prompt_length_is_a_hint(ctx, max_len):
    d = Delta(ctx, np.random.default_rng(21), nh.BF16, 1, 2, 128, 128, [150, 3, 0, 70], zero=True)
    d.run(max_len)
    ctx.sync()
    d.check()


def test_delta_prompt_indexed(ctx):
    d = Delta(ctx, np.random.default_rng(22), nh.BF16, 1, 2, 128, 128, [80, 33, 0, 64, 10], index=[4, -1, 2, 6, 0], states=6)
    d.run()
    ctx.sync()
    d.check()


@pytest.mark.parametrize("dtype", [nh.BF16, nh.F32])
def test_delta_strong_decay(ctx, dtype):
    """Decays from none to all: g = 0, -1e-7, far below -100, -infinity and
    the lowest fp32 (each forgets what was before, whole)."""
    d = Delta(ctx, np.random.default_rng(23), dtype, 1, 2, 128, 128, [200, 130])
    d.g[::3] = 0.0
    d.g[1::7] = -1e-7
    for t, v in ((20, -200.0), (70, -np.inf), (71, -np.finfo(np.float32).max), (127, -1e30), (215, -np.inf)):
        d.g[t] = v
    d.dev[3].upload(d.g)
    d.run()
    ctx.sync()
    d.check()


def test_delta_equal_keys(ctx):
    """One key over and over, beta 1: every token replaces what it stood for."""
    d = Delta(ctx, np.random.default_rng(24), nh.F32, 1, 1, 64, 64, [130])
    d.k[:] = d.k[0]
    d.beta[:] = 1.0
    d.g[:] = 0.0
    for t, a in ((1, d.k), (3, d.g), (4, d.beta)):
        d.dev[t].upload(a)
    d.run()
    ctx.sync()
    d.check()


def test_delta_prompt_then_steps(ctx):
    """A prompt, then tokens one by one on its state, equal one longer prompt."""
    rng = np.random.default_rng(25)
    d = Delta(ctx, rng, nh.BF16, 2, 4, 128, 128, [100], behind=0)
    d.run()
    ctx.sync()
    d.check()
    S = d.state()
    for i in range(3):
        e = Delta(ctx, rng, nh.BF16, 2, 4, 128, 128, [1], behind=0)
        e.bind(d.ds_out, d.ds_out)
        e.step()
        ctx.sync()
        now = d.state()
        e.check(state=now, first=S)
        S = now


def test_delta_other_sequence_not_finite(ctx):
    """NaN and infinities in one sequence, its decay or its state stay there."""
    d = Delta(ctx, np.random.default_rng(28), nh.BF16, 1, 2, 128, 128, [70, 66, 90])
    d.k[70:136] = O.pack(np.full(1, np.inf), nh.BF16)[0]
    d.v[70:136] = O.pack(np.full(1, np.nan), nh.BF16)[0]
    d.g[100:136] = np.nan
    for t, a in ((1, d.k), (2, d.v), (3, d.g)):
        d.dev[t].upload(a)
    d.run()
    ctx.sync()
    d.check(skip=(1,))


def test_delta_offsets_are_held(ctx):
    d = Delta(ctx, np.random.default_rng(26), nh.BF16, 1, 2, 64, 64, [40, 70], behind=0)
    d.dcu.upload(np.array([-9, 40, 1 << 30], np.int32))
    d.run()
    ctx.sync()
    d.check()


# ------------------------------------------------- graphs, streams, a layer

def test_graph_replays(ctx):
    """All five captured into one graph and replayed on new inputs, with eager
    calls in between: lengths, pages and offsets are read on the device."""
    rng = np.random.default_rng(30)
    s = ctx.stream
    T, page, H, K, D = 96, 16, 4, 2, 128
    c = Cache(ctx, rng, nh.BF16, K, D, page, 20, fill=0.0)
    x, xd = None, ctx.alloc(T * (H + 2 * K) * D * 2)
    w = (H + 2 * K) * D
    rows = ctx.qkv_rows(xd, xd + H * D * 2, xd + (H + K) * D * 2, nh.BF16, H, K, D, w, D, w, D, w, D)
    inv = ctx.to_device((1e4 ** (-np.arange(32) / 32)).astype(np.float32))
    prep = ctx.qk_prep(64, inv, False, True, None, None, False, 1e-6)
    pos, slots, lens, table, cu = ctx.alloc(T * 4), ctx.alloc(T * 8), ctx.alloc(12), ctx.alloc(3 * 10 * 4), ctx.alloc(16)
    d = Delta(ctx, rng, nh.BF16, 1, 2, 128, 128, [1, 1, 1])
    pd = Delta(ctx, rng, nh.BF16, 1, 2, 128, 128, [40, 30, 26], behind=0)
    dsz = ctx.attn_decode_workspace(c.desc, H, 3, 160)
    psz = ctx.delta_prompt_workspace(pd.desc, 3, T)

    def bufs():
        return dict(q=ctx.alloc(T * H * D * 2), o=ctx.alloc(T * H * D * 2), od=ctx.alloc(3 * H * D * 2),
                    w1=ctx.alloc(max(dsz, 16)), w2=ctx.alloc(max(psz, 16)), s1=ctx.alloc(3 * 2 * 128 * 128 * 4),
                    s2=ctx.alloc(3 * 2 * 128 * 128 * 4), o1=ctx.alloc(5 * 2 * 128 * 2), o2=ctx.alloc(T * 2 * 128 * 2))

    def rule(e, s_out, out):
        return ctx.delta_rule(*e.dev[:3], nh.BF16, 1, 2, 128, 128, *e.w, *e.dev[3:5], e.scale, True, 1e-6, e.dev[5], s_out,
                              None, 3, out)

    def call(m):
        ctx._check(ctx.kv_append(c.desc, rows, prep, T, pos, slots, m["q"], s))
        r2 = ctx.qkv_rows(m["q"], xd + H * D * 2, xd + (H + K) * D * 2, nh.BF16, H, K, D, H * D, D, w, D, w, D)
        ctx._check(ctx.attn_prompt(r2, 3, cu, None, T, T, T, T, True, 0.1, m["o"], None, s))
        ctx._check(ctx.attn_decode(c.desc, m["q"], H, 3, lens, table, 10, 160, 0.1, m["od"], None, m["w1"], dsz, s))
        ctx._check(ctx.delta_step(rule(d, m["s1"], m["o1"]), 3, s))
        return ctx.delta_prompt(rule(pd, m["s2"], m["o2"]), 3, cu, T, 60, m["w2"], psz, s)

    def inputs(i):
        order = rng.permutation(20).astype(np.int32)
        n = [(40, 30, 26), (1, 94, 1), (96, 0, 0), (33, 31, 32)][i % 4]
        cu.upload(np.cumsum((0,) + n).astype(np.int32))
        tb, sl, p, at = np.zeros((3, 10), np.int32), [], [], 0
        for b, m in enumerate(n):
            k = -(-m // page)
            tb[b, :k] = order[at:at + k]
            at += k
            sl += [int(tb[b, j // page]) * page + j % page for j in range(m)]
            p += list(range(m))
        table.upload(tb)
        slots.upload(np.array(sl, np.int64))
        pos.upload(np.array(p, np.int32))
        lens.upload(np.array(n, np.int32))
        xd.upload(O.pack(randn(rng, T, H + 2 * K, D), nh.BF16))
        for e in (d, pd):
            e.dev[2].upload(O.pack(randn(rng, e.T, e.w[2]), nh.BF16))

    eager, graph = bufs(), bufs()
    inputs(0)
    ctx._check(call(eager))
    ctx.sync()
    g = Graph(hip(), s, lambda: call(graph))
    try:
        for i in range(6):
            inputs(i)
            g.launch()
            if i % 2:
                ctx._check(call(eager))
            ctx.sync()
            got = {k: graph[k].download(np.uint8, graph[k].nbytes) for k in ("q", "o", "od", "s1", "s2", "o1", "o2")}
            ctx._check(call(eager))
            ctx.sync()
            for k, v in got.items():
                np.testing.assert_array_equal(v, eager[k].download(np.uint8, eager[k].nbytes), err_msg=f"replay {i}: {k}")
    finally:
        g.close()


def test_two_streams(ctx):
    """The same calls from two contexts' streams at once, a workspace each,
    over and over: each as alone, and the same bits every time."""
    other = nh.Context(0, max_tokens=1)
    try:
        rng = np.random.default_rng(31)
        jobs = []
        for c in (ctx, other):
            jobs.append((Decode(c, rng, nh.BF16, 16, 2, 256, 16, [3000, 5, 800]),
                         Prompt(c, rng, nh.BF16, 4, 2, 128, [300, 100]),
                         Delta(c, rng, nh.BF16, 2, 4, 128, 128, [150, 20])))
        ws = [(c.alloc(max(16, c.attn_decode_workspace(j[0].cache.desc, 16, 3, 3000))),
               c.alloc(max(16, c.delta_prompt_workspace(j[2].desc, 2, j[2].T)))) for c, j in zip((ctx, other), jobs)]
        seen = None
        for _ in range(5):
            for j, w in zip(jobs, ws):
                j[0].run(ws=w[0])
                j[1].run()
                j[2].run(ws=w[1])
            ctx.sync()
            other.sync()
            now = [(j[0].read()[0].tobytes(), j[1].read()[0].tobytes(), j[2].state().tobytes()) for j in jobs]
            assert seen is None or seen == now
            seen = now
        for j in jobs:
            j[0].check()
            j[1].check(heads=[0, 3])
            j[2].check()
    finally:
        other.close()


def test_layer_prompt_then_token(ctx):
    """An attention layer as it runs: a prompt's rows are prepared and
    appended, attended over; then one more token is appended and attends over
    the cache.  The token's output equals the prompt attention's own answer
    for a prompt that is one longer."""
    rng = np.random.default_rng(32)
    T, H, K, D, page = 130, 8, 2, 256, 16
    w = (H + 2 * K) * D
    x = O.pack(randn(rng, T + 1, w), nh.BF16)
    xd = ctx.to_device(x)
    inv = ctx.to_device((1e7 ** (-np.arange(32) / 32)).astype(np.float32))
    prep = ctx.qk_prep(64, inv, False, True, None, None, False, 1e-6)
    c = Cache(ctx, rng, nh.BF16, K, D, page, 12)
    slots = c.order[np.arange(T + 1) // page].astype(np.int64) * page + np.arange(T + 1) % page
    ds, dp = ctx.to_device(slots), ctx.to_device(np.arange(T + 1, dtype=np.int32))
    q = ctx.alloc((T + 1) * H * D * 2)

    def rows(t0):
        b = xd + t0 * w * 2
        return ctx.qkv_rows(b, b + H * D * 2, b + (H + K) * D * 2, nh.BF16, H, K, D, w, D, w, D, w, D)

    ctx._check(ctx.kv_append(c.desc, rows(0), prep, T, dp, ds, q))
    ctx._check(ctx.kv_append(c.desc, rows(T), prep, 1, dp + 4 * T, ds + 8 * T, q + T * H * D * 2))
    ctx.sync()
    kc, vc = (O.value(c.rows(i, c.download(i))[slots], nh.BF16) for i in range(2))
    qv = O.value(q.download(np.uint16, (T + 1, H, D)), nh.BF16)
    table = ctx.to_device(c.order[None, :9].copy())
    out, size = ctx.alloc(H * D * 2), ctx.attn_decode_workspace(c.desc, H, 1, T + 1)
    ctx._check(ctx.attn_decode(c.desc, q + T * H * D * 2, H, 1, ctx.to_device(np.array([T + 1], np.int32)), table, 9,
                               T + 1, D ** -0.5, out, None, ctx.alloc(max(size, 16)), size))
    k = ctx.to_device(O.pack(kc, nh.BF16))
    v = ctx.to_device(O.pack(vc, nh.BF16))
    r = ctx.qkv_rows(q, k, v, nh.BF16, H, K, D, H * D, D, K * D, D, K * D, D)
    po = ctx.alloc((T + 1) * H * D * 2)
    ctx._check(ctx.attn_prompt(r, 1, ctx.to_device(np.array([0, T + 1], np.int32)), None, T + 1, T + 1, T + 1, T + 1, True,
                               D ** -0.5, po))
    ctx.sync()
    a = O.value(out.download(np.uint16, (H, D)), nh.BF16)
    p = O.value(po.download(np.uint16, (T + 1, H, D)), nh.BF16)
    for h in range(H):
        o, _, tol = O.attention(qv[:, h], kc[:, h // 4], vc[:, h // 4], np.arange(T + 1) + 1, D ** -0.5, nh.BF16)
        within(a[h], o[T], tol[T], f"token, head {h}")
        within(p[:, h], o, tol, f"prompt, head {h}")


def test_attention_then_moe(ctx):
    """What attention gives goes on into the layer's MoE half: h_mid = h +
    out, one block call."""
    from oracle import binding as B
    rng = np.random.default_rng(33)
    H, K, D, layer, k = 8, 2, 256, 0, 8
    d = Decode(ctx, rng, nh.BF16, H, K, D, 16, [50])
    d.run()
    ctx.sync()
    d.check()
    ctx.synth_layer(layer, 4, 3, 0.02)
    router = ctx.alloc(256 * 2048 * 2)
    ctx.synth_bf16(router, 256 * 2048, 3, layer, 16, 0.02)
    x = d.read()[0][0].reshape(2048).astype(np.float32)
    h = randn(rng, 2048)
    out, idx, w = ctx.alloc(8192), ctx.alloc(32), ctx.alloc(32)
    ctx._check(ctx.moe_layer(layer, ctx.router_bf16(router), d.out, nh.BF16, 1, k, ctx.to_device(h), out, idx, w))
    got = out.download(np.float32, (1, 2048))
    W = B.syn_bf16(256 * 2048, 3, layer, 16, 0.02).reshape(256, 2048)
    oi, ow, _ = B.route(B.router_logits_bf16(W, x), k)
    np.testing.assert_array_equal(idx.download(np.uint32, 8), oi)
    pack = np.zeros(256 * B.EXPERT_SIZE[4], np.uint8)
    for e in oi:
        pack[int(e) * B.EXPERT_SIZE[4]:(int(e) + 1) * B.EXPERT_SIZE[4]] = B.syn_expert(4, 3, layer, int(e), 0.02)
    want = B.moe_experts(pack, 4, x[None], k, oi[None], ow[None], h[None])
    assert np.abs(got - want).max() <= 2e-3
