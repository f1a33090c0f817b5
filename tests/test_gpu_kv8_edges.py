"""GPU: the context in 8 bits at its edges: values and scores near fp32's
limits, lengths near 32 bits', hints and row counts far from what there
is."""
import numpy as np
import pytest

import context_oracle as O
import kv8_oracle as O8
import nmoe_hip as nh
from test_gpu_context import ctx  # noqa: F401 (a fixture)
from test_gpu_kv8 import Attend8

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
