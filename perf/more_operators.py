"""Performance cases of the 8-bit context: requests laid out in pages, keys and values held in 8 bits, attention over them.

The operators:
  plan     from each request's length and new tokens: its pages, offsets, positions and slots
  append8  norm and rotate q and k, write k and v in 8 bits, a scale for 16 tokens of a head
  decode8  attention of one new token a sequence over the 8-bit cache
  prompt8  causal attention of whole prompts, or pieces of them, over the 8-bit cache

A case is a dict of plain values:
  op       one of the above
  seqs     requests or sequences
  tokens   plan, append8, prompt8: new tokens of all together; decode8: mean length of the cache's sequences
  page     tokens a page
  mixed    plan: whether prompts are among the requests (else a token each, some idle, some ended)
  scarce   plan: whether the free pages are too few for all
  past     append8, prompt8: tokens that a sequence has before these, about
  dtype    append8: the projections' type; decode8, prompt8: q's and the result's; "bf16", "f16" or "f32"
  out      append8: the prepared q's type
  heads, kvheads, dim, layout      query heads, key and value heads, head size, "token" [page][token][head][dim] or
                                   "head" [page][head][token][dim]
  rotary, interleaved, norm        append8: rotated dimensions, their order, whether q and k are normalised
"""
import math
import os
import sys

import numpy as np
import torch

own = False

_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_F8 = torch.float8_e4m3fn
_BLOCK = 16  # tokens that share a scale
_LOW, _HIGH = -117, 118  # a scale's least and greatest power of two
_EPS = 1e-6
_THETA = 1e7


# ----------------------------------------------------------------- cases

def _plan(name, seqs, tokens, page, mixed, scarce):
    return {"name": name, "op": "plan", "seqs": seqs, "tokens": tokens, "page": page, "mixed": mixed, "scarce": scarce}


def _append(name, dtype, out, heads, kvheads, dim, page, layout, seqs, tokens, past, rotary, interleaved, norm):
    return {"name": name, "op": "append8", "dtype": dtype, "out": out, "heads": heads, "kvheads": kvheads, "dim": dim,
            "page": page, "layout": layout, "seqs": seqs, "tokens": tokens, "past": past, "rotary": rotary,
            "interleaved": interleaved, "norm": norm}


def _attend(name, op, dtype, heads, kvheads, dim, page, layout, seqs, tokens, past):
    return {"name": name, "op": op, "dtype": dtype, "heads": heads, "kvheads": kvheads, "dim": dim, "page": page,
            "layout": layout, "seqs": seqs, "tokens": tokens, "past": past}


def listed():
    return [
        # the next token of one chat
        _plan("plan_1", 1, 1, 16, False, False),
        # a large batch's next step: long prompts that begin among chats that go on, idle and end
        _plan("plan_512x65536", 512, 65536, 64, True, False),
        # the new token of one chat: latency alone
        _append("append8_1", "bf16", "bf16", 16, 2, 256, 16, "token", 1, 1, 777, 64, False, True),
        # a serving batch's new tokens, rows as a projection in 32 bits leaves them
        _append("append8_200", "f32", "bf16", 16, 2, 256, 64, "token", 200, 200, 900, 64, False, True),
        # a long prompt's next piece, which begins and ends inside a page
        _append("append8_4097", "bf16", "bf16", 16, 2, 256, 64, "token", 1, 4097, 2005, 64, False, True),
        # one chat, a short context that ends inside a page
        _attend("decode8_1x777", "decode8", "bf16", 16, 2, 256, 16, "token", 1, 777, 0),
        # a serving batch of ragged contexts, one of a single token and a padded row among them
        _attend("decode8_64x4096", "decode8", "bf16", 16, 2, 256, 64, "token", 64, 4096, 0),
        # one chat over a book, more key heads, the other layout and type
        _attend("decode8_1x131071", "decode8", "f16", 32, 8, 128, 256, "head", 1, 131071, 0),
        # short questions packed together, a head of keys for each of queries
        _attend("prompt8_5x611", "prompt8", "f16", 8, 8, 64, 16, "token", 5, 611, 0),
        # one middle-sized prompt, the model's own heads
        _attend("prompt8_1x2048", "prompt8", "bf16", 16, 2, 256, 64, "token", 1, 2048, 0),
        # a question about a book: few rows, very many keys
        _attend("prompt8_1x96+60001", "prompt8", "bf16", 16, 2, 256, 64, "token", 1, 96, 60001),
        # the largest: long documents packed together
        _attend("prompt8_3x8191", "prompt8", "bf16", 32, 8, 128, 64, "token", 3, 8191, 0),
    ]


def _log(rng, lo, hi):
    return int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1.0))))


def draw(rng):
    op = rng.choice(["plan", "append8", "append8", "decode8", "decode8", "decode8", "prompt8", "prompt8", "prompt8"])
    heads, kvheads, dim = rng.choice([(16, 2, 256), (16, 2, 256), (32, 8, 128), (8, 8, 64), (12, 4, 128), (7, 1, 64)])
    page, layout = rng.choice([16, 32, 48, 64, 256]), rng.choice(["token", "token", "head"])
    t2 = rng.choice(["bf16", "bf16", "f16"])
    if op == "plan":
        seqs = _log(rng, 1, 512)
        mixed = rng.random() < 0.6
        c = _plan("", seqs, _log(rng, seqs, max(seqs, 65536)) if mixed else seqs, page, mixed, rng.random() < 0.3)
    elif op == "append8":
        seqs = rng.choice([1, 1, 2, 5, _log(rng, 1, 200)])
        c = _append("", rng.choice(["bf16", "f16", "f32"]), t2, heads, kvheads, dim, page, layout, seqs,
                    max(seqs, _log(rng, 1, 4097)), rng.choice([0, rng.randint(1, 2500)]),
                    rng.choice([dim, dim // 2, dim // 4]), rng.random() < 0.3, rng.random() < 0.7)
    elif op == "decode8":
        seqs = _log(rng, 1, 200)
        c = _attend("", op, t2, heads, kvheads, dim, page, layout, seqs, _log(rng, 1, 131071 // seqs), 0)
    else:
        seqs = rng.choice([1, 1, 2, 3, 5, 8])
        tokens = _log(rng, 8, 8191 if seqs > 2 else 4500)
        past = rng.choice([0, 0, rng.randint(1, 500), _log(rng, 500, 60001)])
        c = _attend("", op, t2, heads, kvheads, dim, page, layout, seqs, tokens, min(past, 6000000 // tokens))
        while work(c)["flops"] > 2e11:
            c["tokens"] = c["tokens"] * 9 // 10
    del c["name"]
    return c


def _spread(n, total, r):
    """`total` in n parts of one at least, ragged."""
    w = 0.3 + r.rand(n)
    cut = np.floor(np.cumsum(w) / w.sum() * (total - n) + 1e-6).astype(np.int64)
    cut[-1] = total - n
    return np.diff(np.concatenate([[0], cut])) + 1


def _lens(case):
    """New tokens and length after them of each sequence, ragged, the same for every seed."""
    n, t = case["seqs"], case["tokens"]
    r = np.random.RandomState((n * 7919 + t * 31 + case["dim"]) & 0x7FFFFFFF)
    if case["op"] == "decode8":
        lens = np.maximum(1, (t * (0.5 + r.rand(n))).astype(np.int64)) if n > 1 else np.array([t], np.int64)
        if n > 1:
            lens[n // 2] = 1  # a chat that just begins
        if n >= 8:
            lens[-1] = 0  # a padded row
        return np.minimum(lens, 1), lens
    new = _spread(n, t, r)
    if n >= 8 and t == n:
        new[-1] = 0  # a padded row
    past = (case["past"] * (0.5 + r.rand(n))).astype(np.int64) if n > 1 else np.array([case["past"]], np.int64)
    return new, np.where(new > 0, past + new, 0)


# ---------------------------------------------------------------- inputs

class _State:
    pass


def _dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _offsets(lens):
    return np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)


def _prepare_plan(s, case, seed):
    n, page = case["seqs"], case["page"]
    r = np.random.RandomState((n * 7919 + case["tokens"] * 31 + page) & 0x7FFFFFFF)  # lengths: the same for every seed
    lens = np.exp(r.uniform(0, math.log(8192), n)).astype(np.int64)
    new = np.ones(n, np.int64)
    if case["mixed"]:
        first = np.arange(n) % 2 == 0  # prompts, many of them at their beginning
        lens[first] *= r.randint(0, 2, first.sum())
        if case["tokens"] > n:
            new[first] = _spread(int(first.sum()), int(case["tokens"] - (n - first.sum())), r)
    if n >= 8:
        new[r.randint(0, n, n // 8)] = 0  # idle
        new[r.randint(0, n, n // 8)] = -1  # ended
        lens[n - 1], new[n - 1] = 0, 0  # a padded row
    used = -(-lens // page)
    need = np.where(new > 0, -(-(lens + new) // page) - used, 0)
    s.max_pages = int(np.max(-(-(lens + np.maximum(new, 0)) // page))) + 1
    back = int(used[new < 0].sum())
    free = max(0, int(need.sum() * 0.6) - back) if case["scarce"] else int(need.sum()) + 5
    s.num_pages = int(used.sum()) + free + 3
    perm = np.random.RandomState(int(seed) & 0x7FFFFFFF).permutation(s.num_pages).astype(np.int32)
    table = np.zeros((n, s.max_pages), np.int32)
    held = np.arange(s.max_pages)[None] < used[:, None]
    table[held] = perm[:used.sum()]
    stack = np.zeros(s.num_pages, np.int32)
    stack[:free] = perm[used.sum():used.sum() + free]
    s.max_rows = max(1, int(np.maximum(new, 0).sum())) + (13 if n > 1 else 0)
    s.lens, s.new, s.table, s.stack = _dev(lens.astype(np.int32)), _dev(new.astype(np.int32)), _dev(table), _dev(stack)
    s.free = _dev(np.array([free], np.int32))
    z = lambda k, dt=torch.int32: torch.zeros(k, dtype=dt, device="cuda")
    s.lens_out, s.free_out, s.cu, s.status = z(n), z(1), z(n + 1), z(n)
    s.positions, s.slots = z(s.max_rows), z(s.max_rows, torch.int64)


def _scale_of(amax):
    """The least power of two s with amax <= 448 s, as its exponent, within the exponents there are."""
    m, e = torch.frexp(amax)  # amax = m 2^e, 1/2 <= m < 1
    e = torch.where(m <= 0.875, e - 9, e - 8)
    return torch.where(amax > 0, e, _LOW).clamp(_LOW, _HIGH)


def _in_8_bits(x, case):
    """Pages of values as codes, and their scales [page][block][head]."""
    x = x if case["layout"] == "token" else x.transpose(1, 2)
    pages, page, K, D = x.shape
    x = x.reshape(pages, page // _BLOCK, _BLOCK, K, D)
    scale = torch.ldexp(torch.ones((), device="cuda"), _scale_of(x.abs().amax(dim=(2, 4))))
    codes = (x / scale[:, :, None, :, None]).to(_F8).reshape(pages, page, K, D)
    return (codes if case["layout"] == "token" else codes.transpose(1, 2)).contiguous().view(torch.uint8), scale


def prepare(case, seed):
    s = _State()
    s.case, s.call = dict(case), None
    if case["op"] == "plan":
        _prepare_plan(s, case, seed)
        return s
    g = torch.Generator(device="cuda")
    g.manual_seed((int(seed) * 1000003 + case["tokens"] * 8191 + case["dim"]) & 0x7FFFFFFFFFFF)
    r = np.random.RandomState((int(seed) * 2654435761 + case["tokens"]) & 0x7FFFFFFF)
    randn = lambda *shape: torch.randn(*shape, generator=g, device="cuda")
    op, H, K, D, n, dt = case["op"], case["heads"], case["kvheads"], case["dim"], case["seqs"], _DT[case["dtype"]]
    page = case["page"]
    s.new, s.lens = _lens(case)
    T = int(s.new.sum()) if op != "decode8" else n
    s.T, s.max_new, s.max_len = T, int(s.new.max()), int(s.lens.max())
    per = -(-s.lens // page)
    s.pages = int(per.sum()) + 2
    perm = r.permutation(s.pages).astype(np.int32)
    table = np.zeros((n, max(1, int(per.max()))), np.int32)
    table[np.arange(table.shape[1])[None] < per[:, None]] = perm[:per.sum()]
    s.table, s.dlens, s.cu = _dev(table), _dev(s.lens.astype(np.int32)), _dev(_offsets(s.new))
    shape = (s.pages, page, K, D) if case["layout"] == "token" else (s.pages, K, page, D)
    heads = (1, 1, K, D) if case["layout"] == "token" else (1, K, 1, D)
    # what the cache holds: dimensions of unequal size, normalised keys that share a direction
    k = (randn(*shape) + 0.3 * randn(*heads)) * torch.exp(0.3 * randn(*heads))
    s.kc, s.ks = _in_8_bits(k, case)
    del k
    s.vc, s.vs = _in_8_bits(randn(*shape) * torch.exp(0.5 * randn(*heads)), case)
    if op != "append8":
        s.q = (1.2 * randn(T, H, D) + 0.3 * randn(1, H, D)).to(dt)
        s.out = torch.zeros(T, H, D, dtype=dt, device="cuda")
        return s
    # one projection's rows hold q, k and v side by side
    x = randn(T, H + 2 * K, D)
    x[:, :H + K] *= torch.exp(0.5 * randn(1, H + K, 1))
    s.x = x.to(dt)
    s.q, s.k, s.v = s.x[:, :H], s.x[:, H:H + K], s.x[:, H + K:]
    s.inv = (_THETA ** (-torch.arange(0, case["rotary"], 2, dtype=torch.float64) / case["rotary"])).float().cuda()
    s.qw, s.kw = ((0.1 * randn(D)).to(torch.bfloat16) for _ in range(2))
    s.q_out = torch.zeros(T, H, D, dtype=_DT[case["out"]], device="cuda")
    # behind a sequence's end nothing has been written yet
    at = torch.arange(page, device="cuda")
    last = torch.zeros(s.pages, dtype=torch.int64, device="cuda")
    past = _dev(s.lens - s.new)
    held = (past[:, None] - torch.arange(table.shape[1], device="cuda")[None] * page).clamp(0, page)
    mine = torch.arange(table.shape[1], device="cuda")[None] < _dev(per)[:, None]
    last[s.table[mine].long()] = held[mine]
    there = at[None] < last[:, None]
    for c in (s.kc, s.vc):
        _by_token(c, case).masked_fill_(~there[:, :, None, None], 0)
    return s


# ----------------------------------------------------------- plain forms

def _by_token(t, case):
    return t if case["layout"] == "token" else t.transpose(1, 2)


def _up(a, b):
    return (a + b - 1) // b


def _plain_plan(s):
    page, cap = s.case["page"], s.max_pages * s.case["page"]
    lens, new, j = s.lens.long(), s.new.long(), torch.arange(s.max_pages, device="cuda")
    bad = (lens < 0) | (lens > cap)
    held = _up(lens, page)
    # pages of ended requests go on the stack
    back = torch.where((new < 0) & ~bad, held, 0)
    free = s.free.long().clamp(0, s.num_pages)
    at = (free + back.cumsum(0) - back)[:, None] + j
    stack = torch.cat([s.stack, s.stack[:1]])
    stack[torch.where((j < back[:, None]) & (at < s.num_pages), at, s.num_pages)] = s.table
    free = (free + back.sum()).clamp(max=s.num_pages)
    # who gets what is asked for
    fits = ~bad & (new >= 0) & (lens + new <= cap)
    need, rows = torch.where(fits, _up(lens + new, page) - held, 0), torch.where(fits, new, 0)
    ok = fits & ((need == 0) | (need.cumsum(0) <= free)) & ((rows == 0) | (rows.cumsum(0) <= s.max_rows))
    need, rows = torch.where(ok, need, 0), torch.where(ok, rows, 0)
    # new pages from the stack's top
    first = need.cumsum(0) - need
    i = j - held[:, None]
    got = (i >= 0) & (i < need[:, None])
    table = torch.where(got, stack[(free - 1 - first[:, None] - i).clamp(0, s.num_pages)], s.table)
    cu = torch.cat([rows[:1] * 0, rows.cumsum(0)])
    # the rows
    t = torch.arange(s.max_rows, device="cuda")
    b = torch.searchsorted(cu[1:], t, right=True).clamp(max=s.case["seqs"] - 1)
    real = t < cu[-1]
    position = torch.where(real, lens[b] + t - cu[b], 0)
    slot = torch.where(real, table[b, position // page].long() * page + position % page, -1)
    i32 = lambda x: x.to(torch.int32)
    return {"lens": i32(torch.where((new < 0) & ~bad, 0, lens + rows)), "table": table, "stack": stack[:-1],
            "free": i32(free - need.sum()), "cu": i32(cu), "positions": i32(position), "slots": slot,
            "status": i32(torch.where(bad, 2, torch.where(ok | (new < 0), 0, 1)))}


def _pairs(x, rotary, interleaved):
    x = x[..., :rotary]
    return (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :rotary // 2], x[..., rotary // 2:])


def _rotated(s, x, w, position):
    c = s.case
    x = x.float()
    if c["norm"]:
        x = x * torch.rsqrt(x.square().mean(dim=-1, keepdim=True) + _EPS) * (1.0 + w.float())
    angle = position.double()[:, None] * s.inv.double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    a, b = _pairs(x, c["rotary"], c["interleaved"])
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([a, b], dim=-1).flatten(-2) if c["interleaved"] else torch.cat([a, b], dim=-1)
    return torch.cat([turned, x[..., c["rotary"]:]], dim=-1)


def _plain_append(s):
    c = s.case
    K, D, page, n = c["kvheads"], c["dim"], c["page"], c["seqs"]
    cu, lens = s.cu.long(), s.dlens.long()
    new = cu[1:] - cu[:-1]
    b = torch.repeat_interleave(torch.arange(n, device="cuda"), new, output_size=s.T)
    position = (lens - new)[b] + torch.arange(s.T, device="cuda") - cu[b]
    where = s.table[b, position // page].long()
    slot = where * page + position % page
    # blocks that a sequence goes on with: their tokens before these, and their scales
    begin = lens - new
    on = ((begin % _BLOCK > 0) & (new > 0)).nonzero()[:, 0]
    old = s.table[on, begin[on] // page].long() * page + begin[on] % page // _BLOCK * _BLOCK
    older = old[:, None] + torch.arange(_BLOCK, device="cuda")
    behind = torch.arange(_BLOCK, device="cuda") >= (begin[on] % _BLOCK)[:, None]
    for x, codes, scale in ((_rotated(s, s.k, s.kw, position), s.kc, s.ks), (s.v.float(), s.vc, s.vs)):
        by, flat = _by_token(codes, c), scale.view(-1, K)
        top = torch.zeros(flat.shape[0], K, device="cuda")
        top.scatter_reduce_(0, (slot // _BLOCK)[:, None].expand(-1, K), x.abs().amax(dim=-1), "amax")
        fresh = torch.ldexp(torch.ones((), device="cuda"), _scale_of(top))
        was = flat[old // _BLOCK].clone()
        flat[slot // _BLOCK] = fresh[slot // _BLOCK]
        flat[old // _BLOCK] = torch.maximum(fresh[old // _BLOCK], was)
        ratio = (was / flat[old // _BLOCK])[:, None, :, None]
        held = by[older // page, older % page]
        again = (held.view(_F8).float() * ratio).to(_F8).view(torch.uint8)
        by[older // page, older % page] = torch.where(behind[..., None, None], held, again)
        by[where, position % page] = (x / flat[slot // _BLOCK][..., None]).clamp(-448, 448).to(_F8).view(torch.uint8)
    return {"q": _rotated(s, s.q, s.qw, position).to(s.q_out.dtype), "k": s.kc.view(_F8), "k_scale": s.ks,
            "v": s.vc.view(_F8), "v_scale": s.vs}


def _held(s):
    """Keys and values of every sequence, [n, kvheads, longest, dim], and the keys' numbers."""
    c = s.case
    page = c["page"]
    at = torch.arange(s.max_len, device="cuda")
    rows = s.table[:, at // page].long(), (at % page)[None]
    block = s.table[:, at // page].long(), (at % page // _BLOCK)[None]
    k, v = ((_by_token(t, c)[rows].view(_F8).float() * scale[block][..., None]).transpose(1, 2)
            for t, scale in ((s.kc, s.ks), (s.vc, s.vs)))
    return k, v, at


def _plain_decode(s):
    c = s.case
    n, H, K, D = c["seqs"], c["heads"], c["kvheads"], c["dim"]
    k, v, at = _held(s)
    p = s.q.float().view(n, K, H // K, D) @ k.transpose(2, 3) * D ** -0.5
    p = p.masked_fill(~(at[None] < s.dlens[:, None])[:, None, None], -math.inf)
    p = torch.exp(p - p.amax(dim=-1, keepdim=True).clamp_min(-1e30))
    return ((p @ v) / p.sum(dim=-1, keepdim=True).clamp_min(1e-30)).view(n, H, D).to(s.out.dtype)


def _plain_prompt(s):
    c = s.case
    n, H, K, D = c["seqs"], c["heads"], c["kvheads"], c["dim"]
    k, v, at = _held(s)
    i = torch.arange(s.max_new, device="cuda")
    new = s.cu[1:] - s.cu[:-1]
    real = i[None] < new[:, None]
    q = s.q[torch.where(real, s.cu[:-1, None] + i, 0).long()].float().view(n, -1, K, H // K, D).permute(0, 2, 3, 1, 4)
    p = q @ k[:, :, None].transpose(3, 4)  # [n, kvheads, group, queries, keys]
    p *= D ** -0.5
    seen = at[None, None] <= (i[None] + (s.dlens - new)[:, None])[..., None]
    p.masked_fill_(~(seen & (at < s.dlens[:, None])[:, None])[:, None, None], -math.inf)
    p -= p.amax(dim=-1, keepdim=True).clamp_min(-1e30)
    p.exp_()
    o = (p @ v[:, :, None]) / p.sum(dim=-1, keepdim=True)
    return o.permute(0, 3, 1, 2, 4).reshape(n, -1, H, D)[real].to(s.out.dtype)


_PLAIN = {"plan": _plain_plan, "append8": _plain_append, "decode8": _plain_decode, "prompt8": _plain_prompt}


# ------------------------------------------------- the framework's calls

_program = []  # the binding and the program's one context


def _context():
    if not _program:
        pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "nano-metal-moe-qwen36_amd")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        import nmoe_hip

        _program.extend([nmoe_hip, nmoe_hip.Context(torch.cuda.current_device(), max_tokens=1)])
    return _program


def _bind(s):
    """The descriptors that a program keeps for its buffers, and the call on them."""
    nh, ctx = _context()
    c, p = s.case, (lambda t: t.data_ptr())
    # a state's calls run on the stream that is current at its first, which made its inputs; for torch's default stream,
    # whose handle is 0, on the context's own (None): HIP orders that one with it, before and after
    st = torch.cuda.current_stream().cuda_stream or None
    op, n = c["op"], c["seqs"]
    if op == "plan":
        req = nh.Context.kv_requests(c["page"], s.num_pages, s.max_pages, s.max_rows, p(s.lens), p(s.new), p(s.free),
                                     p(s.stack), p(s.table), p(s.lens_out), p(s.free_out), p(s.cu), p(s.status),
                                     p(s.positions), p(s.slots))
        got = {"lens": s.lens_out, "table": s.table, "stack": s.stack, "free": s.free_out, "cu": s.cu,
               "positions": s.positions, "slots": s.slots, "status": s.status}
        return lambda: ctx._check(ctx.kv_plan(req, n, st)) or got
    H, K, D = c["heads"], c["kvheads"], c["dim"]
    types = {torch.bfloat16: nh.BF16, torch.float16: nh.F16, torch.float32: nh.F32}
    strides = (s.kc.stride(0), _by_token(s.kc, c).stride(1), _by_token(s.kc, c).stride(2))
    cache = nh.Context.kv8_cache(p(s.kc), p(s.vc), p(s.ks), p(s.vs), K, D, c["page"], s.pages, *strides)
    pages = s.table.shape[1]
    if op == "append8":
        rows = nh.Context.qkv_rows(p(s.q), p(s.k), p(s.v), types[s.q.dtype], H, K, D, *s.q.stride()[:2],
                                   *s.k.stride()[:2], *s.v.stride()[:2])
        prep = nh.Context.qk_prep(c["rotary"], p(s.inv), c["interleaved"], c["norm"], p(s.qw), p(s.kw), 1, _EPS)
        got = {"q": s.q_out, "k": s.kc.view(_F8), "k_scale": s.ks, "v": s.vc.view(_F8), "v_scale": s.vs}
        return lambda: ctx._check(ctx.kv8_append(cache, rows, prep, n, p(s.cu), s.T, p(s.dlens), p(s.table), pages, None,
                                                 p(s.q_out), types[s.q_out.dtype], st)) or got
    if op == "decode8":
        size = ctx.attn8_decode_workspace(cache, H, n, s.max_len)
        s.ws = torch.empty(max(size, 16), dtype=torch.uint8, device="cuda")
        return lambda: ctx._check(ctx.attn8_decode(cache, p(s.q), types[s.q.dtype], H, n, p(s.dlens), p(s.table), pages,
                                                   s.max_len, D ** -0.5, p(s.out), None, p(s.ws), size, st)) or s.out
    size = ctx.attn8_prompt_workspace(cache, H, n, s.T, s.max_new, s.max_len)
    s.ws = torch.empty(max(size, 16), dtype=torch.uint8, device="cuda")
    return lambda: ctx._check(ctx.attn8_prompt(cache, p(s.q), types[s.q.dtype], H, n, p(s.cu), s.T, p(s.dlens), p(s.table),
                                               pages, s.max_new, s.max_len, True, D ** -0.5, p(s.out), None, p(s.ws),
                                               size, st)) or s.out


def run(s):
    if not own:
        return _PLAIN[s.case["op"]](s)
    if s.call is None:
        s.call = _bind(s)
    return s.call()


# ------------------------------------------------------------------ work

def work(case):
    n, T = case["seqs"], case["tokens"]
    if case["op"] == "plan":
        # a request's length, tokens, offset, new length and status; a row's position and slot; new pages
        return {"bytes": float(20 * n + 12 * T + 8 * (T // case["page"])), "flops": 0.0}
    H, K, D = case["heads"], case["kvheads"], case["dim"]
    e = 4 if case["dtype"] == "f32" else 2
    new, lens = (v.astype(np.float64) for v in _lens(case))
    scales = 2 * K * 4 / _BLOCK
    if case["op"] == "append8":
        return {"bytes": float(new.sum() * ((H + 2 * K) * D * e + H * D * 2 + 2 * K * D + scales)), "flops": 0.0}
    keys = float(lens.sum()) * (2 * K * D + scales)
    if case["op"] == "decode8":
        return {"bytes": keys + 2.0 * n * H * D * 2, "flops": 4.0 * float(lens.sum()) * H * D}
    pairs = float((new * (lens - new) + new * (new + 1) / 2).sum())
    return {"bytes": keys + 2.0 * T * H * D * 2, "flops": 4.0 * pairs * H * D}


# ----------------------------------------------------------------- exact

def _codes64():
    """What each of the 256 codes stands for: sign, 4 bits of exponent (bias 7), 3 of fraction; the last one no number."""
    value = [(1 if c < 128 else -1) * ((c & 7) * 2.0 ** -9 if c >> 3 & 15 == 0 else (8 + (c & 7)) * 2.0 ** ((c >> 3 & 15) - 10))
             for c in range(256)]
    value[127] = value[255] = math.nan
    return torch.tensor(value, dtype=torch.float64, device="cuda")


def _nearest64(x):
    """The code's value next to x, the even one of two."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.clamp(torch.round(x / step) * step, -448, 448)


def _turn64(s, x, w, position):
    c = s.case
    x = x.double()
    if c["norm"]:
        x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / c["dim"] + _EPS) * (w.double() + 1)
    out, half = x.clone(), c["rotary"] // 2
    i = torch.arange(half, device=x.device)
    a, b = (2 * i, 2 * i + 1) if c["interleaved"] else (i, i + half)
    z = torch.polar(torch.ones((), dtype=torch.float64, device=x.device), position.double()[:, None] * s.inv.double())
    z = torch.complex(x[..., a], x[..., b]) * z[:, None]
    out[..., a], out[..., b] = z.real, z.imag
    return out


def _exact_append(s):
    c = s.case
    K, D, page = c["kvheads"], c["dim"], c["page"]
    value = _codes64()
    position = torch.from_numpy(np.concatenate([np.arange(n - m, n) for m, n in zip(s.new, s.lens)])).cuda()
    codes = [value[(t if c["layout"] == "token" else t.permute(0, 2, 1, 3)).long()].reshape(-1, _BLOCK, K, D)
             for t in (s.kc, s.vc)]  # by blocks
    scales = [t.double().reshape(-1, K).clone() for t in (s.ks, s.vs)]
    table = s.table.cpu().numpy()
    for which, x in enumerate((_turn64(s, s.k, s.kw, position), s.v.double())):
        blocks, places, rows, older = [], [], [], []
        row = 0
        for b, (m, n) in enumerate(zip(s.new, s.lens)):
            j = np.arange(n - m, n)
            slot = table[b, j // page].astype(np.int64) * page + j % page
            blocks.append(slot // _BLOCK), places.append(slot % _BLOCK), rows.append(np.arange(row, row + m))
            row += m
            if m and (n - m) % _BLOCK:
                older.append((slot[0] // _BLOCK, (n - m) % _BLOCK))
        blocks, places, rows = (torch.from_numpy(np.concatenate(t)).cuda() for t in (blocks, places, rows))
        top = torch.zeros(scales[which].shape, dtype=torch.float64, device="cuda")
        for p in range(_BLOCK):
            at = places == p
            top[blocks[at]] = torch.maximum(top[blocks[at]], x[rows[at]].abs().amax(-1))
        want = torch.exp2(torch.ceil(torch.log2((top / 448).clamp_min(2.0 ** _LOW))))
        new = scales[which].clone()
        new[blocks] = want[blocks]
        for at, held in older:
            new[at] = torch.maximum(want[at], scales[which][at])
            again = _nearest64(codes[which][at, :held] * (scales[which][at] / new[at])[None, :, None])
            codes[which][at, :held] = again
        codes[which][blocks, places] = _nearest64(x[rows] / new[blocks][..., None])
        scales[which] = new
    shape = (s.pages, page, K, D)
    k, v = (t.reshape(shape) if c["layout"] == "token" else t.reshape(shape).transpose(1, 2).contiguous() for t in codes)
    return {"q": _turn64(s, s.q, s.qw, position), "k": k, "k_scale": scales[0].reshape(s.ks.shape), "v": v,
            "v_scale": scales[1].reshape(s.vs.shape)}


def exact(case, seed):
    if case["op"] == "plan":
        return None  # whole numbers
    s = prepare(case, seed)
    if case["op"] == "append8":
        return _exact_append(s)
    H, K, D, page = case["heads"], case["kvheads"], case["dim"], case["page"]
    value = _codes64()
    out = torch.zeros(s.T, H, D, dtype=torch.float64, device="cuda")
    q0 = 0
    for b, n in enumerate(int(v) for v in s.lens):
        nq = int(s.new[b]) if case["op"] == "prompt8" else 1
        pages = s.table[b, :-(-n // page)].long()
        ban = torch.ones(nq, n, dtype=torch.bool, device="cuda").triu(n - nq + 1)
        for h in range(K if n and nq else 0):
            kh, vh = ((value[(t[pages, :, h] if case["layout"] == "token" else t[pages, h]).long()].reshape(-1, _BLOCK, D) *
                       scale[pages, :, h].double().reshape(-1, 1, 1)).reshape(-1, D)[:n] for t, scale in ((s.kc, s.ks), (s.vc, s.vs)))
            for a in range(h * (H // K), (h + 1) * (H // K)):
                score = (s.q[q0:q0 + nq, a].double() @ kh.T / math.sqrt(D)).masked_fill_(ban, -math.inf)
                out[q0:q0 + nq, a] = torch.softmax(score, dim=-1) @ vh
        q0 += nq
    return out
