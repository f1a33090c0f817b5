"""Performance cases of the context operators: what a layer runs in front of its MoE half.

The operators, for prompts and for single tokens:
  append  norm and rotate q and k, write k and v to the pages of a key-value cache
  decode  attention of one new token a sequence over the paged cache
  prompt  causal attention over packed prompts, grouped heads
  step    the gated delta rule, one token a sequence
  delta   the gated delta rule over packed prompts

A case is a dict of plain values:
  op       one of the above
  dtype    "bf16", "f16" or "f32": the inputs' type (append: the projections'; step, delta: q, k and v)
  cache    append: the cache's type, "bf16" or "f16"
  heads    query heads (step, delta: heads of v and of the state)
  kvheads  key and value heads (step, delta: heads of q and k)
  dim      head size (step, delta: of k and of v)
  page     tokens a page; layout "token" [page][token][head][dim] or "head" [page][head][token][dim]
  tokens   append: rows; prompt, delta: tokens of all sequences together; decode: mean length
  seqs     sequences
  past     prompt: tokens that a sequence's keys begin before its queries
  rotary, interleaved, norm    append: rotated dimensions, their order, whether q and k are normalised
  l2       step, delta: whether q and k are normalised
"""
import math
import os
import sys

import numpy as np
import torch

own = False

_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_EPS = 1e-6
_THETA = 1e7


# ----------------------------------------------------------------- cases

def _append(name, dtype, cache, heads, kvheads, dim, page, layout, tokens, rotary, interleaved, norm):
    return {"name": name, "op": "append", "dtype": dtype, "cache": cache, "heads": heads, "kvheads": kvheads,
            "dim": dim, "page": page, "layout": layout, "tokens": tokens, "rotary": rotary,
            "interleaved": interleaved, "norm": norm}


def _decode(name, dtype, heads, kvheads, dim, page, layout, tokens, seqs):
    return {"name": name, "op": "decode", "dtype": dtype, "heads": heads, "kvheads": kvheads, "dim": dim,
            "page": page, "layout": layout, "tokens": tokens, "seqs": seqs}


def _prompt(name, dtype, heads, kvheads, dim, tokens, seqs, past):
    return {"name": name, "op": "prompt", "dtype": dtype, "heads": heads, "kvheads": kvheads, "dim": dim,
            "tokens": tokens, "seqs": seqs, "past": past}


def _rule(name, op, dtype, heads, kvheads, dim, tokens, seqs, l2):
    return {"name": name, "op": op, "dtype": dtype, "heads": heads, "kvheads": kvheads, "dim": dim,
            "tokens": tokens, "seqs": seqs, "l2": l2}


def listed():
    return [
        # the new token of one chat: latency alone
        _append("append_1", "bf16", "bf16", 16, 2, 256, 16, "token", 1, 64, False, True),
        # a long prompt's rows, odd length
        _append("append_4097", "bf16", "bf16", 16, 2, 256, 64, "token", 4097, 64, False, True),
        # one chat, a short context that ends inside a page
        _decode("decode_1x777", "bf16", 16, 2, 256, 16, "token", 777, 1),
        # a serving batch of ragged contexts, one of a single token and a padded row among them
        _decode("decode_64x4096", "bf16", 16, 2, 256, 64, "token", 4096, 64),
        # one chat over a book, more key heads, the other layout and type
        _decode("decode_1x131071", "f16", 32, 8, 128, 256, "head", 131071, 1),
        # a few short questions packed together, a head of keys for each of queries
        _prompt("prompt_5x611", "f16", 8, 8, 64, 611, 5, 0),
        # one middle-sized prompt, the model's own heads
        _prompt("prompt_1x2048", "bf16", 16, 2, 256, 2048, 1, 0),
        # the largest: long documents packed together
        _prompt("prompt_3x8191", "bf16", 32, 8, 128, 8191, 3, 0),
        # the new token of one chat, the model's own heads
        _rule("step_1", "step", "bf16", 32, 16, 128, 1, 1, True),
        # a serving batch's new tokens
        _rule("step_200", "step", "bf16", 32, 16, 128, 200, 200, True),
        # short questions packed together, activations as the residual holds them
        _rule("delta_3x251", "delta", "f32", 32, 16, 128, 251, 3, True),
        # one long prompt
        _rule("delta_1x4096", "delta", "bf16", 32, 16, 128, 4096, 1, True),
    ]


def _log(rng, lo, hi):
    return int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1.0))))


def draw(rng):
    op = rng.choice(["append", "decode", "decode", "prompt", "prompt", "step", "delta", "delta"])
    heads, kvheads, dim = rng.choice([(16, 2, 256), (16, 2, 256), (32, 8, 128), (8, 8, 64), (12, 4, 128), (7, 1, 64)])
    page, layout = rng.choice([16, 32, 48, 64, 256]), rng.choice(["token", "token", "head"])
    t2 = rng.choice(["bf16", "bf16", "f16"])
    if op == "append":
        c = _append("", rng.choice(["bf16", "f16", "f32"]), t2, heads, kvheads, dim, page, layout, _log(rng, 1, 4097),
                    rng.choice([dim, dim // 2, dim // 4]), rng.random() < 0.3, rng.random() < 0.7)
    elif op == "decode":
        seqs = _log(rng, 1, 200)
        c = _decode("", t2, heads, kvheads, dim, page, layout, _log(rng, 1, 131071 // seqs), seqs)
    elif op == "prompt":
        seqs = rng.choice([1, 1, 2, 3, 5, 8])
        c = _prompt("", t2, heads, kvheads, dim, _log(rng, 8, 8191 if seqs > 2 else 4500), seqs,
                    rng.choice([0, 0, rng.randint(1, 500)]))
    else:
        heads, kvheads, dim = rng.choice([(32, 16, 128), (32, 16, 128), (16, 16, 128), (6, 2, 128), (8, 4, 64)])
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        if op == "step":
            seqs = _log(rng, 1, 200)
            c = _rule("", op, dtype, heads, kvheads, dim, seqs, seqs, rng.random() < 0.8)
        else:
            seqs = rng.choice([1, 1, 2, 3, 8])
            c = _rule("", op, dtype, heads, kvheads, dim, max(seqs, _log(rng, 1, 4096)), seqs, rng.random() < 0.8)
    del c["name"]
    return c


def _lens(case):
    """Lengths of a case's sequences, ragged, the same for every seed."""
    n, t = case["seqs"], case["tokens"]
    r = np.random.RandomState((n * 7919 + t * 31 + case["dim"]) & 0x7FFFFFFF)
    if case["op"] == "step":
        return [1] * n
    if case["op"] == "decode":
        if n == 1:
            return [t]
        lens = np.maximum(1, (t * (0.5 + r.rand(n))).astype(np.int64))
        lens[n // 2] = 1  # a chat that just begins
        if n >= 8:
            lens[-1] = 0  # a padded row
        return [int(v) for v in lens]
    w = 0.3 + r.rand(n)
    cut = np.floor(np.cumsum(w) / w.sum() * (t - n) + 1e-6).astype(np.int64)
    cut[-1] = t - n
    return [int(v) + 1 for v in np.diff(np.concatenate([[0], cut]))]


# ---------------------------------------------------------------- inputs

class _State:
    pass


def _offsets(lens):
    return np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)


def prepare(case, seed):
    s = _State()
    s.case, s.call = dict(case), None
    g = torch.Generator(device="cuda")
    g.manual_seed((int(seed) * 1000003 + case["tokens"] * 8191 + case["dim"]) & 0x7FFFFFFFFFFF)
    r = np.random.RandomState((int(seed) * 2654435761 + case["tokens"]) & 0x7FFFFFFF)
    randn = lambda *shape: torch.randn(*shape, generator=g, device="cuda")
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()
    op, H, K, D, T, dt = case["op"], case["heads"], case["kvheads"], case["dim"], case["tokens"], _DT[case["dtype"]]
    if op in ("append", "decode"):
        cdt, page = _DT[case.get("cache", case["dtype"])], case["page"]
        lens = [T] if op == "append" else _lens(case)
        per = [-(-n // page) for n in lens]
        s.pages = sum(per) + 2
        shape = (s.pages, page, K, D) if case["layout"] == "token" else (s.pages, K, page, D)
        perm = r.permutation(s.pages).astype(np.int32)
    if op == "append":
        # one projection's rows hold q, k and v side by side
        x = randn(T, H + 2 * K, D)
        x[:, :H + K] *= torch.exp(0.5 * randn(1, H + K, 1))
        s.x = x.to(dt)
        s.q, s.k, s.v = s.x[:, :H], s.x[:, H:H + K], s.x[:, H + K:]
        start = int(r.randint(0, 200000))  # this chunk continues a context
        s.pos = dev((start + np.arange(T)).astype(np.int32))
        at = np.arange(T)
        slots = perm[at // page].astype(np.int64) * page + at % page
        if T > 4:
            slots[T // 2] = -1  # a padded row
        s.slots = dev(slots)
        s.inv = (_THETA ** (-torch.arange(0, case["rotary"], 2, dtype=torch.float64) / case["rotary"])).float().cuda()
        s.qw, s.kw = ((0.1 * randn(D)).to(torch.bfloat16) for _ in range(2))
        s.kc, s.vc = torch.zeros(shape, dtype=cdt, device="cuda"), torch.zeros(shape, dtype=cdt, device="cuda")
        s.q_out = torch.zeros(T, H, D, dtype=cdt, device="cuda")
    elif op == "decode":
        n = case["seqs"]
        s.q = (1.5 * randn(n, H, D)).to(dt)
        s.kc, s.vc = randn(*shape).to(dt), randn(*shape).to(dt)
        s.max_len, s.lens = max(lens), dev(np.array(lens, np.int32))
        table = np.zeros((n, max(per)), np.int32)
        at = 0
        for b, p in enumerate(per):
            table[b, :p] = perm[at:at + p]
            at += p
        s.table = dev(table)
        s.out = torch.zeros(n, H, D, dtype=dt, device="cuda")
    elif op == "prompt":
        s.lq = _lens(case)
        s.lk = [n + case["past"] for n in s.lq]
        # normalised queries and keys share a direction, which lets some keys stand out
        s.q = (1.2 * randn(T, H, D) + 0.3 * randn(1, H, D)).to(dt)
        s.k = (randn(sum(s.lk), K, D) + 0.3 * randn(1, K, D)).to(dt)
        s.v = randn(sum(s.lk), K, D).to(dt)
        s.cu_q, s.cu_k = dev(_offsets(s.lq)), dev(_offsets(s.lk))
        s.out = torch.zeros(T, H, D, dtype=dt, device="cuda")
    else:
        n = case["seqs"]
        s.lens = _lens(case)
        shared = 0.0 if case["l2"] else 1.0 / math.sqrt(D)
        s.q, s.k = randn(T, K, D) + 0.4 * randn(1, K, D), randn(T, K, D) + 0.4 * randn(1, K, D)
        if shared:  # a caller that has normalised them already
            s.q, s.k = (t / t.norm(dim=-1, keepdim=True) for t in (s.q, s.k))
        s.q, s.k, s.v = s.q.to(dt), s.k.to(dt), randn(T, H, D).to(dt)
        # decays as a trained gate gives them: from near 1 to forgetting within a few tokens
        s.g = -torch.exp(1.5 * randn(1, H) - 2.5) * torch.nn.functional.softplus(randn(T, H) + 0.5)
        s.beta = torch.sigmoid(randn(T, H))
        s.s_in = 0.1 * randn(n, H, D, D)
        s.s_out = torch.zeros_like(s.s_in)
        s.cu = dev(_offsets(s.lens))
        s.out = torch.zeros(T, H, D, dtype=dt, device="cuda")
    return s


# ----------------------------------------------------------- plain forms

def _pairs(x, rotary, interleaved):
    x = x[..., :rotary]
    return (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :rotary // 2], x[..., rotary // 2:])


def _rotated(s, x, w):
    c = s.case
    x = x.float()
    if c["norm"]:
        x = x * torch.rsqrt(x.square().mean(dim=-1, keepdim=True) + _EPS) * (1.0 + w.float())
    angle = s.pos.double()[:, None] * s.inv.double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    a, b = _pairs(x, c["rotary"], c["interleaved"])
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([a, b], dim=-1).flatten(-2) if c["interleaved"] else torch.cat([a, b], dim=-1)
    return torch.cat([turned, x[..., c["rotary"]:]], dim=-1)


def _by_token(t, case):
    return t if case["layout"] == "token" else t.transpose(1, 2)


def _plain_append(s):
    c = s.case
    page, dt = c["page"], s.kc.dtype
    keep = (s.slots >= 0).nonzero()[:, 0] if c["tokens"] > 4 else slice(None)
    at = s.slots[keep]
    _by_token(s.kc, c)[at // page, at % page] = _rotated(s, s.k, s.kw)[keep].to(dt)
    _by_token(s.vc, c)[at // page, at % page] = s.v[keep].to(dt)
    return {"q": _rotated(s, s.q, s.qw).to(dt), "k": s.kc, "v": s.vc}


def _plain_decode(s):
    c = s.case
    n, H, K, D, page = c["seqs"], c["heads"], c["kvheads"], c["dim"], c["page"]
    at = torch.arange(s.max_len, device="cuda")
    rows = s.table[:, at // page].long(), (at % page)[None]
    k, v = (_by_token(t, c)[rows].float().transpose(1, 2) for t in (s.kc, s.vc))  # [n, K, len, D]
    q = s.q.float().view(n, K, H // K, D)
    p = q @ k.transpose(2, 3) * D ** -0.5
    seen = (at[None] < s.lens[:, None])[:, None, None]
    p = p.masked_fill(~seen, -math.inf)
    top = p.amax(dim=-1, keepdim=True).clamp_min(-1e30)
    p = torch.exp(p - top)
    o = (p @ v) / p.sum(dim=-1, keepdim=True).clamp_min(1e-30)
    return o.view(n, H, D).to(s.out.dtype)


def _padded(lens, cu):
    """Row numbers [sequences, longest] of packed sequences, and which of them are rows."""
    at = torch.arange(max(lens), device="cuda")
    real = at[None] < (cu[1:] - cu[:-1])[:, None]
    return torch.where(real, cu[:-1, None] + at[None], 0).long(), real


def _plain_prompt(s):
    c = s.case
    n, H, K, D = c["seqs"], c["heads"], c["kvheads"], c["dim"]
    iq, rq = _padded(s.lq, s.cu_q)
    ik, rk = _padded(s.lk, s.cu_k)
    q = s.q[iq].float().view(n, -1, K, H // K, D).permute(0, 2, 3, 1, 4)  # [n, K, G, Lq, D]
    k, v = (t[ik].float().transpose(1, 2)[:, :, None] for t in (s.k, s.v))  # [n, K, 1, Lk, D]
    p = q @ k.transpose(3, 4)
    p *= D ** -0.5
    i, j = torch.arange(max(s.lq), device="cuda"), torch.arange(max(s.lk), device="cuda")
    seen = (j[None] <= i[:, None] + c["past"]) & rk[:, None]
    p.masked_fill_(~seen[:, None, None], -math.inf)
    p -= p.amax(dim=-1, keepdim=True).clamp_min(-1e30)
    p.exp_()
    o = (p @ v) / p.sum(dim=-1, keepdim=True)
    return o.permute(0, 3, 1, 2, 4).reshape(n, -1, H, D)[rq].to(s.out.dtype)


def _unit(x, case):
    x = x.float()
    return x * torch.rsqrt(x.square().sum(dim=-1, keepdim=True) + _EPS) if case["l2"] else x


def _plain_step(s):
    c = s.case
    G, D = c["heads"] // c["kvheads"], c["dim"]
    q, k = (_unit(t, c).repeat_interleave(G, dim=1) for t in (s.q, s.k))
    S = s.s_in * torch.exp(s.g)[..., None, None]
    u = s.beta[..., None] * (s.v.float() - (k[..., None, :] @ S)[..., 0, :])
    S = S + k[..., None] * u[..., None, :]
    o = (q[..., None, :] @ S)[..., 0, :] * D ** -0.5
    return {"out": o.to(s.out.dtype), "state": S}


_CHUNK = 64


def _unit_lower_inverse(a):
    """(I + a)^-1 of strictly lower triangular a, by halves: [[x,0],[c,y]]^-1 = [[x',0],[-y'cx',y']]."""
    n = a.shape[-1]
    inv = torch.eye(n, device=a.device).expand_as(a).clone()
    for h in (1, 2, 4, 8, 16, 32):
        m = n // (2 * h)
        grid = lambda t: t.view(*t.shape[:-2], m, 2, h, m, 2, h).diagonal(dim1=-6, dim2=-3)  # [..., 2, h, 2, h, m]
        d, f = grid(inv), grid(a)
        x, y, low = (t.movedim(-1, -3).contiguous() for t in (d[..., 0, :, 0, :, :], d[..., 1, :, 1, :, :], f[..., 1, :, 0, :, :]))
        d[..., 1, :, 0, :, :] = -(y @ low @ x).movedim(-3, -1)
    return inv


def _plain_delta(s):
    c = s.case
    n, H, K, D = c["seqs"], c["heads"], c["kvheads"], c["dim"]
    G, N = H // K, -(-max(s.lens) // _CHUNK)
    rows, real = _padded(s.lens, s.cu)

    def chunks(t):  # [n, heads, N, chunk, ...], zeros behind a sequence
        t = torch.where(real.view(*real.shape, *(1,) * (t.dim() - 1)), t[rows], 0.0)
        t = torch.nn.functional.pad(t, (0, 0) * (t.dim() - 2) + (0, N * _CHUNK - t.shape[1]))
        return t.view(n, N, _CHUNK, *t.shape[2:]).movedim(3, 1)

    q, k = (chunks(_unit(t, c)).repeat_interleave(G, dim=1) for t in (s.q, s.k))
    v, g, beta = chunks(s.v.float()), chunks(s.g), chunks(s.beta)[..., None]
    total = g.double().cumsum(dim=-1)
    decay = torch.exp((total[..., :, None] - total[..., None, :]).tril().float()).tril()
    a = (beta * (k @ k.transpose(-1, -2)) * decay).tril(-1)
    t = _unit_lower_inverse(a)
    since = torch.exp(total.float())[..., None]
    w, u0 = t @ (beta * since * k), t @ (beta * v)
    p = (q @ k.transpose(-1, -2)) * decay
    q, left = q * since, torch.exp((total[..., -1:] - total).float())[..., None] * k
    S, o = s.s_in, []
    for i in range(N):  # a chunk needs the state that the one before leaves
        u = u0[:, :, i] - w[:, :, i] @ S
        o.append(q[:, :, i] @ S + p[:, :, i] @ u)
        S = S * since[:, :, i, -1:] + left[:, :, i].transpose(-1, -2) @ u
    o = torch.stack(o, dim=2).movedim(1, 3).reshape(n, -1, H, D)[:, :rows.shape[1]][real] * D ** -0.5
    return {"out": o.to(s.out.dtype), "state": S}


_PLAIN = {"append": _plain_append, "decode": _plain_decode, "prompt": _plain_prompt, "step": _plain_step,
          "delta": _plain_delta}


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
    op, H, K, D, T = c["op"], c["heads"], c["kvheads"], c["dim"], c["tokens"]
    types = {torch.bfloat16: nh.BF16, torch.float16: nh.F16, torch.float32: nh.F32}
    if op in ("append", "decode"):
        strides = (s.kc.stride(0), _by_token(s.kc, c).stride(1), _by_token(s.kc, c).stride(2))
        cache = nh.Context.kv_cache(p(s.kc), p(s.vc), types[s.kc.dtype], K, D, c["page"], s.pages, *strides)
    if op == "append":
        rows = nh.Context.qkv_rows(p(s.q), p(s.k), p(s.v), types[s.q.dtype], H, K, D, *s.q.stride()[:2],
                                   *s.k.stride()[:2], *s.v.stride()[:2])
        prep = nh.Context.qk_prep(c["rotary"], p(s.inv), c["interleaved"], c["norm"], p(s.qw), p(s.kw), 1, _EPS)
        got = {"q": s.q_out, "k": s.kc, "v": s.vc}
        return lambda: ctx._check(ctx.kv_append(cache, rows, prep, T, p(s.pos), p(s.slots), p(s.q_out), st)) or got
    if op == "decode":
        n = c["seqs"]
        size = ctx.attn_decode_workspace(cache, H, n, s.max_len)
        s.ws = torch.empty(max(size, 16), dtype=torch.uint8, device="cuda")
        return lambda: ctx._check(ctx.attn_decode(cache, p(s.q), H, n, p(s.lens), p(s.table), s.table.shape[1],
                                                  s.max_len, D ** -0.5, p(s.out), None, p(s.ws), size, st)) or s.out
    if op == "prompt":
        rows = nh.Context.qkv_rows(p(s.q), p(s.k), p(s.v), types[s.q.dtype], H, K, D, *s.q.stride()[:2],
                                   *s.k.stride()[:2], *s.v.stride()[:2])
        return lambda: ctx._check(ctx.attn_prompt(rows, c["seqs"], p(s.cu_q), p(s.cu_k), T, s.k.shape[0], max(s.lq),
                                                  max(s.lk), True, D ** -0.5, p(s.out), None, st)) or s.out
    rule = nh.Context.delta_rule(p(s.q), p(s.k), p(s.v), types[s.q.dtype], K, H, D, D, s.q.stride(0), s.k.stride(0),
                                 s.v.stride(0), p(s.g), p(s.beta), D ** -0.5, c["l2"], _EPS, p(s.s_in), p(s.s_out),
                                 None, c["seqs"], p(s.out))
    got = {"out": s.out, "state": s.s_out}
    if op == "step":
        return lambda: ctx._check(ctx.delta_step(rule, c["seqs"], st)) or got
    size = ctx.delta_prompt_workspace(rule, c["seqs"], T)
    s.ws = torch.empty(max(size, 16), dtype=torch.uint8, device="cuda")
    return lambda: ctx._check(ctx.delta_prompt(rule, c["seqs"], p(s.cu), T, max(s.lens), p(s.ws), size, st)) or got


def run(s):
    if not own:
        return _PLAIN[s.case["op"]](s)
    if s.call is None:
        s.call = _bind(s)
    return s.call()


# ------------------------------------------------------------------ work

def work(case):
    op, H, K, D, T = case["op"], case["heads"], case["kvheads"], case["dim"], case["tokens"]
    e = 4 if case["dtype"] == "f32" else 2
    if op == "append":
        return {"bytes": float(T * ((H + 2 * K) * D * (e + 2) + 12)), "flops": 0.0}
    lens = _lens(case)
    if op == "decode":
        n = sum(lens)
        return {"bytes": float(n * 2 * K * D * 2 + 2 * case["seqs"] * H * D * 2), "flops": 4.0 * n * H * D}
    if op == "prompt":
        past = case["past"]
        pairs = sum(n * past + n * (n + 1) / 2 for n in lens)
        return {"bytes": float(2 * T * H * D * 2 + 2 * (T + past * len(lens)) * K * D * 2), "flops": 4.0 * pairs * H * D}
    # k.S, the update by k and u, and q.S of each token and head, as the recurrence has them
    states = 2 * case["seqs"] * H * D * D * 4
    return {"bytes": float(T * ((2 * K + 2 * H) * D * e + 8 * H) + states), "flops": 6.0 * T * H * D * D}


# ----------------------------------------------------------------- exact

def _turn64(s, x, w):
    c = s.case
    x = x.double()
    if c["norm"]:
        x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / c["dim"] + _EPS) * (w.double() + 1)
    out, half = x.clone(), c["rotary"] // 2
    i = torch.arange(half, device=x.device)
    a, b = (2 * i, 2 * i + 1) if c["interleaved"] else (i, i + half)
    z = torch.polar(torch.ones((), dtype=torch.float64, device=x.device), s.pos.double()[:, None] * s.inv.double())
    z = torch.complex(x[..., a], x[..., b]) * z[:, None]
    out[..., a], out[..., b] = z.real, z.imag
    return out


def exact(case, seed):
    s = prepare(case, seed)
    op, H, K, D = case["op"], case["heads"], case["kvheads"], case["dim"]
    if op == "append":
        k, v = torch.zeros_like(s.kc, dtype=torch.float64), torch.zeros_like(s.vc, dtype=torch.float64)
        here = s.slots.cpu().numpy() >= 0
        at = s.slots[torch.from_numpy(here).cuda()]
        for cache, rows in ((k, _turn64(s, s.k, s.kw)), (v, s.v.double())):
            rows = rows[torch.from_numpy(here).cuda()]
            if case["layout"] == "token":
                cache.view(-1, K, D)[at] = rows
            else:
                cache[at // case["page"], :, at % case["page"]] = rows
        return {"q": _turn64(s, s.q, s.qw), "k": k, "v": v}
    if op == "decode":
        out = torch.zeros(case["seqs"], H, D, dtype=torch.float64, device="cuda")
        for b, n in enumerate(_lens(case)):
            if n == 0:
                continue
            pages = s.table[b, :-(-n // case["page"])].long()
            k, v = (t[pages] if case["layout"] == "token" else t[pages].transpose(1, 2) for t in (s.kc, s.vc))
            for h in range(K):
                mine = slice(h * (H // K), (h + 1) * (H // K))
                kh, vh = (t[:, :, h].reshape(-1, D)[:n].double() for t in (k, v))
                out[b, mine] = torch.softmax(s.q[b, mine].double() @ kh.T / math.sqrt(D), dim=-1) @ vh
        return out
    if op == "prompt":
        out = torch.zeros(case["tokens"], H, D, dtype=torch.float64, device="cuda")
        q0 = k0 = 0
        for nq, nk in zip(s.lq, s.lk):
            ban = torch.ones(nq, nk, dtype=torch.bool, device="cuda").triu(nk - nq + 1)
            for h in range(H):
                kh, vh = (t[k0:k0 + nk, h // (H // K)].double() for t in (s.k, s.v))
                p = (s.q[q0:q0 + nq, h].double() @ kh.T / math.sqrt(D)).masked_fill_(ban, -math.inf)
                out[q0:q0 + nq, h] = torch.softmax(p, dim=-1) @ vh
            q0, k0 = q0 + nq, k0 + nk
        return out
    q, k = s.q.double(), s.k.double()
    if case["l2"]:
        q, k = (t / torch.sqrt((t * t).sum(-1, keepdim=True) + _EPS) for t in (q, k))
    q, k = (t[:, torch.arange(H, device="cuda") // (H // K)] / (math.sqrt(D) if t is q else 1) for t in (q, k))
    v, keep, beta = s.v.double(), s.g.double().exp(), s.beta.double()
    S, out = s.s_in.double(), torch.zeros(case["tokens"], H, D, dtype=torch.float64, device="cuda")
    first = np.cumsum([0] + s.lens)
    for t in range(max(s.lens)):  # token t of every sequence that has one
        live = [b for b, n in enumerate(s.lens) if n > t]
        at, live = torch.tensor([int(first[b]) + t for b in live], device="cuda"), torch.tensor(live, device="cuda")
        M = S[live] * keep[at][..., None, None]
        u = (v[at] - (M * k[at][..., None]).sum(-2)) * beta[at][..., None]
        M += k[at][..., None] * u[..., None, :]
        out[at] = (M * q[at][..., None]).sum(-2)
        S[live] = M
    return {"out": out, "state": S}
