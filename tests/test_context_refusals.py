"""The context operators' checks of their arguments, on the CPU: every check
is made on the host before the first HIP call, so a zeroed stand-in for the
context's memory is enough to hold the message.  Each call is good but for
one argument; the good call itself passes the checks (and then finds no
device here, or is not made where there is one)."""
import ctypes as C

import pytest

import nmoe_hip as nh

A = 0x7F0000001000  # an address, 16-byte aligned, never followed


class Stub:
    """Memory that a refused call may write its message to."""

    def __init__(self):
        self.mem = C.create_string_buffer(1 << 20)
        self.h = C.addressof(self.mem)


@pytest.fixture()
def call():
    ctx = nh.Context.__new__(nh.Context)
    ctx.stub = Stub()
    ctx.h = ctx.stub.h
    yield ctx
    ctx.h = None


def cache(**kw):
    d = dict(k=A, v=A, dtype=nh.BF16, kv_heads=2, head_dim=128, page_size=16, num_pages=4, page_stride=16 * 256,
             token_stride=256, head_stride=128)
    d.update(kw)
    return nh.Context.kv_cache(**d)


def rows(**kw):
    d = dict(q=A, k=A, v=A, dtype=nh.BF16, q_heads=4, kv_heads=2, head_dim=128, q_stride=512, q_head_stride=128,
             k_stride=256, k_head_stride=128, v_stride=256, v_head_stride=128)
    d.update(kw)
    return nh.Context.qkv_rows(**d)


def prep(**kw):
    d = dict(rotary_dim=64, inv_freq=A, qk_norm=True, q_norm=A, k_norm=A)
    d.update(kw)
    return nh.Context.qk_prep(**d)


def rule(**kw):
    d = dict(q=A, k=A, v=A, dtype=nh.BF16, k_heads=2, v_heads=4, k_dim=128, v_dim=128, q_stride=256, k_stride=256,
             v_stride=512, g=A, beta=A, scale=1.0, l2=1, eps=1e-6, state_in=A, state_out=A, state_index=None,
             num_states=3, out=A)
    d.update(kw)
    return nh.Context.delta_rule(**d)


BAD_CACHE = [dict(k=None), dict(v=None), dict(k=A + 8), dict(v=A + 2), dict(dtype=nh.F32), dict(dtype=7),
             dict(kv_heads=0), dict(kv_heads=-1), dict(kv_heads=2000), dict(head_dim=96), dict(head_dim=0),
             dict(page_size=0), dict(page_size=8), dict(page_size=20), dict(page_size=-16), dict(num_pages=0),
             dict(num_pages=1 << 28), dict(page_stride=-8), dict(token_stride=4), dict(head_stride=129),
             dict(page_stride=1 << 34), dict(token_stride=1 << 30), dict(head_stride=1 << 30)]
BAD_ROWS = [dict(q=A + 4), dict(k=None), dict(v=None), dict(k=A + 8), dict(dtype=3), dict(dtype=-1), dict(q_heads=0),
            dict(q_heads=3), dict(q_heads=2000), dict(kv_heads=0), dict(head_dim=32), dict(q_stride=-512),
            dict(k_stride=12), dict(v_head_stride=4), dict(q_stride=1 << 30), dict(k_head_stride=1 << 30)]
BAD_PREP = [dict(rotary_dim=8), dict(rotary_dim=-16), dict(rotary_dim=144), dict(inv_freq=None),
            dict(inv_freq=A + 2), dict(eps=-1.0), dict(eps=float("nan")), dict(q_norm=A + 2), dict(k_norm=A + 8)]
BAD_RULE = [dict(q=None), dict(k=A + 8), dict(v=None), dict(dtype=5), dict(k_heads=0), dict(v_heads=3),
            dict(v_heads=0), dict(v_heads=2048), dict(k_dim=96), dict(v_dim=256), dict(q_stride=4),
            dict(v_stride=-512), dict(k_stride=1 << 30), dict(g=None), dict(beta=None), dict(beta=A + 2), dict(scale=float("inf")),
            dict(eps=-1.0), dict(eps=float("nan")), dict(state_out=None), dict(state_out=A + 4),
            dict(state_in=A + 8), dict(state_index=A + 1), dict(num_states=0), dict(out=None), dict(out=A + 8)]


def append(c, cache_=None, rows_=None, prep_=None, ntok=3, positions=A, slots=A, q_out=A):
    return c.kv_append(cache_ or cache(), rows_ or rows(), prep_ or prep(), ntok, positions, slots, q_out)


def decode(c, cache_=None, q=A, q_heads=4, nseq=2, lens=A, table=A, max_pages=4, max_len=64, scale=0.1, out=A,
           lse=None, ws=A, ws_bytes=1 << 30):
    return c.attn_decode(cache_ or cache(), q, q_heads, nseq, lens, table, max_pages, max_len, scale, out, lse, ws,
                         ws_bytes)


def prompt(c, rows_=None, nseq=2, cu_q=A, cu_k=None, ntok_q=9, ntok_k=9, max_q=5, max_k=5, causal=1, scale=0.1,
           out=A, lse=None):
    return c.attn_prompt(rows_ or rows(), nseq, cu_q, cu_k, ntok_q, ntok_k, max_q, max_k, causal, scale, out, lse)


def _refused(c, rc):
    assert rc == nh.EINVAL, rc
    assert c.last_error()


@pytest.mark.parametrize("kw", BAD_CACHE, ids=str)
def test_bad_cache(call, kw):
    _refused(call, append(call, cache_=cache(**kw)))
    _refused(call, decode(call, cache_=cache(**kw)))
    assert call.attn_decode_workspace(cache(**kw), 4, 2, 64) == 0


@pytest.mark.parametrize("kw", BAD_ROWS, ids=str)
def test_bad_rows(call, kw):
    _refused(call, append(call, rows_=rows(**kw)))
    _refused(call, prompt(call, rows_=rows(**kw)))


@pytest.mark.parametrize("kw", BAD_PREP, ids=str)
def test_bad_prep(call, kw):
    _refused(call, append(call, prep_=prep(**kw)))


@pytest.mark.parametrize("kw", [dict(ntok=-1), dict(ntok=(1 << 22) + 1), dict(positions=None), dict(slots=None), dict(slots=A + 4),
                                dict(q_out=None), dict(q_out=A + 2), dict(rows_=rows(q=None)),
                                dict(rows_=rows(kv_heads=4)), dict(rows_=rows(head_dim=64))], ids=str)
def test_bad_append(call, kw):
    _refused(call, append(call, **kw))


@pytest.mark.parametrize("kw", [dict(q=None), dict(q=A + 8), dict(q_heads=3), dict(q_heads=0), dict(q_heads=2048),
                                dict(nseq=-1), dict(nseq=1 << 30), dict(lens=None), dict(table=None),
                                dict(table=A + 2), dict(max_pages=0), dict(max_len=-1), dict(scale=float("nan")),
                                dict(scale=float("inf")), dict(out=None), dict(out=A + 8), dict(lse=A + 2),
                                dict(cache_=cache(token_stride=1 << 24))], ids=str)
def test_bad_decode(call, kw):
    _refused(call, decode(call, **kw))


@pytest.mark.parametrize("kw", [dict(nseq=-1), dict(nseq=1 << 21), dict(cu_q=None), dict(cu_q=A + 2),
                                dict(cu_k=A + 1), dict(ntok_q=-1), dict(ntok_q=(1 << 30) + 1), dict(ntok_k=-1), dict(max_q=-1), dict(max_k=-1),
                                dict(scale=float("nan")), dict(out=None), dict(out=A + 4), dict(lse=A + 3),
                                dict(rows_=rows(dtype=nh.F32)), dict(rows_=rows(k_stride=1 << 24)),
                                dict(rows_=rows(v_stride=1 << 24))], ids=str)
def test_bad_prompt(call, kw):
    _refused(call, prompt(call, **kw))


@pytest.mark.parametrize("kw", BAD_RULE, ids=str)
def test_bad_rule(call, kw):
    _refused(call, call.delta_step(rule(**kw), 2))
    _refused(call, call.delta_prompt(rule(**kw), 2, A, 9, 5, A, 1 << 40))
    assert call.delta_prompt_workspace(rule(**kw), 2, 9) == 0


def test_bad_delta_sizes(call):
    _refused(call, call.delta_step(rule(), -1))
    _refused(call, call.delta_step(rule(), 1 << 30))
    for nseq, cu, ntok, max_len in ((-1, A, 9, 5), (2, None, 9, 5), (2, A + 2, 9, 5), (2, A, -1, 5), (2, A, 9, -1)):
        _refused(call, call.delta_prompt(rule(), nseq, cu, ntok, max_len, A, 1 << 40))


def test_no_context():
    c = nh.Context.__new__(nh.Context)
    c.h = None
    assert append(c) == decode(c) == prompt(c) == nh.EINVAL
    assert c.delta_step(rule(), 1) == c.delta_prompt(rule(), 1, A, 9, 5) == nh.EINVAL
    assert c.attn_decode_workspace(cache(), 4, 2, 64) == c.delta_prompt_workspace(rule(), 2, 9) == 0


def test_nothing_to_do(call):
    """No rows or sequences: accepted, with nothing launched."""
    assert append(call, ntok=0) == nh.OK
    assert decode(call, nseq=0) == nh.OK
    assert prompt(call, nseq=0) == nh.OK
    assert prompt(call, ntok_q=0) == nh.OK
    assert call.delta_step(rule(), 0) == nh.OK
    assert call.delta_prompt(rule(), 0, A, 9, 5, A, 1 << 40) == nh.OK


def test_workspace_too_small(call):
    need = call.attn_decode_workspace(cache(), 4, 2, 100000)
    if need:
        _refused(call, decode(call, max_len=100000, ws_bytes=need - 1))
        _refused(call, decode(call, max_len=100000, ws=None, ws_bytes=need))
        _refused(call, decode(call, max_len=100000, ws=A + 8, ws_bytes=need))
    need = call.delta_prompt_workspace(rule(), 2, 300)
    if need:
        _refused(call, call.delta_prompt(rule(), 2, A, 300, 200, A, need - 1))
        _refused(call, call.delta_prompt(rule(), 2, A, 300, 200, None, need))
        _refused(call, call.delta_prompt(rule(), 2, A, 300, 200, A + 8, need))


@pytest.mark.parametrize("scale", [2.0 ** 127, -2.0 ** 127, 3.4e38])
def test_scale_in_powers_of_two_overflows(call, scale):
    """Scores are taken in powers of two: scale * log2(e) has to be finite."""
    _refused(call, decode(call, scale=scale))
    _refused(call, prompt(call, scale=scale))
