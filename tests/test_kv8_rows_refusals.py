"""The checks of nmoe_attn8_decode_rows' arguments, on the CPU, as in
test_kv8_refusals.py: those of nmoe_attn8_decode, and the offsets'."""
import pytest

import nmoe_hip as nh
from test_context_refusals import A, _refused, call  # noqa: F401 (call is a fixture)
from test_kv8_refusals import BAD_ATTEND, BAD_CACHE, cache8


def decode(c, cache_=None, q=A, q_dtype=nh.BF16, q_heads=4, nseq=2, cu=A, ntok=3, lens=A, table=A, max_pages=4, max_len=64,
           scale=0.1, out=A, lse=None, ws=A, ws_bytes=1 << 30):
    return c.attn8_decode_rows(cache_ or cache8(), q, q_dtype, q_heads, nseq, cu, ntok, lens, table, max_pages, max_len, scale,
                               out, lse, ws, ws_bytes)


@pytest.mark.parametrize("kw", BAD_CACHE, ids=str)
def test_bad_cache(call, kw):  # noqa: F811
    _refused(call, decode(call, cache_=cache8(**kw)))


@pytest.mark.parametrize("kw", BAD_ATTEND + [dict(cu=None), dict(cu=A + 2), dict(ntok=-1), dict(ntok=(1 << 22) + 1)], ids=str)
def test_bad_arguments(call, kw):  # noqa: F811
    _refused(call, decode(call, **kw))


def test_workspace(call):  # noqa: F811
    """As much as without offsets, and refused with less."""
    need = call.attn8_decode_workspace(cache8(), 4, 2, 64)
    assert need > 0
    _refused(call, decode(call, ws_bytes=need - 1))
    _refused(call, decode(call, ws=None, ws_bytes=need))
    _refused(call, decode(call, ws=A + 8, ws_bytes=need))


def test_nothing_to_do(call):  # noqa: F811
    assert decode(call, nseq=0) == nh.OK and decode(call, ntok=0) == nh.OK


def test_no_context():
    sig = nh._SIGS["nmoe_attn8_decode_rows"][1]
    args = [t(0) if t in (nh.C.c_int, nh.C.c_float, nh.C.c_size_t) else None for t in sig]
    assert nh.lib().nmoe_attn8_decode_rows(*args) == nh.EINVAL
