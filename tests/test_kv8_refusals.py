"""The checks of the 8-bit context's arguments, on the CPU (as in
test_context_refusals.py: each call is good but for one argument), and that
its structs lie in the header as in the binding."""
import os
import subprocess

import pytest

import nmoe_hip as nh
from conftest import ROOT
from test_context_refusals import A, BAD_PREP, BAD_ROWS, _refused, call, prep, rows  # noqa: F401 (call is a fixture)

STRUCTS = {"nmoe_hip_kv_requests": nh.KvRequests, "nmoe_hip_kv8_cache": nh.Kv8Cache}


def requests(**kw):
    d = dict(page_size=16, num_pages=40, max_pages=8, max_rows=100, lens=A, new_tokens=A, free_count=A, free_pages=A,
             page_table=A, lens_out=A, free_count_out=A, cu=A, status=A, positions=A, slots=A)
    d.update(kw)
    return nh.Context.kv_requests(**d)


def cache8(**kw):
    d = dict(k=A, v=A, k_scale=A, v_scale=A, kv_heads=2, head_dim=128, page_size=16, num_pages=4, page_stride=16 * 256,
             token_stride=256, head_stride=128)
    d.update(kw)
    return nh.Context.kv8_cache(**d)


def append(c, cache_=None, rows_=None, prep_=None, nseq=2, cu=A, ntok=5, lens=A, table=A, max_pages=4, positions=None,
           q_out=A, q_dtype=nh.BF16):
    return c.kv8_append(cache_ or cache8(), rows_ or rows(), prep_ or prep(), nseq, cu, ntok, lens, table, max_pages, positions,
                        q_out, q_dtype)


def decode(c, cache_=None, q=A, q_dtype=nh.BF16, q_heads=4, nseq=2, lens=A, table=A, max_pages=4, max_len=64, scale=0.1,
           out=A, lse=None, ws=A, ws_bytes=1 << 30):
    return c.attn8_decode(cache_ or cache8(), q, q_dtype, q_heads, nseq, lens, table, max_pages, max_len, scale, out, lse,
                          ws, ws_bytes)


def prompt(c, cache_=None, q=A, q_dtype=nh.BF16, q_heads=4, nseq=2, cu=A, ntok=9, lens=A, table=A, max_pages=4, max_q=5,
           max_len=64, causal=1, scale=0.1, out=A, lse=None, ws=A, ws_bytes=1 << 30):
    return c.attn8_prompt(cache_ or cache8(), q, q_dtype, q_heads, nseq, cu, ntok, lens, table, max_pages, max_q, max_len,
                          causal, scale, out, lse, ws, ws_bytes)


BAD_CACHE = [dict(k=None), dict(v=None), dict(k=A + 8), dict(v=A + 4), dict(k_scale=None), dict(v_scale=None),
             dict(k_scale=A + 2), dict(kv_heads=0), dict(kv_heads=2000), dict(head_dim=96), dict(page_size=0),
             dict(page_size=24), dict(num_pages=0), dict(num_pages=1 << 28), dict(page_stride=-16), dict(token_stride=8),
             dict(head_stride=100), dict(page_stride=1 << 34), dict(token_stride=1 << 30), dict(head_stride=1 << 30)]
BAD_ATTEND = [dict(q=None), dict(q=A + 8), dict(q_dtype=nh.F32), dict(q_dtype=5), dict(q_heads=0), dict(q_heads=3),
              dict(q_heads=2000), dict(nseq=-1), dict(nseq=1 << 21), dict(lens=None), dict(lens=A + 2), dict(table=None),
              dict(table=A + 2), dict(max_pages=0), dict(max_len=-1), dict(scale=float("inf")), dict(scale=float("nan")),
              dict(scale=2.0 ** 127), dict(out=None), dict(out=A + 8), dict(lse=A + 2)]


@pytest.mark.parametrize("kw", BAD_CACHE, ids=str)
def test_bad_cache(call, kw):  # noqa: F811
    _refused(call, append(call, cache_=cache8(**kw)))
    _refused(call, decode(call, cache_=cache8(**kw)))
    _refused(call, prompt(call, cache_=cache8(**kw)))
    assert call.attn8_decode_workspace(cache8(**kw), 4, 2, 64) == 0
    assert call.attn8_prompt_workspace(cache8(**kw), 4, 2, 9, 5, 64) == 0


@pytest.mark.parametrize("kw", BAD_ROWS, ids=str)
def test_bad_rows(call, kw):  # noqa: F811
    _refused(call, append(call, rows_=rows(**kw)))


@pytest.mark.parametrize("kw", BAD_PREP, ids=str)
def test_bad_prep(call, kw):  # noqa: F811
    _refused(call, append(call, prep_=prep(**kw)))


@pytest.mark.parametrize("kw", [dict(nseq=-1), dict(nseq=(1 << 20) + 1), dict(ntok=-1), dict(ntok=(1 << 22) + 1),
                                dict(cu=None), dict(cu=A + 2), dict(lens=None), dict(lens=A + 1), dict(table=None),
                                dict(table=A + 2), dict(max_pages=0), dict(positions=A + 2), dict(q_out=None),
                                dict(q_out=A + 4), dict(rows_=rows(q=None)), dict(q_dtype=nh.F32), dict(q_dtype=9),
                                dict(rows_=rows(kv_heads=4)), dict(rows_=rows(head_dim=64))], ids=str)
def test_bad_append(call, kw):  # noqa: F811
    _refused(call, append(call, **kw))


@pytest.mark.parametrize("kw", BAD_ATTEND, ids=str)
def test_bad_attention(call, kw):  # noqa: F811
    _refused(call, decode(call, **kw))
    _refused(call, prompt(call, **kw))


def test_wide_tokens(call):  # noqa: F811
    wide = cache8(token_stride=1 << 24)
    _refused(call, decode(call, cache_=wide))
    _refused(call, prompt(call, cache_=wide))


@pytest.mark.parametrize("kw", [dict(cu=None), dict(cu=A + 2), dict(ntok=-1), dict(ntok=(1 << 22) + 1), dict(max_q=-1),
                                dict(ntok=(1 << 20) + 1, q_heads=1024)], ids=str)
def test_bad_prompt(call, kw):  # noqa: F811
    _refused(call, prompt(call, **kw))


@pytest.mark.parametrize("kw", [dict(page_size=0), dict(page_size=8), dict(page_size=20), dict(num_pages=0),
                                dict(num_pages=1 << 27), dict(max_pages=0), dict(max_pages=(1 << 27) + 1),
                                dict(max_rows=-1), dict(max_rows=(1 << 22) + 1), dict(slots=A + 4), dict(positions=A + 2)] +
                         [{f: p} for f in ("lens", "new_tokens", "free_count", "free_pages", "page_table", "lens_out",
                                           "free_count_out", "cu", "status") for p in (None, A + 2)], ids=str)
def test_bad_requests(call, kw):  # noqa: F811
    _refused(call, call.kv_plan(requests(**kw), 3))


def test_bad_request_counts(call):  # noqa: F811
    _refused(call, call.kv_plan(requests(), -1))
    _refused(call, call.kv_plan(requests(), 65537))
    _refused(call, call.kv_plan(None, 1))


def test_nothing_to_do(call):  # noqa: F811
    """No sequences or no rows: nothing is launched."""
    assert append(call, nseq=0) == nh.OK and append(call, ntok=0) == nh.OK
    assert decode(call, nseq=0) == nh.OK
    assert prompt(call, nseq=0) == nh.OK and prompt(call, ntok=0) == nh.OK


@pytest.mark.parametrize("fn", ["nmoe_kv_plan", "nmoe_kv8_append", "nmoe_attn8_decode", "nmoe_attn8_prompt"])
def test_no_context(fn):
    sig = nh._SIGS[fn][1]
    args = [t(0) if t in (nh.C.c_int, nh.C.c_float, nh.C.c_size_t) else None for t in sig]
    assert getattr(nh.lib(), fn)(*args) == nh.EINVAL


@pytest.mark.parametrize("name", STRUCTS)
def test_struct_layout(name, tmp_path):
    struct = STRUCTS[name]
    fields = [f[0] for f in struct._fields_]
    lines = [f'    printf("%zu %zu\\n", offsetof({name}, {f}), sizeof((({name} *)0)->{f}));' for f in fields]
    (tmp_path / "layout.c").write_text("#include <stdio.h>\n#include \"nmoe_hip.h\"\nint main(void) {\n" +
                                       "\n".join(lines) + f'\n    printf("%zu 0\\n", sizeof({name}));\n    return 0;\n}}\n')
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-I" + os.path.join(ROOT, "include"), "-o",
                    str(tmp_path / "layout"), str(tmp_path / "layout.c")], check=True)
    out = subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True).stdout.split("\n")
    got = [tuple(map(int, line.split())) for line in out if line]
    want = [(getattr(struct, f).offset, getattr(struct, f).size) for f in fields]
    assert got == want + [(nh.C.sizeof(struct), 0)]
