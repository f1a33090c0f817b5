"""The context operators' structs lie in the header as in the binding: sizes
and every field's offset, from a C program on the header."""
import os
import subprocess

import pytest

import nmoe_hip as nh
from conftest import ROOT

STRUCTS = {"nmoe_hip_qkv": nh.Qkv, "nmoe_hip_kv_cache": nh.KvCache, "nmoe_hip_qk_prep": nh.QkPrep,
           "nmoe_hip_delta_rule": nh.DeltaRule}


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
