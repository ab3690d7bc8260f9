"""The serving table without a GPU: the C header against the ctypes mirror, the
table's place in the quantized extension, and the refusals that need no device."""
import ctypes
import os
import subprocess

import pytest

from mlx_amd import abi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "lux_gpu_serving_backend.h")
RECORDS = {"lux_paged_plan_args": abi.PagedPlanArgs, "lux_paged_append_args": abi.PagedAppendArgs,
           "lux_paged_attention_args": abi.PagedAttentionArgs, "lux_block_norm_args": abi.BlockNormArgs,
           "lux_gpu_serving_vtbl": abi.ServingVtbl}


def test_header_compiles_as_c_and_cpp(tmp_path):
    src = tmp_path / "t.c"
    src.write_text(f'#include "{HEADER}"\nint main(void){{return 0;}}\n')
    for cc in (["gcc", "-std=c11"], ["g++", "-std=c++17", "-x", "c++"]):
        r = subprocess.run([*cc, "-Wall", "-Werror", "-fsyntax-only", str(src)], capture_output=True, text=True)
        assert r.returncode == 0, r.stderr


def test_every_field_is_where_the_mirror_has_it(tmp_path):
    lines, want = [], []
    for c_name, t in RECORDS.items():
        for f in t._fields_:
            lines.append(f'printf("%zu %zu\\n", offsetof({c_name}, {f[0]}), sizeof((({c_name}*)0)->{f[0]}));')
            want.append((getattr(t, f[0]).offset, getattr(t, f[0]).size))
        lines.append(f'printf("%zu 0\\n", sizeof({c_name}));')
        want.append((ctypes.sizeof(t), 0))
    src = tmp_path / "t.c"
    src.write_text(f'#include <stddef.h>\n#include <stdio.h>\n#include "{HEADER}"\nint main(void){{{" ".join(lines)} return 0;}}\n')
    subprocess.run(["gcc", "-std=c11", str(src), "-o", str(tmp_path / "t")], check=True)
    out = subprocess.run([str(tmp_path / "t")], capture_output=True, text=True, check=True).stdout
    assert [tuple(map(int, line.split())) for line in out.splitlines()] == want


@pytest.fixture(scope="module")
def table():
    import mlx_amd
    assert mlx_amd.plugin_built(), "run __graft_entry__.build() first"
    lib = ctypes.CDLL(mlx_amd.PLUGIN_PATH, mode=os.RTLD_NOW | os.RTLD_LOCAL)
    p = ctypes.POINTER(abi.QuantVtbl)()
    assert abi.QUANT_INIT_FN((abi.QUANT_INIT_SYMBOL.decode(), lib))(ctypes.byref(p))
    return p.contents.serving.contents


def test_table(table):
    assert table.ext_version == abi.SERVING_EXT_VERSION and table.struct_size == ctypes.sizeof(abi.ServingVtbl)
    assert list(table._reserved) == [None] * 5


def test_no_context_is_refused(table):
    for op, t in [("op_paged_plan", abi.PagedPlanArgs), ("op_paged_append", abi.PagedAppendArgs),
                  ("op_paged_attention", abi.PagedAttentionArgs), ("op_block_norm", abi.BlockNormArgs)]:
        assert getattr(table, op)(None, t()) == abi.ERR_INVALID_ARGUMENT
        assert getattr(table, op)(None, None) == abi.ERR_INVALID_ARGUMENT
    assert table.buffer_wrap(None, 4096, 16) is None


def test_records_carry_their_size():
    for t in list(RECORDS.values())[:4]:
        assert t().struct_size == ctypes.sizeof(t)
    a = abi.BlockNormArgs(rows=3, eps=0.5, out=0x1000)
    assert (a.rows, a.eps, a.out, a.x) == (3, 0.5, 0x1000, None)
