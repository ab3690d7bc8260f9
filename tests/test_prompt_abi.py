"""The prompt table without a GPU: the C header against the ctypes mirror, the
table's place in the quantized extension, and the refusals that need no device."""
import ctypes
import os
import subprocess

import pytest

from mlx_amd import abi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "lux_gpu_prompt_backend.h")
RECORDS = {"lux_paged_chunk_args": abi.PagedChunkArgs, "lux_paged_fork_args": abi.PagedForkArgs, "lux_paged_release_args": abi.PagedReleaseArgs,
           "lux_paged_compact_args": abi.PagedCompactArgs, "lux_paged_copy_args": abi.PagedCopyArgs,
           "lux_token_logprobs_args": abi.TokenLogprobsArgs, "lux_gpu_prompt_vtbl": abi.PromptVtbl}
OPS = {"op_paged_chunk_attention": abi.PagedChunkArgs, "op_paged_fork": abi.PagedForkArgs, "op_paged_release": abi.PagedReleaseArgs,
       "op_paged_compact": abi.PagedCompactArgs, "op_paged_copy": abi.PagedCopyArgs, "op_token_logprobs": abi.TokenLogprobsArgs}


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
    return p.contents.prompt.contents


def test_table(table):
    assert table.ext_version == abi.PROMPT_EXT_VERSION and table.struct_size == ctypes.sizeof(abi.PromptVtbl)
    assert list(table._reserved) == [None] * 8
    assert all(ctypes.cast(getattr(table, op), ctypes.c_void_p).value for op in OPS)


def test_no_context_is_refused(table):
    for op, t in OPS.items():
        assert getattr(table, op)(None, t()) == abi.ERR_INVALID_ARGUMENT
        assert getattr(table, op)(None, None) == abi.ERR_INVALID_ARGUMENT


def test_records_carry_their_size():
    for t in OPS.values():
        assert t().struct_size == ctypes.sizeof(t)
    a = abi.TokenLogprobsArgs(rows=3, vocab=7, scale=0.5, lse=0x1000)
    assert (a.rows, a.vocab, a.scale, a.lse, a.tokens) == (3, 7, 0.5, 0x1000, None)


def test_a_plugin_without_the_table():
    """Contexts of plugins that predate the table say so instead of calling nothing."""
    from mlx_amd import runtime
    ctx = runtime.Context.__new__(runtime.Context)
    quant = abi.QuantVtbl()
    ctx.q = quant
    ctx.p = None
    with pytest.raises(runtime.LuxError) as e:
        ctx.paged_fork(abi.PagedForkArgs())
    assert e.value.code == abi.ERR_NOT_SUPPORTED
