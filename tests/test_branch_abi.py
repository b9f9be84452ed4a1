"""include/dsr_branch.h against the binding and the library, without a GPU:
exports, constants, struct layouts, argument errors ahead of any launch."""
import ctypes
import os
import re
import subprocess

import pytest

from deepseekrpc_amd import _native as N
from tests.test_tree_abi import refused

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "dsr_branch.h")
STRUCTS = {"dsr_select_beams_args_t": N.SelectBeamsArgs, "dsr_fork_args_t": N.ForkArgs,
           "dsr_compact_args_t": N.CompactArgs, "dsr_prefix_attention_args_t": N.PrefixAttentionArgs}
CALLS = {"dsr_select_beams": N.SelectBeamsArgs, "dsr_fork_pages": N.ForkArgs, "dsr_compact_pages": N.CompactArgs,
         "dsr_prefix_attention": N.PrefixAttentionArgs}


def test_exports_and_constants():
    text = open(HEADER).read()
    lib = N.load()
    names = set(re.findall(r"^\s*(?:int32_t|size_t)\s+(dsr_\w+)\s*\(", text, re.M))
    assert names == set(N.BRANCH_EXPORTS)
    for name in names:
        assert hasattr(lib, name), name
    defs = {m.group(1): int(m.group(2)) for m in re.finditer(r"#define (DSR_\w+) \(?(-?\d+)u?\)?", text)}
    for name in ("E_PARENT", "BEAMS_MAX_KEEP", "BEAMS_MAX_VOCAB", "BEAMS_MAX_ROWS"):
        assert getattr(N, name) == defs["DSR_" + name], name
    assert "unknown" not in N.status_message(N.E_PARENT)


def test_struct_layouts(tmp_path):
    lines = [f'printf("{c} size %zu\\n", sizeof({c}));' for c in STRUCTS]
    lines += [f'printf("{c} {f} %zu\\n", offsetof({c}, {f}));' for c, s in STRUCTS.items() for f, _ in s._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "dsr_branch.h"\nint main(void) {\n'
                   + "\n".join(lines) + "\nreturn 0; }\n")
    subprocess.run(["gcc", "-std=c99", f"-I{os.path.dirname(HEADER)}", str(src), "-o", str(exe)], check=True)
    got = {}
    for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines():
        c, f, off = line.split()
        got[c, f] = int(off)
    for c, s in STRUCTS.items():
        assert got[c, "size"] == ctypes.sizeof(s), c
        for f, _ in s._fields_:
            assert got[c, f] == getattr(s, f).offset, (c, f)


@pytest.mark.parametrize("name", list(CALLS))
def test_null_arguments(name):
    lib = N.load()
    assert getattr(lib, name)(None, None) == -1
    assert getattr(lib, name)(ctypes.byref(CALLS[name]()), None) == -1


def test_beam_arguments():
    lib = N.load()
    a = N.SelectBeamsArgs()
    for f in ("logits", "scores", "offsets", "parents", "tokens", "out_scores", "status", "workspace"):
        setattr(a, f, 4096)
    a.dtype, a.keep, a.rows, a.groups, a.vocab, a.ld = N.BF16, 8, 6, 2, 100, 104
    a.workspace_bytes = lib.dsr_select_beams_workspace_bytes(ctypes.byref(a))
    assert a.workspace_bytes > 0
    refused(lib.dsr_select_beams, a, [("dtype", 0), ("dtype", N.F64), ("keep", 0), ("keep", 65), ("rows", -1),
                                      ("rows", N.BEAMS_MAX_ROWS + 1), ("groups", -1), ("groups", N.BEAMS_MAX_ROWS + 1),
                                      ("vocab", 0), ("vocab", N.BEAMS_MAX_VOCAB + 1), ("ld", 99), ("logits", None),
                                      ("scores", None), ("offsets", None), ("parents", None), ("tokens", None),
                                      ("out_scores", None), ("status", None)])
    refused(lib.dsr_select_beams, a, [("workspace", None), ("workspace", 4104),
                                      ("workspace_bytes", a.workspace_bytes - 1)], -3)
    a.rows = a.groups = 0
    assert lib.dsr_select_beams(ctypes.byref(a), None) == 0
    a.keep = 0
    assert lib.dsr_select_beams_workspace_bytes(ctypes.byref(a)) == 0
    assert lib.dsr_select_beams_workspace_bytes(None) == 0


CACHES = [("cache_count", -1), ("cache_count", 65536), ("caches", None), ("host_caches", 4096), ("heads", 0),
          ("heads", 65537), ("row_bytes", 0), ("row_bytes", 24), ("row_bytes", 65552), ("c_block", 8), ("c_token", 8),
          ("c_head", 8)]
TABLES = [("rows", -1), ("rows", N.TREE_MAX_REQUESTS + 1), ("table_ld", 3), ("table_out_ld", 3), ("width", 0),
          ("width", 2**28), ("page", 0), ("page", 12), ("page", 2048), ("blocks", 0), ("blocks", 2**28),
          ("pool_size", 0), ("pool_size", 2**30 + 1)]


def test_fork_arguments():
    lib = N.load()
    a = N.ForkArgs()
    for i, f in enumerate(("lengths", "held", "table", "parents", "shared", "pool_state", "pool", "table_out",
                           "held_out", "lengths_out", "status", "source_status", "caches", "workspace")):
        setattr(a, f, 4096 * (i + 1))
    a.shared_out, a.pool_state_out = a.shared, a.pool_state
    a.sources, a.rows, a.table_ld, a.table_out_ld, a.width, a.page, a.blocks, a.pool_size = 3, 4, 4, 4, 4, 16, 9, 9
    a.cache_count, a.heads, a.row_bytes, a.c_block, a.c_token, a.c_head = 3, 2, 256, 8192, 512, 256
    a.workspace_bytes = lib.dsr_fork_workspace_bytes(ctypes.byref(a))
    assert a.workspace_bytes > 0
    refused(lib.dsr_fork_pages, a, CACHES + TABLES + [
        ("sources", -1), ("sources", N.TREE_MAX_REQUESTS + 1), ("reserved", 1), ("lengths", None), ("held", None),
        ("table", None), ("parents", None), ("shared", None), ("pool_state", None), ("pool", None),
        ("table_out", None), ("table_out", a.table), ("held_out", None), ("held_out", a.held), ("held_out", a.parents),
        ("lengths_out", None), ("lengths_out", a.lengths), ("lengths_out", a.parents), ("shared_out", None),
        ("pool_state_out", None), ("status", None), ("source_status", None)])
    refused(lib.dsr_fork_pages, a, [("workspace", None), ("workspace", 4104),
                                    ("workspace_bytes", a.workspace_bytes - 1)], -3)
    a.heads, a.row_bytes, a.page = 65536, 65536, 1  # a page of 2^32 bytes
    assert lib.dsr_fork_pages(ctypes.byref(a), None) == -1
    assert lib.dsr_fork_workspace_bytes(ctypes.byref(a)) == lib.dsr_fork_workspace_bytes(None) == 0


def test_compact_arguments():
    lib = N.load()
    a = N.CompactArgs()
    for i, f in enumerate(("held", "table", "shared", "pool", "pool_state", "remap", "status", "caches", "workspace")):
        setattr(a, f, 4096 * (i + 1))
    a.table_out, a.shared_out, a.pool_out, a.pool_state_out = a.table, a.shared, a.pool, a.pool_state
    a.rows, a.table_ld, a.table_out_ld, a.width, a.page, a.blocks, a.pool_size, a.first = 4, 4, 4, 4, 16, 9, 8, 1
    a.cache_count, a.heads, a.row_bytes, a.c_block, a.c_token, a.c_head = 3, 2, 256, 8192, 512, 256
    a.workspace_bytes = lib.dsr_compact_workspace_bytes(ctypes.byref(a))
    assert a.workspace_bytes > 0
    refused(lib.dsr_compact_pages, a, CACHES + TABLES + [
        ("first", -1), ("first", 0), ("first", 9), ("pool_size", 7), ("held", None), ("table", None), ("shared", None),
        ("shared_out", None), ("pool", None), ("pool_out", None), ("pool_state", None), ("pool_state_out", None),
        ("remap", None), ("status", None), ("table_out", None), ("table_out_ld", 5)])
    refused(lib.dsr_compact_pages, a, [("workspace", None), ("workspace", 4104),
                                       ("workspace_bytes", a.workspace_bytes - 1)], -3)
    a.first = 9
    assert lib.dsr_compact_workspace_bytes(ctypes.byref(a)) == lib.dsr_compact_workspace_bytes(None) == 0


def test_prefix_arguments():
    lib = N.load()
    a = N.PrefixAttentionArgs()
    for f in ("q", "k_cache", "v_cache", "table", "offsets", "kv_lengths", "out", "status", "workspace", "groups",
              "prefix_lengths"):
        setattr(a, f, 4096)
    a.dtype, a.q_heads, a.kv_heads, a.head_dim, a.page, a.width, a.blocks = N.BF16, 8, 2, 128, 16, 4, 9
    a.scale, a.requests, a.tokens, a.table_ld, a.group_count = 0.1, 3, 5, 4, 2
    a.workspace_bytes = lib.dsr_prefix_attention_workspace_bytes(ctypes.byref(a))
    assert a.workspace_bytes >= lib.dsr_tree_attention_workspace_bytes(ctypes.byref(a.a)) > 0
    refused(lib.dsr_prefix_attention, a, [("group_count", -1), ("group_count", 4), ("groups", None),
                                          ("prefix_lengths", None), ("dtype", N.F32), ("q_heads", 7), ("kv_heads", 0),
                                          ("head_dim", 4), ("head_dim", 100), ("head_dim", 264), ("page", 5),
                                          ("width", 0), ("blocks", 0), ("scale", float("nan")), ("scale", float("inf")),
                                          ("requests", -1), ("requests", 1), ("requests", N.TREE_MAX_REQUESTS + 1),
                                          ("tokens", -1), ("tokens", 2**31), ("table_ld", 3), ("q", None),
                                          ("out", None), ("q", 4104), ("out", 4104), ("k_cache", 4104),
                                          ("v_cache", 4104), ("table", None), ("offsets", None), ("kv_lengths", None),
                                          ("status", None), ("q_token", 4), ("q_head", 4), ("out_token", 1),
                                          ("out_head", 2), ("k_block", 4), ("k_token", 12), ("k_head", 4),
                                          ("v_block", 4), ("v_token", 4), ("v_head", 4), ("k_block", 2**31),
                                          ("k_token", 2**31), ("v_block", 2**31), ("v_token", 2**31), ("k_head", -8),
                                          ("q_token", -8)])
    refused(lib.dsr_prefix_attention, a, [("workspace", None), ("workspace", 4352 - 128),
                                          ("workspace_bytes", a.workspace_bytes - 1)], -3)
    assert lib.dsr_prefix_attention_workspace_bytes(None) == 0
    # Without groups it is dsr_tree_attention, whose checks hold.
    a.group_count, a.head_dim = 0, 100
    assert lib.dsr_prefix_attention(ctypes.byref(a), None) == -1
    a.head_dim, a.requests, a.tokens = 128, 0, 0
    assert lib.dsr_prefix_attention(ctypes.byref(a), None) == 0
