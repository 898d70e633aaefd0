"""The paged cache's argument structs: the C layout, the ctypes mirror and the command's room."""
from __future__ import annotations

import ctypes as C
import subprocess

import vnpu
from test_abi import INCLUDE

STRUCTS = {"vnpu_b200_paged_cache_t": vnpu.PagedCache, "vnpu_b200_paged_batch_t": vnpu.PagedBatch,
           "vnpu_b200_paged_kv_append_args_t": vnpu.PagedKvAppendArgs,
           "vnpu_b200_paged_kv_read_args_t": vnpu.PagedKvReadArgs,
           "vnpu_b200_paged_attention_args_t": vnpu.PagedAttentionArgs}


def test_layouts_match_the_mirror(tmp_path):
    lines = []
    for name, mirror in STRUCTS.items():
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        lines += [f'printf("{name}.{f} %zu\\n", offsetof({name}, {f}));' for f, _ in mirror._fields_]
    ops = {"VNPU_B200_OP_PAGED_KV_APPEND": vnpu.OP_B200_PAGED_KV_APPEND,
           "VNPU_B200_OP_PAGED_KV_READ": vnpu.OP_B200_PAGED_KV_READ,
           "VNPU_B200_OP_PAGED_ATTENTION": vnpu.OP_B200_PAGED_ATTENTION,
           "VNPU_B200_PAGED_INTERLEAVED": vnpu.PAGED_INTERLEAVED,
           "VNPU_B200_PAGED_NO_ROPE": vnpu.PAGED_NO_ROPE}
    lines += [f'printf("{o} %u\\n", (unsigned){o});' for o in ops]
    src = tmp_path / "paged.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "vnpu_b200.h"\nint main(void){' +
                   "".join(lines) + "return 0;}")
    subprocess.run(["gcc", "-std=c11", "-I", INCLUDE, str(src), "-o", str(tmp_path / "paged")], check=True)
    out = subprocess.run([str(tmp_path / "paged")], check=True, capture_output=True, text=True).stdout
    table = {k: int(v) for k, v in (line.rsplit(" ", 1) for line in out.strip().splitlines())}
    for name, mirror in STRUCTS.items():
        assert table[name] == C.sizeof(mirror) <= 192
        for f, _ in mirror._fields_:
            assert table[f"{name}.{f}"] == getattr(mirror, f).offset, (name, f)
    for o, value in ops.items():
        assert table[o] == value


def test_opcode_names(b200_lib):
    name = b200_lib.h.vnpu_opcode_name
    name.restype, name.argtypes = C.c_char_p, [C.c_uint32]
    assert name(vnpu.OP_B200_PAGED_KV_APPEND) == b"PAGED_KV_APPEND"
    assert name(vnpu.OP_B200_PAGED_KV_READ) == b"PAGED_KV_READ"
    assert name(vnpu.OP_B200_PAGED_ATTENTION) == b"PAGED_ATTENTION"
