"""Waits that gfx9 leaves to the program, in the library as it was built.

The compiler keeps them for the instructions that it issues; it does not look into inline assembly, which the direct
loads into LDS are.  A vector memory access needs 5 wait states behind a vector instruction that writes a scalar register
it reads (a v_readlane that brings back a spilled descriptor), and a load into LDS one behind the write of M0.  An
instruction is a state, s_nop n is n + 1."""
import os
import re
import struct
import subprocess

import pytest

from litevllm_amd import build as B

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"
_MEMORY = re.compile(r"\s*(?:buffer|global|scratch)_")
_SCALAR = re.compile(r"\bs(?:\[(\d+):(\d+)\]|(\d+))")


def _scalars(text):
    out = set()
    for lo, hi, one in _SCALAR.findall(text):
        out.update(range(int(lo), int(hi) + 1) if lo else [int(one)])
    return out


def missing_waits(lines):
    """(line, states there are, states needed) of each access that comes too early; lines of assembly in order."""
    bad, last = [], []  # last: (scalar registers that a vector instruction wrote, whether M0 was written, states)
    for line in lines:
        text = line.split("//")[0].split(";")[0].strip()
        if not text or text.endswith(":"):
            continue
        op = text.split()[0]
        if _MEMORY.match(text):
            reads, into_lds, since = None, text.endswith(" lds"), 0
            for wrote, m0, states in reversed(last):
                if into_lds and m0 and since < 1:
                    bad.append((text, since, 1))
                if wrote and wrote & (reads := _scalars(text) if reads is None else reads):
                    bad.append((text, since, 5))
                since += states
                if since >= 5:
                    break
        wrote = set()
        if op.startswith(("v_readlane", "v_readfirstlane", "v_cmp")):
            wrote = _scalars(text.split(",")[0])
        elif "_co_" in op:
            wrote = _scalars(text.split(",")[1])
        states = int(text.split()[1], 0) + 1 if op == "s_nop" else 1
        last = (last + [(wrote, op.startswith("s_") and bool(re.match(r"\S+\s+m0\b", text)), states)])[-5:]
    return bad


def _code_objects(data):
    """The gfx950 code objects of a library's offload bundles."""
    at = data.find(b"__CLANG_OFFLOAD_BUNDLE__")
    while at >= 0:
        entries, = struct.unpack_from("<Q", data, at + 24)
        p = at + 32
        for _ in range(entries):
            offset, size, length = struct.unpack_from("<QQQ", data, p)
            if size and B.ARCH.encode() in data[p + 24:p + 24 + length]:
                yield data[at + offset:at + offset + size]
            p += 24 + length
        at = data.find(b"__CLANG_OFFLOAD_BUNDLE__", at + 24)


def test_the_scan_finds_what_it_is_for():
    early = ["v_readlane_b32 s4, v107, 3", "s_mov_b32 m0, s8", "buffer_load_dwordx4 v73, s[68:71], s4 offen lds"]
    assert [b[1:] for b in missing_waits(early)] == [(0, 1), (1, 5)]
    assert missing_waits(early[:2] + ["s_nop 3", early[2]]) == []
    assert [b[1:] for b in missing_waits(early[:2] + ["s_nop 2", early[2]])] == [(4, 5)]
    assert [b[1:] for b in missing_waits(["v_readfirstlane_b32 s70, v1", "s_nop 3", "global_load_dword v1, v2, s[70:71]"])] == [(4, 5)]
    assert missing_waits(["v_readlane_b32 s4, v107, 3", "s_add_u32 s5, s4, 1", "buffer_load_dword v1, v2, s[8:11], s5 offen"]) == []


@pytest.mark.skipif(not (os.path.exists(B.OUT) and os.path.exists(OBJDUMP)), reason="needs the built library and a disassembler")
def test_the_built_library_keeps_them(tmp_path):
    objects = list(_code_objects(open(B.OUT, "rb").read()))
    assert objects
    loads = 0
    for i, code in enumerate(objects):
        path = tmp_path / f"{i}.co"
        path.write_bytes(code)
        lines = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", str(path)], check=True, capture_output=True, text=True).stdout.splitlines()
        loads += sum(" lds " in line or line.rstrip().endswith(" lds") for line in lines if "buffer_load" in line)
        bad = missing_waits(lines)
        assert not bad, (len(bad), bad[:3])
    assert loads > 100
