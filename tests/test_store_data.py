"""CPU: the stores of the built gfx950 code.  The memory unit fetches the data of a store of more than 8 bytes after the instruction was issued; a vector instruction right
behind it that writes the same registers comes too early.  hipcc keeps the distance, except behind a buffer store whose scalar offset is a register, where gfx950 stores
the new value in some lanes all the same (seen: 160 of 6 million outputs of a product, in every call)."""
import os
import re
import shutil
import subprocess

import pytest

from dist_amd import build as b

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"
WIDE = re.compile(r"\s+(buffer|global|flat|scratch)_store_(?:dwordx[34]|b96|b128)\s+(.*?)\s*(?://.*)?$")
WRITE = re.compile(r"\s+v_(?!cmp_|cmpx_|nop)\S+\s+(v\[?[0-9:]+\]?)")


def _registers(text):
    m = re.match(r"v\[(\d+):(\d+)\]$", text)
    if m:
        return set(range(int(m[1]), int(m[2]) + 1))
    m = re.match(r"v(\d+)$", text)
    return {int(m[1])} if m else set()


@pytest.fixture(scope="module")
def code(tmp_path_factory):
    """the built library's gfx950 code, one list of instruction lines per source"""
    if not os.path.exists(b.LIB):
        b.build_library(verbose=False)
    at = tmp_path_factory.mktemp("code")
    shutil.copy(b.LIB, at / "lib.so")
    subprocess.run([OBJDUMP, "--offloading", "lib.so"], cwd=at, check=True, stdout=subprocess.DEVNULL)
    parts = sorted(p for p in os.listdir(at) if p.endswith("gfx950"))
    assert len(parts) >= 10
    return [[line for line in subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", p], cwd=at, check=True, stdout=subprocess.PIPE, text=True).stdout.split("\n") if line.startswith("\t")]
            for p in parts]


def _wide_stores(lines):
    for line, after in zip(lines, lines[1:]):
        m = WIDE.match(line)
        if m:
            yield m[1], [t.strip() for t in m[2].split(",")], line, after


def test_wide_buffer_stores_have_a_constant_scalar_offset(code):
    found = [line for lines in code for kind, operands, line, _ in _wide_stores(lines) if kind == "buffer" and re.match(r"(s\d|m0|ttmp)", operands[3])]
    assert not found, f"{len(found)} stores, the first: {found[0]}"
    assert sum(kind == "buffer" for lines in code for kind, *_ in _wide_stores(lines)) > 100


def test_wide_stores_keep_their_data_one_instruction_long(code):
    total = 0
    for lines in code:
        for kind, operands, line, after in _wide_stores(lines):
            total += 1
            data, w = _registers(operands[0] if kind == "buffer" else operands[1]), WRITE.match(after)
            assert len(data) in (3, 4), line
            assert not (w and _registers(w[1]) & data), line + after
    assert total > 1000


def test_sources_pass_constants():
    """the same in the sources, the timing-only ones among them: the scalar offset of every 16-byte buffer store is a literal zero"""
    calls = 0
    for folder, _, names in os.walk(b.CSRC):
        for name in names:
            if name.endswith((".hip", ".h", ".inl")):
                for line in open(os.path.join(folder, name)):
                    for m in re.finditer(r"raw_buffer_store_b(?:96|128)\((.*?)\);", line):
                        calls += 1
                        assert m[1].rsplit(",", 2)[1].strip() == "0", f"{name}: {line.strip()}"
    assert calls >= 4
