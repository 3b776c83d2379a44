"""CPU: rules that the built gfx950 code keeps.

Wide stores.  The memory unit fetches the data of a store of more than 8 bytes after the instruction was issued; a vector instruction right
behind it that writes the same registers comes too early.  hipcc keeps the distance, except behind a buffer store whose scalar offset is a register, where gfx950 stores
the new value in some lanes all the same (seen: 160 of 6 million outputs of a product, in every call).

Rings in LDS.  Loads that go straight to LDS are ordered behind another wave's reads by barriers alone: between the fragments that a kernel reads in front of its loop and the
loop's first load into the same ring there has to be one.  (Without: a wave held up for a microsecond multiplied rows of a later tile, in one training step of 70.)"""
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
    """the built library's gfx950 code, one list of lines per source"""
    if not os.path.exists(b.LIB):
        b.build_library(verbose=False)
    at = tmp_path_factory.mktemp("code")
    shutil.copy(b.LIB, at / "lib.so")
    subprocess.run([OBJDUMP, "--offloading", "lib.so"], cwd=at, check=True, stdout=subprocess.DEVNULL)
    parts = sorted(p for p in os.listdir(at) if p.endswith("gfx950"))
    assert len(parts) >= 10
    return [subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", p], cwd=at, check=True, stdout=subprocess.PIPE, text=True).stdout.split("\n") for p in parts]


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


def test_prologue_reads_are_closed_by_a_barrier(code):
    seen = 0
    for lines in code:
        for at, line in enumerate(lines):
            if not re.match(r"[0-9a-f]+ <.*(gemm_fast8p_kernel|gemm_tn8r_kernel).*>:", line):
                continue
            body = lines[at + 1:next((n for n in range(at + 1, len(lines)) if re.match(r"[0-9a-f]+ <", lines[n])), len(lines))]
            kinds = []
            for text in body:
                if re.match(r"\s+s_barrier", text):
                    kinds.append("barrier")
                elif re.match(r"\s+ds_read", text):
                    kinds.append("read")
                elif re.match(r"\s+(buffer|global)_load_\S+ .*\blds\b|\s+global_load_lds", text):
                    kinds.append("load")
            first = kinds.index("barrier")                                    # the prologue's loads have landed
            assert "load" in kinds[:first] and kinds[first + 1] == "read", line
            after = kinds[first + 1:]
            assert after[after.index("read"):after.index("load")].count("barrier") >= 2, line      # (one of them is the second wave group's alone)
            seen += 1
    assert seen >= 12, seen


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
