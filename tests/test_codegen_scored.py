"""CPU: the built attention objects keep what their inline-asm transposed reads count on.

`ds_read_b64_tr_b16` is inline asm that the compiler takes as finished at once; the code waits for it later. So between a
read and its wait nothing may touch its registers, and no vector register may be spilled (a spill would store the
unfinished value)."""
from __future__ import annotations

import re
import shutil
import subprocess

import pytest

from tests.test_codegen import LLVM, OBJ_DIR, _disassemble

OBJECTS = ("attn_kernels", "attn_scored_64", "attn_scored_96", "attn_scored_128")


def _regs(text: str) -> set[int]:
    out: set[int] = set()
    for m in re.finditer(r"\bv\[(\d+):(\d+)\]|\bv(\d+)\b", text):
        out |= {int(m.group(3))} if m.group(3) else set(range(int(m.group(1)), int(m.group(2)) + 1))
    return out


def touched_in_flight(lines: list[str]) -> tuple[int, list[str]]:
    """(transposed reads, instructions that touch the registers of one before its wait), in the listing's order; LDS
    operations return in order, and lgkmcnt counts those outstanding."""
    reads, hits, queue = 0, [], []
    for ln in lines:
        if ln.endswith(">:"):
            queue = []
        wait = re.search(r"lgkmcnt\((\d+)\)", ln) if ln.startswith("s_waitcnt") else None
        if wait:
            queue = queue[max(0, len(queue) - int(wait.group(1))):]
            continue
        flying = set().union(*queue)
        if ln.startswith("ds_read_b64_tr"):
            mine = _regs(ln.split(",")[0])
            reads += 1
            hits += [ln] if mine & flying else []
            queue.append(mine)
            continue
        hits += [ln] if _regs(ln) & flying else []
        if ln.startswith("ds_"):
            queue.append(set())
    return reads, hits


def test_the_check_finds_a_touch():
    read, use = "ds_read_b64_tr_b16 v[4:5], v9", "v_add_f32 v4, v1, v2"
    assert touched_in_flight([read, use]) == (1, [use])
    assert touched_in_flight([read, "s_waitcnt lgkmcnt(0)", use]) == (1, [])
    assert touched_in_flight([read, "ds_write_b32 v1, v2", "s_waitcnt lgkmcnt(1)", use]) == (1, [])
    assert touched_in_flight([read, "ds_write_b32 v1, v2", "s_waitcnt lgkmcnt(2)", use]) == (1, [use])


@pytest.mark.parametrize("name", OBJECTS)
def test_transposed_reads_in_flight(name, tmp_path):
    obj = OBJ_DIR / f"{name}.o"
    if not obj.exists() or not (LLVM / "llvm-objdump").exists() or shutil.which(str(LLVM / "clang-offload-bundler")) is None:
        pytest.skip("built objects or the ROCm LLVM tools are not here (run build() first)")
    reads, hits = touched_in_flight(_disassemble(obj, tmp_path))
    assert reads > 0 and not hits, hits[:5]
    notes = subprocess.run([str(LLVM / "llvm-readelf"), "--notes", str(tmp_path / f"{name}.co")], check=True,
                           capture_output=True, text=True).stdout
    spills = re.findall(r"\.vgpr_spill_count:\s+(\d+)", notes)
    assert spills and set(spills) == {"0"}, spills
