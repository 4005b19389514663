"""Wait states that the machine code of the built library has to keep for itself (no GPU needed).

A vector store of more than 8 bytes reads its data registers after it has issued: two wait states have to
lie between it and a vector instruction that overwrites them. The compiler sees to that for its own
stores, not for those written in inline assembly."""

import re
import shutil
import subprocess
from pathlib import Path

import pytest

from conftest import PKG

STORE = re.compile(r"^\s*(?:global|flat)_store_dwordx[34] \S+ (?P<g>v\[\d+:\d+\])|^\s*buffer_store_dwordx[34] (?P<b>v\[\d+:\d+\])")


def registers(text):
    out = set()
    for a, b, one in re.findall(r"\bv(?:\[(\d+):(\d+)\]|(\d+)\b)", text):
        out |= set(range(int(a), int(b) + 1)) if a else {int(one)}
    return out


def overwritten(lines):
    """(store, instruction) pairs of an assembly listing that lie fewer than two wait states apart."""
    bad = []
    for i, line in enumerate(lines):
        m = STORE.match(line)
        if not m:
            continue
        data, waits = registers(m.group("g") or m.group("b")), 0
        for after in lines[i + 1:i + 3]:
            op, _, rest = after.split("//")[0].strip().partition(" ")
            # v_cmp and the like write no vector register; a swap writes both of its operands
            dst = rest if "swap" in op else rest.split(",")[0]
            if waits < 2 and op.startswith("v_") and registers(dst) & data:
                bad.append((line.split("//")[0].strip(), after.split("//")[0].strip()))
            waits += int(rest, 0) + 1 if op == "s_nop" else 1
    return bad


def test_the_listing_is_read_right():
    store, wait = "\tglobal_store_dwordx4 v[8:9], v[18:21], off sc0 sc1 // 0071: DE7D8000", "\ts_nop 1"
    near, other = "\tv_lshl_add_u64 v[18:19], v[8:9], 0, 64", "\tv_mov_b32_e32 v3, v18"
    assert len(overwritten([store, near])) == 1 and len(overwritten([store, other, near])) == 1
    assert not overwritten([store, wait, near]) and not overwritten([store, other, other, near])
    assert len(overwritten([store, "\ts_nop 0", near])) == 1
    assert not overwritten(["\tglobal_store_dwordx2 v[8:9], v[18:19], off", near])
    assert len(overwritten(["\tbuffer_store_dwordx4 v[2:5], v0, s[0:3], 0 offen", "\tv_add_f32_e32 v4, v1, v1"])) == 1


def test_wide_stores_keep_their_data(tmp_path):
    objdump = shutil.which("llvm-objdump") or "/opt/rocm/llvm/bin/llvm-objdump"
    if not Path(objdump).exists():
        pytest.skip("no llvm-objdump")
    so = tmp_path / "lib.so"
    shutil.copy(PKG / "pico_hip" / "libpico_hip.so", so)
    subprocess.run([objdump, "--offloading", so.name], cwd=tmp_path, check=True, capture_output=True)
    parts, stores, bad = sorted(tmp_path.glob("lib.so.*gfx950")), 0, []
    assert parts
    for part in parts:
        text = subprocess.run([objdump, "-d", "--no-show-raw-insn", part], check=True, capture_output=True, text=True).stdout
        lines = [x for x in text.splitlines() if x.startswith("\t")]
        stores += sum(1 for x in lines if STORE.match(x))
        bad += overwritten(lines)
    assert stores > 0 and not bad, bad[:5]
