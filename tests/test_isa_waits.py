"""Wait states that the machine code of the built library has to keep for itself (no GPU needed).

A vector store of more than 8 bytes reads its data registers after it has issued: two wait states have to
lie between it and a vector instruction that overwrites them. A memory instruction reads a scalar register that a
vector instruction wrote (a spilled one read back among them) only five wait states later. The compiler sees to
that for its own memory instructions, not for those written in inline assembly."""

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


MEMORY = re.compile(r"(?:global|flat|buffer|scratch)_")


def scalars(text):
    out = set()
    for a, b, one in re.findall(r"\bs(?:\[(\d+):(\d+)\]|(\d+)\b)", text):
        out |= set(range(int(a), int(b) + 1)) if a else {int(one)}
    return out | ({"vcc"} if re.search(r"\bvcc", text) else set())


def scalars_too_soon(lines):
    """(vector instruction, memory instruction) pairs: the scalar registers that one wrote, read fewer than five wait
    states later by the other."""
    bad, written = [], {}       # register -> (wait states gone by, instruction that wrote it)
    for line in lines:
        text = line.split("//")[0].strip()
        op, _, rest = text.partition(" ")
        dst, _, src = rest.partition(",")
        if MEMORY.match(op):
            bad += sorted({(written[r][1], text) for r in scalars(rest) & written.keys()})
        step = int(rest, 0) + 1 if op == "s_nop" else 1
        written = {r: (n + step, by) for r, (n, by) in written.items() if n + step < 5}
        if op.startswith("v_") and (op.startswith(("v_readlane", "v_readfirstlane", "v_cmp")) or "_co_" in op):
            # v_cmp's destination, or a carry's behind the sum
            for r in scalars(dst) | (scalars(src.partition(",")[0]) if "_co_" in op else set()):
                written[r] = (0, text)
        elif op.startswith("s_") and not op.startswith(("s_cmp", "s_nop", "s_waitcnt", "s_cbranch", "s_barrier")):
            for r in scalars(dst):
                written.pop(r, None)
    return bad


def test_the_listing_is_read_right():
    store, wait = "\tglobal_store_dwordx4 v[8:9], v[18:21], off sc0 sc1 // 0071: DE7D8000", "\ts_nop 1"
    near, other = "\tv_lshl_add_u64 v[18:19], v[8:9], 0, 64", "\tv_mov_b32_e32 v3, v18"
    assert len(overwritten([store, near])) == 1 and len(overwritten([store, other, near])) == 1
    assert not overwritten([store, wait, near]) and not overwritten([store, other, other, near])
    assert len(overwritten([store, "\ts_nop 0", near])) == 1
    assert not overwritten(["\tglobal_store_dwordx2 v[8:9], v[18:19], off", near])
    assert len(overwritten(["\tbuffer_store_dwordx4 v[2:5], v0, s[0:3], 0 offen", "\tv_add_f32_e32 v4, v1, v1"])) == 1


def test_scalars_of_a_listing():
    lane, load = "\tv_readlane_b32 s7, v205, 7 // D281", "\tglobal_load_lds_dwordx4 v12, s[6:7]"
    other, wait = "\ts_mov_b32 m0, s9", "\ts_nop 0"
    assert len(scalars_too_soon([lane, load])) == 1 and len(scalars_too_soon([lane, other, wait, load])) == 1
    assert not scalars_too_soon([lane, "\ts_nop 4", load]) and not scalars_too_soon([lane] + [other] * 5 + [load])
    assert len(scalars_too_soon([lane, "\ts_nop 3", load])) == 1
    # the register itself written anew by a scalar instruction; another one read
    assert not scalars_too_soon([lane, "\ts_mov_b64 s[6:7], s[4:5]", load])
    assert not scalars_too_soon([lane, "\tglobal_load_dwordx4 v[0:3], v12, s[8:9]"])
    assert len(scalars_too_soon(["\tv_readfirstlane_b32 s15, v2", "\tbuffer_load_dwordx4 v[2:5], v85, s[16:19], s15 offen"])) == 1
    assert len(scalars_too_soon(["\tv_cmp_gt_u32_e64 s[6:7], v1, v2", load])) == 1


@pytest.fixture(scope="module")
def listing(tmp_path_factory):
    """The library's vector code, a list of instructions per kernel file."""
    tmp_path = tmp_path_factory.mktemp("isa")
    objdump = shutil.which("llvm-objdump") or "/opt/rocm/llvm/bin/llvm-objdump"
    if not Path(objdump).exists():
        pytest.skip("no llvm-objdump")
    so = tmp_path / "lib.so"
    shutil.copy(PKG / "pico_hip" / "libpico_hip.so", so)
    subprocess.run([objdump, "--offloading", so.name], cwd=tmp_path, check=True, capture_output=True)
    parts, out = sorted(tmp_path.glob("lib.so.*gfx950")), []
    assert parts
    for part in parts:
        text = subprocess.run([objdump, "-d", "--no-show-raw-insn", part], check=True, capture_output=True, text=True).stdout
        out.append([x for x in text.splitlines() if x.startswith("\t")])
    return out


def test_wide_stores_keep_their_data(listing):
    bad = [b for lines in listing for b in overwritten(lines)]
    assert any(STORE.match(x) for lines in listing for x in lines) and not bad, bad[:5]


def test_memory_instructions_wait_for_their_scalars(listing):
    bad = [b for lines in listing for b in scalars_too_soon(lines)]
    assert not bad, (len(bad), bad[:5])
