"""A wait that neither the hardware nor the compiler puts in front of hand-written memory instructions.

Memory instructions read scalar registers without asking whether a vector instruction (a readlane, say) has written them yet: five
wait states have to lie in between.  The compiler sees to that for its own instructions, but does not look into blocks of inline assembly,
as the copies into LDS are, while it may well keep their scalars in lanes of a vector register and read them back right in front
of such a block.  So the built library is looked through, all ways into each memory instruction."""
import re
import shutil
import subprocess
from pathlib import Path

import pytest

WAIT = 5


def _registers(text):
    out = set()
    for a, b, one in re.findall(r"\bs\[(\d+):(\d+)\]|\bs(\d+)\b", text):
        out |= set(range(int(a), int(b) + 1)) if a else {int(one)}
    return out


def _written(name, operands):
    """Scalar registers that a vector instruction writes: its result, and the carry behind it."""
    if not name.startswith("v_"):
        return set()
    n = 2 if "_co_" in name or name.startswith(("v_div_scale", "v_mad_u64", "v_mad_i64")) else 1
    return _registers(",".join(operands.split(",")[:n]))


def too_early(listing):
    """(kernel, vector instruction, memory instruction, wait states between) of all that are too close, in an assembly listing with
    addresses and branch targets as llvm-objdump writes it."""
    found, checked, kernel, code, at, into = [], 0, None, [], {}, {}

    def finish():
        nonlocal checked
        for k, (name, operands, _) in enumerate(code):
            if not name.startswith(("buffer_", "global_", "flat_", "scratch_")) or not (need := _registers(operands)):
                continue
            checked += 1
            ways, seen = [(k, 0)], set()
            while ways:
                here, waited = ways.pop()
                before = [j for j in into.get(code[here][2], ()) if j in at]
                before = [at[j] for j in before]
                if here and code[here - 1][0] not in ("s_branch", "s_endpgm", "s_setpc_b64"):
                    before.append(here - 1)
                for j in before:
                    if (j, waited) in seen:
                        continue
                    seen.add((j, waited))
                    n, ops, _ = code[j]
                    if _written(n, ops) & need:
                        found.append((kernel, f"{n} {ops}", f"{name} {operands}", waited))
                        continue
                    more = waited + (int(ops, 0) + 1 if n == "s_nop" else 1)
                    if more < WAIT:
                        ways.append((j, more))

    for line in listing.splitlines():
        if head := re.match(r"[0-9a-f]+ <(\S+)>:$", line):
            if kernel:
                finish()
            kernel, code, at, into = head[1], [], {}, {}
            start = int(line.split()[0], 16)
        elif kernel and (m := re.match(r"\t(\S+)\s*(.*?)\s*// ([0-9A-F]{12}):(.*)$", line)):
            address = int(m[3], 16)
            at[address] = len(code)
            code.append((m[1], m[2], address))
            if m[1].startswith(("s_branch", "s_cbranch")) and (target := re.search(r"\+0x([0-9a-f]+)>|>$", m[4])):
                into.setdefault(start + int(target[1] or "0", 16), []).append(address)
    if kernel:
        finish()
    return found, checked


def _listing(*lines):
    text = "0000000000001000 <kernel>:\n"
    for n, line in enumerate(lines):
        target = re.search(r"-> (\d+)", line)
        text += f"\t{line.split(' ->')[0]}  // {0x1000 + 4 * n:012X}: 00000000" + (f" <kernel+0x{4 * int(target[1]):x}>\n" if target else "\n")
    return text


COPY = "global_load_lds_dword v49, s[4:5]"


@pytest.mark.parametrize("lines,states", [
    (["v_readlane_b32 s5, v250, 4", "s_mov_b32 m0, s98", "s_nop 0", COPY], [2]),
    (["v_readlane_b32 s5, v250, 4", "s_mov_b32 m0, s98", "s_nop 3", COPY], []),
    (["v_readlane_b32 s5, v250, 4", "s_mov_b32 m0, s98", "s_nop 2", COPY], [4]),
    (["v_readlane_b32 s6, v250, 4", COPY], []),
    (["v_cmp_lt_f32_e64 s[4:5], v1, s7", COPY], [0]),
    (["v_add_co_u32_e64 v1, s[4:5], v2, v3", COPY], [0]),
    (["v_mov_b32_e32 v1, s4", COPY], []),
    # into the instruction from a loop's end, and not from what stands in front of it behind a jump
    (["s_nop 7", COPY, "v_readfirstlane_b32 s4, v1", "s_cbranch_scc1 65533 -> 1", "s_endpgm"], [1]),
    (["v_readfirstlane_b32 s4, v1", "s_branch 9 -> 3", COPY, "s_nop 7", "s_endpgm"], [])])
def test_search(lines, states):
    found, checked = too_early(_listing(*lines))
    assert checked == 1 and [f[3] for f in found] == states


def test_scalars_of_memory_instructions_have_arrived(tmp_path):
    from dsv3fp8 import _lib
    import build
    objdump = Path(build._hipcc()).resolve().parent.parent / "llvm" / "bin" / "llvm-objdump"
    if not objdump.exists():
        objdump = Path("/opt/rocm/llvm/bin/llvm-objdump")
    shutil.copy(_lib.LIB_PATH, tmp_path / "lib.so")                 # (the parts are written beside the library)
    subprocess.run([objdump, "--offloading", tmp_path / "lib.so"], check=True, capture_output=True)
    parts = sorted(tmp_path.glob("lib.so.*" + build.ARCH))
    assert len(parts) == len(build.sources())
    found, checked = [], 0
    for part in parts:
        text = subprocess.run([objdump, "-d", "--no-show-raw-insn", part], check=True, capture_output=True, text=True).stdout
        more, n = too_early(text)
        found += more
        checked += n
    assert checked > 1000
    assert not found, "\n".join(f"{k}: {v} | {w} states | {m}" for k, v, m, w in sorted(set(found)))
