"""Build-time check of the AMD assembly built here with hipcc: the wait states that the
direct-to-LDS loads in inline assembly need, which the compiler does not insert there.
In every path to such a load one wait state at least lies between the write of M0 and
it, and five between a VALU instruction's write of one of its SGPRs (address, buffer
resource) and it."""
import os
import re
import subprocess

import pytest

from test_prefill_m0 import HIPCC, LDS_DMA, ROOT

SGPR_WAITS, M0_WAITS = 5, 1


def _program(asm):
    """(instructions, label -> index of the next instruction); a word that is s_nop's
    counts as one."""
    ins, labels = [], {}
    for line in asm.splitlines():
        code = line.split(";", 1)[0].strip()
        label = re.match(r"^([\w.$]+):$", code)
        word = re.match(r"^\.long\s+0xbf8000([0-9a-f]{2})$", code)
        if label:
            labels[label.group(1)] = len(ins)
        elif word:
            ins.append(f"s_nop {int(word.group(1), 16)}")
        elif code and not code.startswith("."):
            ins.append(code)
    return ins, labels


def _sgprs(operand):
    got = set()
    for a, b, c in re.findall(r"\bs\[(\d+):(\d+)\]|\bs(\d+)\b", operand):
        got |= {int(c)} if c else set(range(int(a), int(b) + 1))
    return got


def _valu_writes(code):
    if not code.startswith("v_"):
        return set()
    name, _, rest = code.partition(" ")
    ops = [o.strip() for o in rest.split(",")]
    got = _sgprs(ops[0])
    if re.search(r"_co_|div_scale|mad_[ui]64", name) and len(ops) > 1:
        got |= _sgprs(ops[1])
    return got


def _too_early(ins, labels, needed, is_write):
    """(writer, load) pairs with fewer than ``needed`` wait states between them on some
    path; is_write(load, instruction)."""
    into = {}
    for i, code in enumerate(ins):
        if re.match(r"^s_(c)?branch", code):
            into.setdefault(labels[code.split()[1]], []).append(i)
    bad = []
    for i, load in enumerate(ins):
        if not LDS_DMA.match(load):
            continue
        todo, seen = [(i, 0)], set()
        while todo:
            at, waits = todo.pop()
            before = list(into.get(at, ()))
            if at > 0 and not re.match(r"^s_(branch|endpgm|setpc)", ins[at - 1]):
                before.append(at - 1)
            for j in before:
                if is_write(load, ins[j]):
                    bad.append((ins[j], waits, load))
                    continue
                nop = re.match(r"^s_nop (\d+)$", ins[j])
                w = waits + (int(nop.group(1)) + 1 if nop else 1)
                if w < needed and (j, w) not in seen:
                    seen.add((j, w))
                    todo.append((j, w))
    return bad


def _sgpr_write(load, code):
    return bool(_valu_writes(code) & _sgprs(load))


def _m0_write(load, code):
    return code.startswith("s_") and re.search(r"^\S+ m0\b", code) is not None


def test_the_check_itself():
    """On listings with and without the waits, a branch among the paths."""
    head, load = "v_readfirstlane_b32 s6, v1\n", "buffer_load_dwordx4 v2, s[4:7], 0 offen lds\n"
    for text, sgpr, m0 in (
            (head + "s_mov_b32 m0, s9\n" + load, True, True),
            (head + "s_mov_b32 m0, s9\n.long 0xbf800000\n" + load, True, False),
            (head + "s_nop 2\ns_mov_b32 m0, s9\n.long 0xbf800000\n" + load, False, False),
            (head + "s_nop 2\ns_mov_b32 m0, s9\ns_nop 0\n" + load, False, False),
            (head + "s_branch .L1\ns_nop 7\n.L1:\ns_mov_b32 m0, s9\ns_nop 0\n" + load, True, False),
            ("v_mad_u64_u32 v[0:1], s[6:7], v2, v3, v[4:5]\ns_nop 0\n" + load, True, False),
            ("v_mov_b32 v6, s6\n" + load, False, False)):
        ins, labels = _program(text)
        assert bool(_too_early(ins, labels, SGPR_WAITS, _sgpr_write)) == sgpr, text
        assert bool(_too_early(ins, labels, M0_WAITS, _m0_write)) == m0, text


@pytest.mark.skipif(not os.access(HIPCC, os.X_OK), reason="hipcc not available")
@pytest.mark.parametrize("source", ["prompt", "weights", "prefill"])
def test_direct_lds_loads_wait_for_their_scalars(tmp_path, source):
    out = tmp_path / (source + ".s")
    subprocess.run([HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", "-Xclang",
                    "-target-feature", "-Xclang", "-packed-fp32-ops",
                    "-I" + os.path.join(ROOT, "include"),
                    "-I" + os.path.join(ROOT, "gpu_offloading_amd", "csrc"),
                    "--cuda-device-only", "-S",
                    os.path.join(ROOT, "gpu_offloading_amd", "csrc", source + ".hip"),
                    "-o", str(out)], check=True, capture_output=True)
    ins, labels = _program(out.read_text())
    assert any(LDS_DMA.match(code) for code in ins)
    assert _too_early(ins, labels, SGPR_WAITS, _sgpr_write) == []
    assert _too_early(ins, labels, M0_WAITS, _m0_write) == []
