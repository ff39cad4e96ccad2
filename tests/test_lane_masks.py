"""The attention kernels' assembly: no register is copied where only some lanes are on and the others still need it.

While the sums of the matrix products are live, the compiler has placed copies of other values (an index, a thread's
number) at the top of the block where divided lanes come together, before the instruction that brings the other lanes
back: these kept garbage.  The kernels divide no lanes there, and this looks whether the compiler still agrees."""

from __future__ import annotations

import concurrent.futures as cf
import re
import subprocess

from dsv4_carve_amd import build

COPY = re.compile(r"v_mov_b(32|64)(_e32|_e64)? v\S+, v|v_accvgpr_(read|write|mov)|v_pk_mov_b32|scratch_load|scratch_store|v_swap")
LEAVES = ("s_cbranch", "s_branch", "s_endpgm", "s_and_saveexec", "s_andn2_saveexec", "s_barrier", "s_setpc", "s_swappc")


def early_copies(text):
    """(kernel, block, copies) of each block that copies registers before it brings the other lanes back."""
    found, kernel, block, before = [], "?", "?", None
    for line in text.splitlines():
        label = re.match(r"^(\.?[A-Za-z_]\w*):", line)
        if label:
            if line.startswith(".LBB"):
                block, before = label.group(1), []
            elif not line.startswith("."):
                kernel, block, before = label.group(1), "entry", []
            continue
        code = line.split(";")[0].strip()
        if not code or code.startswith(".") or before is None:
            continue
        if re.match(r"s_or_b64 exec, exec, ", code):
            copies = [c for c in before if COPY.match(c)]
            if copies:
                found.append((kernel, block, copies))
            before = None
        elif code.startswith(LEAVES) or re.match(r"s_\w+ exec\b", code):
            before = None
        else:
            before.append(code)
    return found


def test_finds_copies_before_the_lanes_are_back():
    block = "_Zkernel:\n\ts_and_saveexec_b64 s[0:1], vcc\n\tv_mov_b32_e32 v3, v9\n.LBB0_7:                 ; %join\n%s\ts_or_b64 exec, exec, s[0:1]\n\ts_endpgm\n"
    bad = ("\tv_accvgpr_write_b32 a3, v70\n", "\tv_mov_b32_e32 v1, v70\n", "\ts_nop 0\n\tv_mov_b64_e32 v[2:3], v[70:71]\n",
           "\tscratch_store_dword off, v70, off offset:4\n")
    good = ("", "\tv_mov_b32_e32 v1, 0\n\tglobal_store_dword v1, v2, s[6:7] offset:16\n", "\ts_mov_b32 s4, 0\n",
            "\ts_and_saveexec_b64 s[2:3], vcc\n\tv_mov_b32_e32 v1, v70\n")
    assert [len(early_copies(block.replace("%s", b))) for b in bad] == [1] * 4
    assert not any(early_copies(block.replace("%s", g)) for g in good)


def test_attention_kernels_copy_nothing_before_the_lanes_are_back(tmp_path):
    units = [u for u in build.UNITS if u[0] == "exl3_attn_inst.hip"]
    assert units

    def assemble(unit):
        src, defs, obj = unit
        out = tmp_path / f"{obj}.s"
        subprocess.run([build.HIPCC, *build.COMMON, *defs, "--cuda-device-only", "-S", f"{build.CSRC}/{src}", "-o", str(out)],
                       check=True, capture_output=True)
        return out.read_text()

    with cf.ThreadPoolExecutor(max_workers=4) as ex:
        texts = list(ex.map(assemble, units))
    for text in texts:
        assert "v_mfma" in text and "s_or_b64 exec, exec" in text
        assert early_copies(text) == []
        assert not re.search(r"ScratchSize: [1-9]", text)                       # spilled sums would be such copies too
