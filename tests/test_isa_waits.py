"""The waits that gfx9 leaves to software, in the built library's own code.

The compiler places them between its instructions, but does not look inside inline assembly, so a
statement there has to bring its own. Of the hazards that the CDNA3/CDNA4 instruction set documents
(manually inserted wait states), those that this library's assembly can meet:

- an SGPR written by a VALU instruction (v_readlane, v_readfirstlane, a compare) and read by a
  vector memory instruction as its base or resource: 5 wait states
- M0 written by a scalar instruction and read by a load into LDS: 1
- an SGPR written by a VALU instruction and read by another: 2

An instruction is a wait state, ``s_nop n`` is n + 1. Every kernel of the library is read, in order."""

import re
import shutil
import subprocess
from pathlib import Path

import pytest

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"
VMEM = ("buffer_", "global_", "flat_", "scratch_")
SREG = re.compile(r"\bs(?:(\d+)\b|\[(\d+):(\d+)\])")


def _sregs(text):
    out = {"vcc"} if re.search(r"\bvcc\b", text) else set()
    for one, lo, hi in SREG.findall(text):
        out |= set(range(int(one), int(one) + 1)) if one else set(range(int(lo), int(hi) + 1))
    return out


def _parts(line):
    """(mnemonic, operands, SGPRs that a VALU instruction writes, SGPRs it reads)"""
    op, _, rest = line.partition(" ")
    args = [a.strip() for a in rest.split(",")]
    if not op.startswith("v_"):
        return op, args, set(), _sregs(rest)
    written = _sregs(args[0])
    first = 1
    if re.match(r"v_(add|sub|subrev|addc|subb|subbrev)_co_|v_div_scale|v_mad_[ui]64", op):
        written |= _sregs(args[1])
        first = 2
    return op, args, written, _sregs(",".join(args[first:]))


def hazards(lines):
    """Of (function, instruction) pairs in order: those that read too early, with the reason."""
    found = []
    past = []  # (wait states since, what it wrote): the last few instructions
    for fn, line in lines:
        op, args, written, read = _parts(line)
        lds = op.startswith(VMEM) and ("_lds_" in op or line.endswith(" lds"))
        for since, kind, regs in past:
            if op.startswith(VMEM) and kind == "valu" and since < 5 and regs & read:
                found.append((fn, line, f"SGPR written by VALU {since} wait states before a vector memory read of it"))
            if lds and kind == "salu" and since < 1 and "m0" in regs:
                found.append((fn, line, "M0 written right before a load into LDS reads it"))
            if op.startswith("v_") and kind == "valu" and since < 2 and regs & read:
                found.append((fn, line, f"SGPR written by VALU {since} wait states before a VALU read of it"))
        states = int(args[0], 0) + 1 if op == "s_nop" else 1
        past = [(n + states, k, r) for n, k, r in past if n + states < 5]
        if written:
            past.append((0, "valu", written))
        if op.startswith("s_") and args[0] == "m0":
            past.append((0, "salu", {"m0"}))
    return found


def instructions(path, tmp):
    """(function, instruction) of every gfx950 code object of the library ``path``."""
    lib = shutil.copy(path, tmp / path.name)
    subprocess.run([OBJDUMP, "--offloading", lib], check=True, capture_output=True)
    out = []
    for obj in sorted(tmp.glob("*gfx950")):
        text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", "--no-leading-addr", str(obj)], check=True,
                              capture_output=True, text=True).stdout  # fmt: skip
        fn = None
        for raw in text.splitlines():
            if raw.endswith(">:"):
                fn = raw.strip("<>:")
            elif raw.startswith("\t"):
                out.append((fn, " ".join(raw.split("//")[0].split())))
    return out


def _on(*text):
    return [why for _, _, why in hazards([("k", t) for t in text])]


def test_the_reading_finds_what_it_should():
    lane = "v_readlane_b32 s3, v1, 4"
    dma = "global_load_lds_dwordx4 v2, s[2:3]"
    assert len(_on(lane, "s_mov_b32 m0, s7", dma)) == 2
    assert len(_on(lane, "s_mov_b32 m0, s7", "s_nop 0", dma)) == 1
    assert len(_on(lane, "s_mov_b32 m0, s7", "s_nop 2", dma)) == 1
    assert not _on(lane, "s_mov_b32 m0, s7", "s_nop 3", dma)
    assert not _on("v_readlane_b32 s4, v1, 4", "s_mov_b32 m0, s7", "s_nop 0", dma)
    assert _on("s_mov_b32 m0, s7", "buffer_load_dwordx4 v1, s[4:7], 0 offen lds")
    assert not _on("s_mov_b32 m0, s7", "buffer_load_dwordx4 v[1:4], v0, s[4:7], 0 offen")
    assert _on("v_cmp_lt_u32_e64 s[4:5], v0, v1", "buffer_load_dword v1, v0, s[4:7], 0 offen")
    assert _on("v_readfirstlane_b32 s4, v0", "v_writelane_b32 v1, s4, 3")
    assert not _on("v_readfirstlane_b32 s4, v0", "s_nop 1", "v_writelane_b32 v1, s4, 3")
    assert not _on("v_readfirstlane_b32 s4, v0", "s_mov_b32 s5, s4")


# the hazards that each part of the library is read for
CHECKED = [("mkmoe_latent", "vector memory"), ("mkmoe_latent", "M0"), ("others", "M0"),
           ("others", "vector memory"), ("mkmoe_latent", "VALU read"), ("others", "VALU read")]  # fmt: skip


@pytest.fixture(scope="module")
def found(tmp_path_factory):
    """The library's instructions, and their hazards: [(kernel, instruction, reason)]."""
    from sgl_amd_mono.moe import _lib

    if not Path(OBJDUMP).exists():
        pytest.skip(f"no {OBJDUMP}")
    lines = instructions(Path(_lib.LIB_PATH), tmp_path_factory.mktemp("isa"))
    for part in (True, False):  # the loads into LDS are there
        assert sum(("mkmoe_latent" in fn) == part and ("_lds_" in t or t.endswith(" lds")) for fn, t in lines) > 100
    return lines, hazards(lines)


@pytest.mark.parametrize("kernels,what", CHECKED)
def test_no_instruction_reads_too_early(found, kernels, what):
    bad = [x for x in found[1] if ("mkmoe_latent" in x[0]) == (kernels == "mkmoe_latent") and what in x[2]]
    assert not bad, (len(bad), bad[:3])


def test_m0_serves_the_loads_into_lds_alone(found):
    """The latent attention's loads into LDS write M0 in their own statements. The compiler is told, but
    counts M0 among its own registers: its code there has no use for it, so that nothing of it is lost."""
    latent = [(fn, t) for fn, t in found[0] if "mkmoe_latent" in fn]
    unnamed = re.compile(r"s_movrel|s_sendmsg|v_interp|s_set_gpr_idx|ds_\w*(addtid|gws)")  # (they read it unnamed)
    assert not [x for x in latent if unnamed.match(x[1])]
    uses = [(i, t) for i, (_, t) in enumerate(latent) if re.search(r"\bm0\b", t)]
    for i, t in uses:  # written, waited for or the address formed, read by a load
        assert re.match(r"s_mov_b32 m0, s\d+$|s_add_u32 m0, m0, 0x[0-9a-f]+$", t), t
        after = [u.split(" ")[0] for _, u in latent[i + 1 : i + 4]]
        load = next(k for k, u in enumerate(after) if "_lds_" in u)
        assert set(after[:load]) <= {"s_nop", "v_add_u32_e32"} and load > 0, (t, after)
    assert len(uses) == sum("_lds_" in t for _, t in latent)
