"""Wait states before the LDS-DMA loads, in the machine code of the built library (CPU only).

The loads are written in asm blocks, where the compiler looks for no hazard, and
the hardware does not hold them back: a write of m0 has to stand one wait state
before the load, a VALU write of an SGPR that the load reads (a resource restored
from spilled lanes, for one) five.  An instruction counts one wait state, s_nop N
counts N + 1.
"""

import re
import shutil
import struct
import subprocess
from pathlib import Path

import pytest

from diffspec_mi355x import _build, _ext

M0_WAIT, SGPR_WAIT = 1, 5


def code_objects(blob):
    """The gfx950 code objects of a library's offload bundles."""
    magic, out, at = b"__CLANG_OFFLOAD_BUNDLE__", [], 0
    while (at := blob.find(magic, at)) >= 0:
        pos = at + len(magic)
        (n,) = struct.unpack_from("<Q", blob, pos)
        pos += 8
        for _ in range(n):
            off, size, k = struct.unpack_from("<QQQ", blob, pos)
            if _build.ARCH.encode() in blob[pos + 24:pos + 24 + k] and size:
                out.append(blob[at + off:at + off + size])
            pos += 24 + k
        at += len(magic)
    return out


def sgprs(operand):
    m = re.fullmatch(r"s(?:(\d+)|\[(\d+):(\d+)\])", operand)
    if not m:
        return set()
    return {int(m[1])} if m[1] else set(range(int(m[2]), int(m[3]) + 1))


def too_close(listing):
    """(DMA loads, those without their wait states) of a disassembly."""
    loads, bad, code = 0, [], []
    for line in listing.splitlines():
        text = line.split("//")[0].strip()
        if not text or text.endswith(":"):
            code = [] if text.endswith(">:") else code
            continue
        op, *args = text.replace(",", " ").split()
        if (op.startswith("global_load_lds") or op.startswith("buffer_load")) and ("lds" in op or "lds" in args):
            loads += 1
            need, waited, m0 = set().union(*map(sgprs, args)), 0, True
            for o, a in reversed(code):
                if waited >= SGPR_WAIT:
                    break
                dst = sgprs(a[0]) if a else set()
                if m0 and a and a[0] == "m0":
                    if waited < M0_WAIT:
                        bad.append((f"{o} {a}", text))
                    m0 = False
                if o.startswith("v_") and dst & need:
                    bad.append((f"{o} {a}", text))
                if o.startswith("s_") and not o.startswith(("s_cmp", "s_bitcmp")):
                    need -= dst
                waited += int(a[0], 0) + 1 if o == "s_nop" else 1
        code.append((op, args))
    return loads, bad


def test_the_scan_itself():
    load = "buffer_load_dwordx4 v1, s[4:7], 0 offen lds"
    for before, ok in [(["s_mov_b32 m0, s3"], False), (["s_mov_b32 m0, s3", "s_nop 0"], True),
                       (["v_readlane_b32 s7, v9, 1", "s_mov_b32 m0, s3", "s_nop 2"], False),
                       (["v_readlane_b32 s7, v9, 1", "s_mov_b32 m0, s3", "s_nop 3"], True),
                       (["v_readlane_b32 s7, v9, 1", "s_mov_b32 s7, s1", "s_mov_b32 m0, s3", "s_nop 0"], True),
                       (["v_readlane_b32 s8, v9, 1", "s_mov_b32 m0, s3", "s_nop 0"], True),
                       (["v_cmp_gt_i32_e64 s[6:7], v1, v2", "s_mov_b32 m0, s3", "s_nop 0"], False)]:
        loads, bad = too_close("\n".join([*before, load]))
        assert loads == 1 and (not bad) == ok, before


def test_dma_loads_have_their_wait_states(dsv_lib, tmp_path):
    tool = Path(_build._hipcc()).resolve().parent.parent / "llvm" / "bin" / "llvm-objdump"
    tool = str(tool) if tool.exists() else shutil.which("llvm-objdump")
    if tool is None:
        pytest.skip("no disassembler beside the compiler")
    total, wrong = 0, []
    objects = code_objects(_ext.lib_path().read_bytes())
    assert len(objects) >= len(_build.SOURCES) - 2  # (two sources hold host code alone)
    for i, obj in enumerate(objects):
        path = tmp_path / f"{i}.co"
        path.write_bytes(obj)
        res = subprocess.run([tool, "-d", "--no-show-raw-insn", str(path)], capture_output=True, text=True, timeout=120, check=True)
        n, bad = too_close(res.stdout)
        total += n
        wrong += bad
    assert total > 0
    assert not wrong, (len(wrong), total, wrong[:4])
