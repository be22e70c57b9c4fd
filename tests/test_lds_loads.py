"""Loads from memory to LDS that are written as instructions of their own: the
compiler adds no wait states inside inline assembly, so the built kernels have to
hold those that the instruction set asks for.  CPU only: reads the library's own
device code."""

import re
import shutil
import struct
import subprocess

import pytest

MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"
ADDRESS_STATES = 5  # a VALU instruction writes an SGPR, a memory instruction reads it
M0_STATES = 1       # a scalar instruction writes m0, a load to LDS uses it


def device_code(library):
    """The gfx950 code objects of a host library's offload bundles."""
    data, at = library.read_bytes(), -1
    while (at := data.find(MAGIC, at + 1)) >= 0:
        count, = struct.unpack_from("<Q", data, at + len(MAGIC))
        place = at + len(MAGIC) + 8
        for _ in range(count):
            offset, size, name = struct.unpack_from("<QQQ", data, place)
            if size and data[place + 24:place + 24 + name].endswith(b"gfx950"):
                yield data[at + offset:at + offset + size]
            place += 24 + name


def registers(operand):
    """SGPRs that an operand names."""
    match = re.fullmatch(r"s\[(\d+):(\d+)\]|s(\d+)", operand)
    if not match:
        return set()
    low, high, one = match.groups()
    return {int(one)} if one else set(range(int(low), int(high) + 1))


def missing_waits(lines):
    """(loads to LDS, those that come too soon, with the instruction they follow) of a disassembly."""
    code = []
    for line in lines:
        match = re.match(r"\s+([a-z_0-9]+)(?:\s+([^/]*?))?\s*(?://.*)?$", line)
        code.append((match[1], [o.strip() for o in (match[2] or "").split(",")]) if match else ("", []))
    loads, found = 0, []
    for i, (name, operands) in enumerate(code):
        if not re.search(r"_lds_|_load_.*lds", name) and operands[-1:] != ["lds"]:
            continue
        loads += 1
        read = set().union(*(registers(o.split(" ")[0]) for o in operands))
        states, j = 0, i - 1
        while j >= 0 and states < ADDRESS_STATES and code[j][0]:
            before, written = code[j]
            if before.startswith("s_") and written[:1] == ["m0"] and states < M0_STATES:
                found.append((code[j], code[i]))
            if before.startswith("v_"):
                results = written[:2] if "_co_" in before or "div_scale" in before else written[:1]
                if read & set().union(*map(registers, results)):
                    found.append((code[j], code[i]))
            elif before.startswith("s_"):
                read = read - registers(written[0])  # (what a scalar instruction wrote needs no wait)
            states += int(written[0], 0) + 1 if before == "s_nop" else 1
            j -= 1
    return loads, found


def test_missing_waits_are_seen():
    load = ["\ts_mov_b32 m0, s4", "\tglobal_load_lds_dwordx4 v1, s[8:9]  // 000: 1"]
    assert missing_waits(load)[1] and missing_waits([load[0], "\ts_nop 0", load[1]]) == (1, [])
    lane = "\tv_readlane_b32 s9, v2, s3"
    assert missing_waits([lane, "\ts_nop 3", load[1]])[1] and missing_waits([lane, "\ts_nop 4", load[1]]) == (1, [])
    assert missing_waits(["\tv_cmp_gt_i32 s[8:9], v2, v3", load[1]])[1]
    assert missing_waits([lane.replace("s9", "s7"), "\ts_mov_b64 s[8:9], s[6:7]", load[1]]) == (1, [])


def test_loads_to_lds_wait_for_their_address_and_place():
    from drama3_amd import _lib

    objdump = shutil.which("llvm-objdump", path="/opt/rocm/llvm/bin")
    if objdump is None or not _lib.LIBRARY.exists():
        pytest.skip("library not built, or no disassembler")
    loads, found = 0, []
    for code in device_code(_lib.LIBRARY):
        if b"paged_tile_kernel" not in code:
            continue
        text = subprocess.run([objdump, "-d", "-"], input=code, capture_output=True, check=True).stdout.decode()
        count, bad = missing_waits(text.splitlines())
        loads, found = loads + count, found + bad
    assert loads > 0 and not found, f"{len(found)} of {loads}: {found[:3]}"
