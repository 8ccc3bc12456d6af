"""CPU tests of the built kernels' own metadata."""
import os
import re
import struct
import subprocess

import msgpack
import pytest

from mamtorch_amd import _native

#: Kernels that may keep no registers in memory: a register that was spilled inside a branch of lanes came back for those lanes alone.
WITHOUT_SPILLS = re.compile("rotary|5pages|page_tiles_kernel|pages_kernel")


def _code_objects(data):
    """The ELF images of the offload bundles in a shared library."""
    magic, at = b"__CLANG_OFFLOAD_BUNDLE__", 0
    while (at := data.find(magic, at)) >= 0:
        count, = struct.unpack_from("<Q", data, at + len(magic))
        entry = at + len(magic) + 8
        for _ in range(count):
            offset, size, length = struct.unpack_from("<QQQ", data, entry)
            name = data[entry + 24:entry + 24 + length]
            entry += 24 + length
            if b"gfx950" in name and size:
                yield data[at + offset:at + offset + size]
        at += len(magic)


def _kernels(elf):
    """The kernels' metadata: the note of type 32 that the compiler writes, as msgpack."""
    shoff, = struct.unpack_from("<Q", elf, 0x28)
    shentsize, shnum = struct.unpack_from("<HH", elf, 0x3a)
    for i in range(shnum):
        head = shoff + i * shentsize
        kind, = struct.unpack_from("<I", elf, head + 4)
        offset, size = struct.unpack_from("<QQ", elf, head + 0x18)
        at = offset
        while kind == 7 and at < offset + size:         # SHT_NOTE
            names, descs, note = struct.unpack_from("<III", elf, at)
            desc = at + 12 + (names + 3) // 4 * 4
            if note == 32 and elf[at + 12:at + 12 + names].startswith(b"AMDGPU"):
                yield from msgpack.unpackb(elf[desc:desc + descs], strict_map_key=False).get("amdhsa.kernels", [])
            at = desc + (descs + 3) // 4 * 4


def test_kernels_that_branch_by_lanes_keep_no_registers_in_memory():
    with open(_native.HIP_LIB_PATH, "rb") as f:
        kernels = {k[".name"]: k for elf in _code_objects(f.read()) for k in _kernels(elf)}
    checked = {n: k for n, k in kernels.items() if WITHOUT_SPILLS.search(n)}
    assert len(kernels) > 200 and len(checked) > 60, (len(kernels), len(checked))
    # (scalar registers go to lanes of a vector register, with a slot of the stack that nothing uses)
    spilled = {n: (k[".vgpr_spill_count"], k[".private_segment_fixed_size"]) for n, k in checked.items()
               if k[".vgpr_spill_count"] or (k[".private_segment_fixed_size"] and not k[".sgpr_spill_count"])}
    assert not spilled, spilled


OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"


def _written_too_early(text):
    """Vector instructions that stand where a branch of lanes ends, before its other lanes are back: those lanes keep what was in the register."""
    found = []
    for kernel in re.split(r"^[0-9a-f]+ <(?=\S+>:$)", text, flags=re.M)[1:]:
        name, lines = kernel[:kernel.index(">")], [m.groups() for m in re.finditer(r"^\t(\S+)(.*?)// ([0-9A-F]+):(.*)$", kernel, flags=re.M)]
        if not WITHOUT_SPILLS.search(name) or not lines:
            continue
        start = int(lines[0][2], 16)
        takes = ["saveexec" in op or operands.strip().startswith("exec") for op, operands, _, _ in lines]
        ends = {start + int(re.search(r"<[^+>]+(?:\+0x([0-9a-f]+))?>", target).group(1) or "0", 16)
                for i, (op, _, _, target) in enumerate(lines) if op == "s_cbranch_execz" and any(takes[max(i - 4, 0):i])}
        at = {int(address, 16): i for i, (_, _, address, _) in enumerate(lines)}
        for end in ends:
            early = []
            for op, operands, _, _ in lines[at[end]:at[end] + 60]:
                if op in ("s_or_b64", "s_mov_b64") and operands.strip().startswith("exec"):
                    found += [(name, hex(end), e) for e in early]
                    break
                if re.match(r"s_(cbranch|branch|endpgm|setpc)|s_\w+_saveexec", op) or (op.startswith("s_") and operands.strip().startswith("exec")):
                    break
                if re.match(r"(v_(?!writelane|readlane|readfirstlane)|scratch_|ds_|global_|buffer_|flat_)", op):
                    early.append(op + operands.rstrip())
    return found


def test_the_check_of_branches_finds_a_copy_before_the_lanes_are_back():
    text = """0000000000001000 <page_tiles_kernel>:
\ts_and_saveexec_b64 s[2:3], vcc                               // 000000001000: BE82206A
\ts_cbranch_execz 1                                            // 000000001004: BF880001 <page_tiles_kernel+0xc>
\tv_mov_b32_e32 v1, 0                                          // 000000001008: 7E020280
%s\ts_or_b64 exec, exec, s[2:3]                                  // 000000001010: 87FE027E
"""
    copy = "\tv_accvgpr_write_b32 a128, v14                                // 00000000100C: D3D94080 1800010E\n"
    assert [f[2].split()[0] for f in _written_too_early(text % copy)] == ["v_accvgpr_write_b32"]
    assert not _written_too_early(text % "\ts_nop 1                                                    // 00000000100C: BF800001\n")


@pytest.mark.skipif(not os.path.exists(OBJDUMP), reason="no disassembler")
def test_kernels_write_no_register_before_a_branch_has_its_lanes_back(tmp_path):
    with open(_native.HIP_LIB_PATH, "rb") as f:
        objects = [elf for elf in _code_objects(f.read()) if any(WITHOUT_SPILLS.search(k[".name"]) for k in _kernels(elf))]
    assert len(objects) >= 3
    for i, elf in enumerate(objects):
        path = tmp_path / f"{i}.elf"
        path.write_bytes(elf)
        text = subprocess.run([OBJDUMP, "-d", str(path)], capture_output=True, text=True, check=True).stdout
        assert "s_cbranch_execz" in text
        assert not (found := _written_too_early(text)), found[:8]
