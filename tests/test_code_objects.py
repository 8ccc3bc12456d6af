"""CPU tests of the built kernels' own metadata."""
import re
import struct

import msgpack

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
    spilled = {n: (k[".vgpr_spill_count"], k[".private_segment_fixed_size"]) for n, k in checked.items() if k[".vgpr_spill_count"] or k[".private_segment_fixed_size"]}
    assert not spilled, spilled
