"""What the compiler says of the kernels in the built library (the metadata of its code objects): none keeps its state in memory.  A
few spilled registers are a choice; a function that was not inlined, whose arguments and arrays all go through memory, is not."""
import struct

import msgpack

from flash_attention_factory_amd import _build, _cabi

MOST_SCRATCH = 512  # bytes per lane: a kernel of 256 registers that spills a third of its state; one call takes over 1000


def _code_objects(path):
    data = open(path, "rb").read()
    at = data.find(b"__CLANG_OFFLOAD_BUNDLE__")
    while at >= 0:
        count, = struct.unpack_from("<Q", data, at + 24)
        entry = at + 32
        for _ in range(count):
            offset, size, name_len = struct.unpack_from("<QQQ", data, entry)
            name = data[entry + 24:entry + 24 + name_len].decode()
            entry += 24 + name_len
            if "gfx950" in name and size:
                yield data[at + offset:at + offset + size]
        at = data.find(b"__CLANG_OFFLOAD_BUNDLE__", at + 24)


def _kernels(elf):
    assert elf[:5] == b"\x7fELF\x02"
    sections, = struct.unpack_from("<Q", elf, 40)
    size, count = struct.unpack_from("<HH", elf, 58)
    for k in range(count):
        head = sections + k * size
        kind, = struct.unpack_from("<I", elf, head + 4)
        offset, length = struct.unpack_from("<QQ", elf, head + 24)
        if kind != 7:  # notes
            continue
        at = offset
        while at < offset + length:
            name_len, desc_len, note = struct.unpack_from("<III", elf, at)
            desc = at + 12 + (name_len + 3) // 4 * 4
            if note == 32:  # the metadata of AMD GPU code objects
                yield from msgpack.unpackb(elf[desc:desc + desc_len], strict_map_key=False)["amdhsa.kernels"]
            at = desc + (desc_len + 3) // 4 * 4


def test_no_kernel_keeps_its_state_in_memory():
    _cabi.load()
    found = [kernel for elf in _code_objects(_build.LIBRARY) for kernel in _kernels(elf)]
    assert len(found) > 200 and any("ragged_tile_kernel" in kernel[".name"] for kernel in found)
    large = {kernel[".name"]: kernel[".private_segment_fixed_size"] for kernel in found
             if kernel[".private_segment_fixed_size"] > MOST_SCRATCH or kernel.get(".uses_dynamic_stack")}
    assert not large, large
