"""What the compiler made of the cache operators' kernels (no GPU): read from the metadata of the built library."""
import struct

import pytest


def gfx950_kernels():
    """``{kernel symbol: metadata}`` of the gfx950 code objects inside ``libolmo355.so``."""
    msgpack = pytest.importorskip("msgpack")
    from olmo_amd import _lib, build

    _lib.lib()
    blob, magic, kernels, at = open(build.LIB, "rb").read(), b"__CLANG_OFFLOAD_BUNDLE__", {}, 0
    while (at := blob.find(magic, at)) >= 0:
        pos, (count,) = at + 32, struct.unpack_from("<Q", blob, at + 24)
        if count > 16:  # the words alone, not a bundle
            at += 1
            continue
        for _ in range(count):
            offset, size, name = struct.unpack_from("<QQQ", blob, pos)
            if b"gfx950" in blob[pos + 24:pos + 24 + name]:
                kernels.update(_notes(blob[at + offset:at + offset + size], msgpack))
            pos += 24 + name
        at += 1
    return kernels


def _notes(elf, msgpack):
    assert elf[:4] == b"\x7fELF"
    shoff, = struct.unpack_from("<Q", elf, 40)
    shentsize, shnum = struct.unpack_from("<HH", elf, 58)
    for i in range(shnum):
        kind, = struct.unpack_from("<I", elf, shoff + i * shentsize + 4)
        offset, size = struct.unpack_from("<QQ", elf, shoff + i * shentsize + 24)
        if kind != 7:  # SHT_NOTE
            continue
        namesz, descsz, _ = struct.unpack_from("<III", elf, offset)
        desc = offset + 12 + (namesz + 3) // 4 * 4
        return {k[".name"]: k for k in msgpack.unpackb(elf[desc:desc + descsz])["amdhsa.kernels"]}
    return {}


KERNELS = ("kv_write_q8_kernel", "kv_read_q8_kernel", "attn_decode_q8_kernel", "attn_shared_prefix_kernel", "attn_prefix_chain_kernel",
           "rows_combine_kernel")


def test_accumulators_and_operands_stay_in_vector_registers():
    """No kernel keeps anything in AGPRs (with which fp32 products have read overwritten operands) or in scratch memory."""
    found = gfx950_kernels()
    for kernel in KERNELS:
        mine = {n: k for n, k in found.items() if kernel in n}
        assert len(mine) >= 4, kernel
        for n, k in mine.items():
            assert k[".agpr_count"] == 0, n
            assert k[".vgpr_spill_count"] == 0 and k[".private_segment_fixed_size"] == 0, n
