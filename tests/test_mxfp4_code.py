"""The built MXFP4 kernels' resources, from the code objects' metadata (no GPU needed):
they keep everything in registers and LDS."""
import struct

import pytest

msgpack = pytest.importorskip("msgpack")

MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"


def code_objects(lib: bytes):
    """the gfx950 ELF images in a host library's offload bundles"""
    at = lib.find(MAGIC)
    while at >= 0:
        n, p = struct.unpack_from("<Q", lib, at + len(MAGIC))[0], at + len(MAGIC) + 8
        for _ in range(n):
            off, size, tlen = struct.unpack_from("<QQQ", lib, p)
            if b"gfx950" in lib[p + 24:p + 24 + tlen]:
                yield lib[at + off:at + off + size]
            p += 24 + tlen
        at = lib.find(MAGIC, at + 1)


def kernels(elf: bytes):
    """the kernels' entries of the code object's AMDGPU metadata note (type 32)"""
    phoff, phentsize, phnum = struct.unpack_from("<Q", elf, 32)[0], *struct.unpack_from("<HH", elf, 54)
    for i in range(phnum):
        kind, _, off, _, _, size = struct.unpack_from("<IIQQQQ", elf, phoff + i * phentsize)
        if kind != 4:   # PT_NOTE
            continue
        p = off
        while p < off + size:
            nlen, dlen, typ = struct.unpack_from("<III", elf, p)
            desc = p + 12 + (nlen + 3) // 4 * 4
            if typ == 32 and elf[p + 12:p + 18] == b"AMDGPU":
                yield from msgpack.unpackb(elf[desc:desc + dlen])["amdhsa.kernels"]
            p = desc + (dlen + 3) // 4 * 4


def test_mxfp4_kernels_use_no_scratch_memory():
    import helexa_amd as hx
    found = {}
    for elf in code_objects(open(hx.moe.LIB_PATH, "rb").read()):
        for k in kernels(elf):
            if "k_mx_" in k[".name"]:
                found[k[".name"]] = (k[".private_segment_fixed_size"], k[".vgpr_spill_count"], k[".sgpr_spill_count"])
    assert len(found) > 20
    assert not {n: v for n, v in found.items() if v != (0, 0, 0)}
