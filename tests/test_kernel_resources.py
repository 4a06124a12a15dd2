"""What the compiler gave the operators' kernels, read from the metadata of the library's own
code object: none may keep values in scratch memory."""
import struct

import pytest

msgpack = pytest.importorskip("msgpack")

BUNDLE = b"__CLANG_OFFLOAD_BUNDLE__"
METADATA = 32  # NT_AMDGPU_METADATA


def code_objects(blob):
    """The GPU code objects of an uncompressed offload bundle in the library."""
    at = blob.find(BUNDLE)
    while at >= 0:
        count, = struct.unpack_from("<Q", blob, at + len(BUNDLE))
        entry = at + len(BUNDLE) + 8
        if count <= 64:
            for _ in range(count):
                offset, size, length = struct.unpack_from("<QQQ", blob, entry)
                name = blob[entry + 24:entry + 24 + length]
                entry += 24 + length
                if b"gfx950" in name and size:
                    yield blob[at + offset:at + offset + size]
        at = blob.find(BUNDLE, at + 1)


def kernels(elf):
    assert elf[:4] == b"\x7fELF"
    start, = struct.unpack_from("<Q", elf, 32)  # program headers
    size, count = struct.unpack_from("<HH", elf, 54)
    for i in range(count):
        kind, _, offset, _, _, length = struct.unpack_from("<IIQQQQ", elf, start + i * size)
        if kind != 4:  # PT_NOTE
            continue
        at, end = offset, offset + length
        while at + 12 <= end:
            name, desc, note = struct.unpack_from("<III", elf, at)
            body = at + 12 + (name + 3) // 4 * 4
            if note == METADATA:
                yield from msgpack.unpackb(elf[body:body + desc], raw=False)["amdhsa.kernels"]
            at = body + (desc + 3) // 4 * 4


def test_operators_keep_their_values_in_registers():
    from cq35 import _lib
    with open(_lib.LIBRARY, "rb") as f:
        blob = f.read()
    found = {k[".name"]: k for elf in code_objects(blob) for k in kernels(elf)}
    mine = {n: k for n, k in found.items() if any(w in n for w in ("k_int8_rows", "k_int8_tiles", "k_int8_few", "k_logprobs"))}
    assert sum("k_int8_rows" in n for n in mine) == 18 and len(mine) > 30, sorted(mine)
    spilled = {n: k[".private_segment_fixed_size"] for n, k in mine.items() if k[".private_segment_fixed_size"]}
    assert not spilled, spilled
