"""What the built library says of the kernels of chunks over the paged cache
(the notes that the compiler puts beside a kernel's code)."""
import struct

import pytest

import g4

msgpack = pytest.importorskip("msgpack")


def code_objects(data):
    """the gfx950 code objects of a library, each source file's own"""
    magic, at = b"__CLANG_OFFLOAD_BUNDLE__", 0
    while (at := data.find(magic, at)) >= 0:
        p = at + len(magic) + 8
        for _ in range(struct.unpack_from("<Q", data, p - 8)[0]):
            offset, size, name = struct.unpack_from("<QQQ", data, p)
            if size and b"amdgcn" in data[p + 24:p + 24 + name]:
                yield data[at + offset:at + offset + size]
            p += 24 + name
        at += len(magic)


def kernels(elf):
    """the metadata of a code object's kernels: its note of type 32"""
    start, (size, count) = struct.unpack_from("<Q", elf, 40)[0], struct.unpack_from("<HH", elf, 58)
    for i in range(count):
        at = start + i * size
        if struct.unpack_from("<I", elf, at + 4)[0] != 7:
            continue
        p, length = struct.unpack_from("<QQ", elf, at + 24)
        end = p + length
        while p < end:
            name, desc, kind = struct.unpack_from("<III", elf, p)
            d = p + 12 + (name + 3) // 4 * 4
            if kind == 32:
                yield from msgpack.unpackb(elf[d:d + desc])["amdhsa.kernels"]
            p = d + (desc + 3) // 4 * 4


def test_no_vector_register_in_memory():
    """No kernel of attn_chunk.hip keeps registers in scratch.  Not for speed alone: where one more register was needed
    (weights as two terms, bf16 of 256) the compiler put the store of one that all lanes need into a branch of one lane, and
    the second launch was told a share's notes from memory that nobody had written."""
    with open(g4.LIB_PATH, "rb") as f:
        data = f.read()
    found = [k for elf in code_objects(data) for k in kernels(elf) if "ChunkArgs" in k[".name"]]
    # 7 pairs of types and 4 head_dims: rows, tiles (bf16 rows: two), 3 types of rows: joins
    assert len(found) == 7 * 4 * 2 + 2 * 4 + 3 * 4
    spilled = [k[".name"] for k in found if k[".private_segment_fixed_size"] or k.get(".vgpr_spill_count")]
    assert not spilled
