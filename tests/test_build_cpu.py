"""The built library's own metadata."""
import struct

import pytest


def code_objects(path):
    """gfx950 code objects of a HIP library: the entries of its offload bundles"""
    data = open(path, 'rb').read()
    at = data.find(b'__CLANG_OFFLOAD_BUNDLE__')
    while at >= 0:
        p = at + 32
        for _ in range(struct.unpack_from('<Q', data, at + 24)[0]):
            offset, size, n = struct.unpack_from('<QQQ', data, p)
            if b'gfx950' in data[p + 24:p + 24 + n]:
                yield data[at + offset:at + offset + size]
            p += 24 + n
        at = data.find(b'__CLANG_OFFLOAD_BUNDLE__', at + 24)


def kernels(code):
    """kernel records of a code object: the AMDGPU metadata note (type 32) of the ELF file"""
    msgpack = pytest.importorskip('msgpack')
    table, = struct.unpack_from('<Q', code, 0x28)
    entry, count = struct.unpack_from('<HH', code, 0x3A)
    for i in range(count):
        kind, = struct.unpack_from('<I', code, table + i * entry + 4)
        p, size = struct.unpack_from('<QQ', code, table + i * entry + 24)
        end = p + size
        while kind == 7 and p < end:
            name, length, note = struct.unpack_from('<III', code, p)
            p += 12 + (name + 3) // 4 * 4
            if note == 32:
                yield from msgpack.unpackb(code[p:p + length])['amdhsa.kernels']
            p += (length + 3) // 4 * 4


def test_no_kernel_uses_scratch_memory():
    """Registers that do not fit are a cost everywhere and have been a wrong result: where half of a four-register value went to scratch and
    half to accumulation registers, the compiler brought three of the four back."""
    from semseg_amd import _lib
    _lib.lib()
    found = [k for c in code_objects(_lib.LIB_PATH) for k in kernels(c)]
    assert len(found) > 500
    assert not [(k['.name'], k['.private_segment_fixed_size']) for k in found if k['.private_segment_fixed_size']]
