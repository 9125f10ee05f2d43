"""The attention kernels as they were built keep everything in registers: what their metadata says of scratch memory is none.  (Their rows and results are sized for
that: a kernel that spills takes twice the time and more, and nothing else would tell.)"""
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BUNDLE = b"__CLANG_OFFLOAD_BUNDLE__"


def code_objects(data):
    """The gfx950 code objects of a library: bundles of (offset, size, name of the target) and what they point to."""
    at = data.find(BUNDLE)
    while at >= 0:
        def number(k):
            return int.from_bytes(data[k:k + 8], "little")
        entries, k = number(at + 24), at + 32
        for _ in range(entries):
            offset, size, name = number(k), number(k + 8), number(k + 16)
            target = data[k + 24:k + 24 + name]
            k += 24 + name
            if b"gfx950" in target:
                yield data[at + offset:at + offset + size]
        at = data.find(BUNDLE, at + 24)


def kernels(obj):
    """{name: (bytes of scratch memory, registers spilled)} from the metadata of a code object: a list of maps, whose keys are in alphabetical order."""
    def value(key, start):
        k = obj.index(key, start) + len(key)
        kind = obj[k]
        if kind < 0x80:
            return kind
        size = {0xcc: 1, 0xcd: 2, 0xce: 4, 0xcf: 8}[kind]
        return int.from_bytes(obj[k + 1:k + 1 + size], "big")
    out = {}
    for m in re.finditer(rb"\xa5\.name(?:[\xa0-\xbf]|\xd9.|\xda..)(_Z[A-Za-z0-9_]+)\xbb\.private_segment_fixed_size", obj, re.S):
        at = m.end() - len(b".private_segment_fixed_size")
        out[m.group(1).decode()] = value(b".private_segment_fixed_size", at), value(b".vgpr_spill_count", at)
    return out


def test_no_attention_kernel_uses_scratch_memory():
    with open(os.path.join(ROOT, "gelib_amd", "libgelib_hip.so"), "rb") as f:
        data = f.read()
    found = {}
    for obj in code_objects(data):
        found.update(kernels(obj))
    attention = {name: v for name, v in found.items() if re.search(r"attention_(fwd|rows|keys)_kernel", name)}
    # three passes, each of float32 with 16, 32, 64 and 128 values and 16-bit types with the last three, with and without points, one wave and four at least
    assert len(attention) >= 3 * (4 + 3 + 3) * 2 * 2, len(attention)
    assert {name: v for name, v in attention.items() if v != (0, 0)} == {}
