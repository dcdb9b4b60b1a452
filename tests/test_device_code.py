"""The device code of the built library, as the assembler lists it (CPU only)."""
import os
import re
import struct
import subprocess

import pytest

from tests.conftest import PKG

LIB = os.path.join(PKG, "libloom_hip.so")
OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"


def code_objects():
    """The gfx950 code objects of the library's offload bundles."""
    data = open(LIB, "rb").read()
    magic = b"__CLANG_OFFLOAD_BUNDLE__"
    for m in re.finditer(magic, data):
        n, = struct.unpack_from("<Q", data, m.end())
        at = m.end() + 8
        for _ in range(n):
            off, size, length = struct.unpack_from("<QQQ", data, at)
            name = data[at + 24:at + 24 + length]
            at += 24 + length
            if name.endswith(b"gfx950") and size:
                yield data[m.start() + off:m.start() + off + size]


def test_no_flat_memory_instructions(tmp_path):
    """Kernels that place their own counted waits rely on memory operations completing in
    the order in which they are issued.  Flat ones (of a pointer that the compiler does not
    know to be global) need not, and count as LDS operations too."""
    if not os.path.exists(OBJDUMP):
        pytest.skip("llvm-objdump is not installed")
    kernels, flat = 0, {}
    for i, code in enumerate(code_objects()):
        path = tmp_path / f"{i}.co"
        path.write_bytes(code)
        name = None
        for line in subprocess.run([OBJDUMP, "-d", str(path)], check=True, capture_output=True,
                                   text=True).stdout.splitlines():
            if m := re.match(r"[0-9a-f]+ <(\w+)>:", line):
                name, kernels = m.group(1), kernels + 1
            elif re.search(r"\sflat_(load|store|atomic)", line):
                flat[name] = flat.get(name, 0) + 1
    assert kernels > 100
    assert not flat, flat
