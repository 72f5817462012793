"""The gfx950 code of a library that was built here, disassembled (for tests of what the compiler made)."""

import functools
import os
import struct
import subprocess

import pytest

OBJDUMP = os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "llvm", "bin", "llvm-objdump")
MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"


def code_objects(path):
    """The gfx950 ELF images in the library's offload bundles."""
    with open(path, "rb") as f:
        data = f.read()
    at = data.find(MAGIC)
    while at >= 0:
        p = at + len(MAGIC)
        (count,) = struct.unpack_from("<Q", data, p)
        p += 8
        for _ in range(count):
            offset, size, idlen = struct.unpack_from("<QQQ", data, p)
            name = data[p + 24:p + 24 + idlen]
            p += 24 + idlen
            if size and name.endswith(b"gfx950"):
                yield data[at + offset:at + offset + size]
        at = data.find(MAGIC, p)


@functools.cache
def disassembly(path, tmp):
    """{kernel: its instructions' texts} of a library, or of a plain code object."""
    if not os.path.exists(OBJDUMP):
        pytest.skip("no llvm-objdump to read the built code with")
    with open(path, "rb") as f:
        head = f.read(64)
    images = list(code_objects(path))
    if not images and head[18:20] == b"\xe0\x00":  # e_machine: AMDGPU
        with open(path, "rb") as f:
            images = [f.read()]
    assert images, f"{path}: no gfx950 code"
    kernels = {}
    for i, image in enumerate(images):
        obj = os.path.join(tmp, f"{os.path.basename(path)}.{i}")
        with open(obj, "wb") as f:
            f.write(image)
        out = subprocess.run([OBJDUMP, "-d", "--mcpu=gfx950", "--no-show-raw-insn", obj], capture_output=True, text=True, check=True).stdout
        lines = None
        for line in out.splitlines():
            if line.endswith(">:"):
                lines = kernels.setdefault(line[line.index("<") + 1:-2], [])
            elif lines is not None and line.startswith(("\t", " ")):
                lines.append(line.split("//")[0].strip())
    return kernels
