"""The built kernels' 16-byte buffer stores: none takes a scalar register as its offset.

A vector instruction right behind such a store that reuses one of its data registers
has changed what was stored on this hardware, in the last lanes of each 16, now and then.
The compiler keeps the two apart only for stores without a register offset."""
import os
import re
import shutil
import struct
import subprocess

import pytest

from onnxsharp_amd import native as N

OBJDUMP = shutil.which("llvm-objdump") or "/opt/rocm/llvm/bin/llvm-objdump"
STORE = re.compile(r"\b(buffer_store_dwordx[34]|buffer_store_b(?:96|128))\s+\S+ \S+ s\[\d+:\d+\], (s\d+|m0|ttmp\d+)\b")


def _code_objects(data: bytes):
    """The GPU code objects (ELF files of machine 224) inside the library."""
    at = data.find(b"\x7fELF", 1)
    while at >= 0:
        machine, = struct.unpack_from("<H", data, at + 18)
        if machine == 224:
            off, = struct.unpack_from("<Q", data, at + 40)  # section headers stand last
            size, count = struct.unpack_from("<HH", data, at + 58)
            yield data[at:at + off + size * count]
        at = data.find(b"\x7fELF", at + 4)


def test_wide_buffer_stores_have_no_scalar_offset(tmp_path):
    if not os.path.exists(OBJDUMP):
        pytest.skip("no llvm-objdump")
    with open(N.LIB_PATH, "rb") as f:
        objects = list(_code_objects(f.read()))
    assert objects
    stores, found = 0, []
    for i, code in enumerate(objects):
        path = tmp_path / f"{i}.co"
        path.write_bytes(code)
        run = subprocess.Popen([OBJDUMP, "-d", "--no-show-raw-insn", str(path)], stdout=subprocess.PIPE, text=True)
        for line in run.stdout:
            if "buffer_store" in line:
                stores += 1
                if STORE.search(line):
                    found.append(line.strip())
        assert run.wait() == 0
    assert stores
    assert not found, f"{len(found)} stores, the first: {found[0]}"
