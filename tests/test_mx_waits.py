"""The tile kernels of mx_linear reuse LDS behind barriers of their own: in the code that the library
holds, no wave reaches a barrier with an LDS read under way. No GPU."""
import ctypes
import os
import re
import subprocess

import pytest

from dli import hip

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"


def kernels(tmp_path):
    """The instructions of every kernel of this library's mx_linear code object."""
    image, size = ctypes.c_void_p(), ctypes.c_size_t()
    assert hip.load().dli_hip_code_object(b"mx_linear", ctypes.byref(image), ctypes.byref(size)) == 0
    path = tmp_path / "mx_linear.co"
    path.write_bytes(ctypes.string_at(image, size.value))
    text = subprocess.run([OBJDUMP, "-d", str(path)], check=True, capture_output=True, text=True).stdout
    out = {}
    for line in text.splitlines():
        name = re.match(r"^[0-9a-f]+ <(\w+)>:", line)
        if name:
            out[name[1]] = code = []
        elif out and line.startswith("\t"):
            code.append(line.split("//")[0].strip())
    return out


@pytest.mark.skipif(not os.path.exists(OBJDUMP), reason="no disassembler")
def test_no_lds_read_crosses_a_barrier(tmp_path):
    found = kernels(tmp_path)
    tiles = [n for n in found if n.startswith("mx_tile_")]
    assert len(tiles) == 36
    crossed = []
    for name in tiles:
        code = found[name]
        barriers = [i for i, ins in enumerate(code) if ins.startswith("s_barrier")]
        # the stages' three, and the one before the epilogue writes over the last stage
        assert len(barriers) >= 4
        for i in barriers:
            for ins in reversed(code[:i]):
                if ins.startswith("s_waitcnt") and "lgkmcnt(0)" in ins:
                    break
                if ins.startswith("ds_read"):
                    crossed.append((name, i))
                    break
    assert not crossed
