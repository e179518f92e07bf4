"""The compiled kernels, as built here: none calls a function out of line.  (A
lambda that the compiler leaves out of line reaches LDS and its captured
variables through generic pointers, whose flat accesses end where LDS offsets
pass 64 KB.)"""

import os
import shutil
import struct
import subprocess

import pytest

from sunshape_mlx_amd import _hip

LIB = os.path.join(os.path.dirname(_hip.__file__), "libsunshape_hip.so")
MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"


def code_objects(data):
    """The device code objects of the library's offload bundles."""
    at = data.find(MAGIC)
    while at >= 0:
        n, = struct.unpack_from("<Q", data, at + len(MAGIC))
        place = at + len(MAGIC) + 8
        for _ in range(n):
            offset, size, name = struct.unpack_from("<QQQ", data, place)
            triple = data[place + 24:place + 24 + name]
            if b"gfx" in triple and size:
                yield data[at + offset:at + offset + size]
            place += 24 + name
        at = data.find(MAGIC, at + len(MAGIC))


def test_no_kernel_calls_a_function(tmp_path):
    objdump = shutil.which("llvm-objdump", path="/opt/rocm/llvm/bin:" + os.environ.get("PATH", ""))
    if objdump is None:
        pytest.skip("llvm-objdump is not there")
    with open(LIB, "rb") as f:
        objects = list(code_objects(f.read()))
    assert objects
    for i, code in enumerate(objects):
        path = tmp_path / f"{i}.co"
        path.write_bytes(code)
        with subprocess.Popen([objdump, "-d", "--no-show-raw-insn", str(path)], stdout=subprocess.PIPE,
                              text=True) as p:
            name, calls, kernels = "", [], 0
            for line in p.stdout:
                if line.endswith(">:\n"):
                    name, kernels = line, kernels + 1
                elif "s_swappc" in line or "s_call" in line:
                    calls.append(name)
        assert p.returncode == 0 and kernels and not calls, calls[:3]
