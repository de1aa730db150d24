"""What the compiler gave the built kernels, from the metadata of the library's own code
objects: kernels whose registers were counted stay out of scratch memory."""
import os
import re
import shutil
import struct
import subprocess

import pytest

import obsidian_hip as oh

READELF = shutil.which("llvm-readelf") or os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "llvm", "bin", "llvm-readelf")
MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"


def code_objects(data):
    """The gfx950 objects of every bundle: (count, then offset, size, length of the name and the name of each)."""
    at = data.find(MAGIC)
    while at >= 0:
        p = at + len(MAGIC)
        n, = struct.unpack_from("<Q", data, p)
        p += 8
        for _ in range(n):
            off, size, ln = struct.unpack_from("<QQQ", data, p)
            name = data[p + 24:p + 24 + ln]
            p += 24 + ln
            if b"gfx950" in name and size:
                yield data[at + off:at + off + size]
        at = data.find(MAGIC, at + 1)


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    """name -> (bytes of scratch a lane, spilled vector registers)."""
    if not os.path.exists(READELF):
        pytest.skip("no llvm-readelf")
    out, dir_ = {}, tmp_path_factory.mktemp("objects")
    with open(oh.LIB_PATH, "rb") as f:
        data = f.read()
    for i, obj in enumerate(code_objects(data)):
        path = dir_ / f"{i}.o"
        path.write_bytes(obj)
        notes = subprocess.run([READELF, "--notes", str(path)], check=True, capture_output=True, text=True).stdout
        # a kernel's fields stand in alphabetical order
        for m in re.finditer(r"\.name: +(\S+)\n(?:.*\n)*? +\.private_segment_fixed_size: (\d+)\n(?:.*\n)*? +\.vgpr_spill_count: (\d+)", notes):
            out[m.group(1)] = int(m.group(2)), int(m.group(3))
    return out


@pytest.mark.parametrize("kernel,forms", [("paged_prefill_kernel", 6)])
def test_no_scratch(kernels, kernel, forms):
    found = {n: v for n, v in kernels.items() if kernel in n}
    assert len(found) == forms
    assert not {n: v for n, v in found.items() if v != (0, 0)}
