"""What the compiler reports of the attention kernels' registers, read from the built
library's own notes: scalar registers that it keeps in lanes of vector registers, and
memory of a work-item's own.  Gradient kernels that kept most of their lane masks so once
gave wrong gradients, for a cause that was not found; here only sizes, strides and
addresses are left, and no more than a stated number of them.  No device is needed."""

from __future__ import annotations

import re
import shutil
import struct
import subprocess
from pathlib import Path

import pytest

LIBRARY = Path(__file__).resolve().parent.parent / "nanotorch_amd" / "libnt.so"
MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"
READELF = shutil.which("llvm-readelf", path="/opt/rocm/llvm/bin:/opt/rocm/bin")

# (kernels, scalar registers, bytes of scratch) at most
LIMITS = [
    (r"attn_(wide_)?fwd_kernel|attn_split_fwd|attn_pack|attn_pad|attn_join|attn_split_join"
     r"|attn_split_parts", 0, 0),
    (r"attn_fwd_left_kernel", 80, 0),
    (r"attn_(wide_)?bwd_kernel", 80, 0),
    (r"attn_bwd_left_kernel", 120, 0),
    (r"attn_split_dq_kernel|attn_split_dkv_kernel", 80, 80),
]


def code_objects(data: bytes):
    """The device ELF files of every bundle."""
    at = data.find(MAGIC)
    while at >= 0:
        count, = struct.unpack_from("<Q", data, at + len(MAGIC))
        p = at + len(MAGIC) + 8
        for _ in range(count):
            offset, size, n = struct.unpack_from("<QQQ", data, p)
            name = data[p + 24:p + 24 + n]
            p += 24 + n
            if b"gfx950" in name and size:
                yield data[at + offset:at + offset + size]
        at = data.find(MAGIC, p)


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    if READELF is None:
        pytest.skip("needs llvm-readelf")
    found = {}
    path = tmp_path_factory.mktemp("objects") / "object"
    for elf in code_objects(LIBRARY.read_bytes()):
        if b"attn_" not in elf:
            continue
        path.write_bytes(elf)
        notes = subprocess.run([READELF, "--notes", str(path)], capture_output=True, text=True,
                               check=True).stdout
        for entry in re.split(r"^  - \.a", notes, flags=re.M)[1:]:
            value = {k: int(re.search(rf"\.{k}: +(\d+)", entry).group(1)) for k in
                     ("sgpr_spill_count", "private_segment_fixed_size")}
            found[re.search(r"\.name: +(\S*attn_\S*|\S+)", entry).group(1)] = value
    return {k: v for k, v in found.items() if "attn_" in k}


def test_every_kernel_is_known(kernels):
    assert len(kernels) > 60
    for name in kernels:
        assert sum(bool(re.search(pattern, name)) for pattern, *_ in LIMITS) == 1, name


@pytest.mark.parametrize("pattern,scalars,scratch", LIMITS)
def test_registers_that_do_not_fit(kernels, pattern, scalars, scratch):
    some = {k: v for k, v in kernels.items() if re.search(pattern, k)}
    assert some
    over = {k: v for k, v in some.items() if v["sgpr_spill_count"] > scalars
            or v["private_segment_fixed_size"] > scratch}
    assert not over
