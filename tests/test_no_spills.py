"""The kernels of the norm, the 4-bit integer products and the experts keep what they hold in registers: none of them uses memory for spilled
registers, by the descriptions that the compiler puts beside each kernel in the built library."""
import os
import re
import struct
import subprocess

import pytest
from launch_recorder import LIBRARY

MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"
READELF = "/opt/rocm/llvm/bin/llvm-readelf"


@pytest.fixture(scope="module")
def descriptions(tmp_path_factory):
    """{kernel: {field: value}} of every kernel in the library"""
    if not os.path.exists(READELF):
        pytest.skip("no llvm-readelf")
    path = str(tmp_path_factory.mktemp("code") / "code.elf")
    data = open(LIBRARY, "rb").read()
    out = {}
    for at in (m.start() for m in re.finditer(MAGIC, data)):
        (entries,) = struct.unpack_from("<Q", data, at + len(MAGIC))
        place = at + len(MAGIC) + 8
        for _ in range(entries):
            offset, size, length = struct.unpack_from("<QQQ", data, place)
            target = data[place + 24:place + 24 + length]
            place += 24 + length
            if b"gfx950" not in target:
                continue
            with open(path, "wb") as f:
                f.write(data[at + offset:at + offset + size])
            notes = subprocess.run([READELF, "--notes", path], check=True, capture_output=True, text=True).stdout
            for kernel in re.split(r"\n  - \.a", notes)[1:]:
                fields = dict(re.findall(r"^\s+\.(\w+):\s+(\S+)\s*$", kernel, re.M))
                out[fields["symbol"]] = fields
    return out


def test_no_register_is_spilled(descriptions):
    ours = {n: f for n, f in descriptions.items() if re.search(r"rmsnorm_|int4_|moe_", n)}
    assert len(ours) > 200
    spilled = {n: f for n, f in ours.items() if int(f["vgpr_spill_count"]) or int(f["sgpr_spill_count"]) or int(f["private_segment_fixed_size"])}
    assert not spilled
