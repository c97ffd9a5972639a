"""Scratch memory of the built attention kernels, from the metadata of libsa_hip.so's own code objects: forms of the
forward kernel that store no row sums for a backward pass are not to pay for it with spilled registers."""
import re
import shutil
import struct
import subprocess

import pytest

from sparseattnfunctions_amd import _lib

READELF = shutil.which("llvm-readelf", path="/opt/rocm/llvm/bin:/opt/rocm/bin")


def _code_objects(data):
    """The gfx ELF files embedded in the library's bytes."""
    at = data.find(b"\x7fELF", 1)
    while at >= 0:
        if struct.unpack_from("<H", data, at + 18)[0] == 224:  # EM_AMDGPU
            shoff, = struct.unpack_from("<Q", data, at + 40)
            size, count = struct.unpack_from("<HH", data, at + 58)
            yield data[at:at + shoff + size * count]
        at = data.find(b"\x7fELF", at + 1)


@pytest.mark.skipif(READELF is None, reason="no llvm-readelf")
def test_inference_forms_keep_their_registers(tmp_path):
    with open(_lib.LIB_PATH, "rb") as f:
        data = f.read()
    scratch = {}
    for i, elf in enumerate(_code_objects(data)):
        path = tmp_path / f"{i}.o"
        path.write_bytes(elf)
        notes = subprocess.run([READELF, "--notes", str(path)], check=True, capture_output=True, text=True).stdout
        for name, size in re.findall(r"\.name:\s+(\S+)\n(?:.*\n)*?\s+\.private_segment_fixed_size:\s+(\d+)", notes):
            scratch[name] = int(size)
    # bsa_fwd_kernel<bias, mask, pool, T, D, value columns, fp16 scores, shared, lse>
    form = re.compile(r"bsa_fwd_kernelILb(\d)ELb(\d)ELi(\d+)E(DF16_|DF16b)Li(\d+)ELi(\d+)ELb(\d)ELb(\d)ELb(\d)E")
    seen = 0
    for name, size in scratch.items():
        m = form.search(name)
        if m and m[9] == "0":
            seen += 1
            shared_bias = m[1] == "1" and m[8] == "1" and m[6] == "64"  # (their two extra rows of partials)
            assert size <= (28 if shared_bias else 0), (name, size)
    assert seen >= 30, sorted(scratch)
    # the pair kernel and fp32: as before they could store row sums
    pairs = {n: s for n, s in scratch.items() if "bsa_fwd_pair_kernel" in n}
    assert len(pairs) >= 4 and not any(pairs.values()), pairs
    plain = [s for n, s in scratch.items() if "bsa_fwd_f32_kernelILi64ELi0ELb0E" in n]
    assert len(plain) == 1 and plain[0] <= 36, plain
