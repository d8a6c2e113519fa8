"""The paged attention's kernels keep what they hold in registers: none of them spills vector registers to memory, whatever their launch bounds ask for."""
import os
import re
import subprocess

import pytest

from keys_values_amd import build

TOOLS = os.path.join(os.path.dirname(os.path.dirname(build.HIPCC)), "llvm", "bin")
OBJECT = os.path.join(build.OBJ, "paged_decode.o")


@pytest.mark.skipif(not os.path.isfile(OBJECT) or not os.path.isfile(os.path.join(TOOLS, "clang-offload-bundler")), reason="needs the built object and the compiler's tools")
def test_no_kernel_spills(tmp_path):
    fat, code = str(tmp_path / "fat"), str(tmp_path / "code")
    subprocess.check_call([os.path.join(TOOLS, "llvm-objcopy"), f"--dump-section=.hip_fatbin={fat}", OBJECT, str(tmp_path / "copy.o")])
    subprocess.check_call([os.path.join(TOOLS, "clang-offload-bundler"), "--unbundle", "--type=o", "--targets=hipv4-amdgcn-amd-amdhsa--gfx950", f"--input={fat}", f"--output={code}"])
    notes = subprocess.check_output([os.path.join(TOOLS, "llvm-readelf"), "--notes", code], text=True)
    kernels = re.findall(r"\.name:\s+(\S*paged_\w+_kernel\S*)\n(?:.*\n)*?\s+\.private_segment_fixed_size: (\d+)\n(?:.*\n)*?\s+\.vgpr_spill_count: (\d+)\n", notes)
    decode = [k for k in kernels if "paged_decode_kernel" in k[0]]
    assert len(decode) == 36  # three head sizes, six stores, all pages or chosen ones
    assert all(scratch == "0" and spilled == "0" for _, scratch, spilled in kernels), [k for k in kernels if k[1:] != ("0", "0")]
