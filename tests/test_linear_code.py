"""What int8_linear.hip's large tiles rest on, read from the AMD assembly that
the source is compiled to (no GPU needed).

A tile of 256 x 256 fills the registers.  Once an address that had been spilled
was brought back under a guarded store's partial mask, and the lanes that were
masked there read from anywhere: so nothing here may be spilled."""
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")


def test_nothing_is_spilled(tmp_path):
    if not os.path.exists(HIPCC):
        pytest.skip("no hipcc")
    out = tmp_path / "int8_linear.s"
    csrc = os.path.join(ROOT, "vectorstorekit_amd", "csrc")
    subprocess.run([HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC",
                    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
                    "-I" + os.path.join(ROOT, "include"), "-I" + csrc, "--cuda-device-only", "-S",
                    os.path.join(csrc, "int8_linear.hip"), "-o", str(out)],
                   check=True, capture_output=True, timeout=600)
    text = out.read_text()
    kernels = re.findall(r"\.name:\s+(\S*k_int8_\w+)$", text, re.M)
    # tiles: four of each output type; few tokens: two; one launch: three sizes of
    # nine pairs of types; quantising: two of each type; all of these but tiles
    # and few tokens aligned and not; and the codes of the caller's own
    assert len(kernels) == 3 * 4 + 3 * 2 + 9 * 3 * 2 + 3 * 2 * 2 + 1
    for what in ("vgpr_spill_count", "sgpr_spill_count", "private_segment_fixed_size"):
        values = re.findall(r"\." + what + r":\s+(\d+)$", text, re.M)
        assert len(values) == len(kernels) and set(values) == {"0"}, what
