"""What int8_linear.hip's large tiles rest on, read from the AMD assembly that
the source is compiled to (no GPU needed).

A tile of 256 x 256 fills the registers.  Once an address that had been spilled
was brought back under a guarded store's partial mask, and the lanes that were
masked there read from anywhere: so nothing here may be spilled.

A tile's wait for the next step's operands counts the loads of the later steps,
which have to be all that its loop asks memory for."""
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")


@pytest.fixture(scope="module")
def text(tmp_path_factory):
    if not os.path.exists(HIPCC):
        pytest.skip("no hipcc")
    out = tmp_path_factory.mktemp("asm") / "int8_linear.s"
    csrc = os.path.join(ROOT, "vectorstorekit_amd", "csrc")
    subprocess.run([HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC",
                    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
                    "-I" + os.path.join(ROOT, "include"), "-I" + csrc, "--cuda-device-only", "-S",
                    os.path.join(csrc, "int8_linear.hip"), "-o", str(out)],
                   check=True, capture_output=True, timeout=600)
    return out.read_text()


def test_nothing_is_spilled(text):
    kernels = re.findall(r"\.name:\s+(\S*k_int8_\w+)$", text, re.M)
    # tiles: four of each output type; few tokens: two; one launch: three sizes of
    # nine pairs of types; quantising: two of each type; all of these but tiles
    # and few tokens aligned and not; and the codes of the caller's own
    assert len(kernels) == 3 * 4 + 3 * 2 + 9 * 3 * 2 + 3 * 2 * 2 + 1
    for what in ("vgpr_spill_count", "sgpr_spill_count", "private_segment_fixed_size"):
        values = re.findall(r"\." + what + r":\s+(\d+)$", text, re.M)
        assert len(values) == len(kernels) and set(values) == {"0"}, what


def test_tiles_wait_for_what_they_load(text):
    found = 0
    for m in re.finditer(r"^(\S*k_int8_tileI\w*?Li(\d)ELi(\d)ELi(\d)ELi(\d)EEEv\S+):(.*?)^\.Lfunc_end",
                         text, re.M | re.S):
        name, (fn, fm, step, stages) = m[1], map(int, m.groups()[1:5])
        lines = [x.strip() for x in m[6].split("\n")]
        loads = 2 * (fn + fm) * step // 4  # of a wave and step
        wait = [i for i, x in enumerate(lines) if x.startswith("s_waitcnt vmcnt(")
                and "#ASMSTART" in lines[i - 1]]
        counts = [int(re.search(r"vmcnt\((\d+)\)", lines[i])[1]) for i in wait]
        assert counts == [0, (stages - 3) * loads, 0], (name, counts)
        # the pipelined loop: from its label to the one branch back there
        head = max(i for i in range(wait[1]) if re.match(r"\.LBB\w+:", lines[i]))
        label = re.escape(lines[head].split(":")[0])
        back = [i for i in range(wait[1], len(lines))
                if re.match(r"s_c?branch\S*\s+" + label + "$", lines[i])]
        assert len(back) == 1, name
        asked = [x.split()[0] for x in lines[head:back[0]]
                 if re.match(r"(global|flat|scratch|buffer)_", x)]
        assert asked == ["global_load_lds_dwordx4"] * loads, (name, asked)
        found += 1
    assert found == 3 * 4
