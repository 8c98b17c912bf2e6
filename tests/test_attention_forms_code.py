"""What test_attention_code.py holds of the token kernel, of the kernels that
have its loop in other forms (cross attention, shared prefixes): their waits
count the value loads behind a step's keys, which have to be just so many
global loads.  Read from the AMD assembly (no GPU needed)."""
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")


def memory(line):
    return re.match(r"(global|flat|scratch|buffer)_\w+", line)


@pytest.mark.parametrize("source,pattern,instances", [
    # as of k_attn_rows; each 16-bit type at heads of 64, 96 and 128
    ("attn_forms", r"k_attn_formsI\w+?Lb1EEEv", 7 + 2 * 8), ("attn_shared", "k_attn_sharedI", 2 * 3)])
def test_counted_loads_are_the_values(tmp_path, source, pattern, instances):
    if not os.path.exists(HIPCC):
        pytest.skip("no hipcc")
    out = tmp_path / (source + ".s")
    csrc = os.path.join(ROOT, "vectorstorekit_amd", "csrc")
    subprocess.run([HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC",
                    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
                    "-I" + os.path.join(ROOT, "include"), "-I" + csrc, "--cuda-device-only", "-S",
                    os.path.join(csrc, source + ".hip"), "-o", str(out)],
                   check=True, capture_output=True, timeout=600)
    found = 0
    for m in re.finditer(r"^(\S*" + pattern + r"\S+):(.*?)^\.Lfunc_end", out.read_text(),
                         re.M | re.S):
        name, lines = m[1], [x.strip() for x in m[2].split("\n")]
        found += 1
        assert not [x for x in lines if x.startswith("flat_")], name
        wait = [i for i, x in enumerate(lines) if x.startswith("s_waitcnt vmcnt(")
                and "#ASMSTART" in lines[i - 1]]
        assert len(wait) == 1, name
        count = int(re.search(r"vmcnt\((\d+)\)", lines[wait[0]])[1])
        # the loop's head, and every way there
        head = max(i for i in range(wait[0]) if re.match(r"\.LBB\w+:", lines[i]))
        assert not [x for x in lines[head:wait[0]] if memory(x)], name
        label = lines[head].split(":")[0]
        ways = [head] + [i for i, x in enumerate(lines)
                         if re.match(r"s_c?branch\S*\s+" + re.escape(label) + "$", x)]
        assert len(ways) == 2, (name, len(ways))
        for at in ways:
            issued = [memory(x)[0] for x in lines[:at] if memory(x)][-count:]
            assert len(issued) == count, name
            assert all(re.fullmatch(r"global_load_dwordx[24]", x) for x in issued), (name, issued)
    assert found == instances
