"""What attn_rows.hip's hand-written waits rest on, read from the AMD assembly
that this source is compiled to (no GPU needed).

A wave waits for the keys in LDS with a count of the value loads issued after
them.  That is sound where those are exactly that many global loads, which
return in order; flat loads need not, and count as loads of LDS as well."""
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    """Name -> instructions (labels and branches among them) of every instance
    of the token kernel for aligned operands."""
    if not os.path.exists(HIPCC):
        pytest.skip("no hipcc")
    out = tmp_path_factory.mktemp("asm") / "attn_rows.s"
    csrc = os.path.join(ROOT, "vectorstorekit_amd", "csrc")
    subprocess.run([HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC",
                    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
                    "-I" + os.path.join(ROOT, "include"), "-I" + csrc, "--cuda-device-only", "-S",
                    os.path.join(csrc, "attn_rows.hip"), "-o", str(out)],
                   check=True, capture_output=True, timeout=600)
    text = out.read_text()
    found = {}
    for m in re.finditer(r"^(\S*k_attn_rowsI\w+?Lb1EEEv\S+):(.*?)^\.Lfunc_end", text, re.M | re.S):
        found[m[1]] = [x.strip() for x in m[2].split("\n")]
    # f32: heads to 64 in three forms (8, 4 and 1 waves a tile), 128 and 256 in
    # two; each 16-bit type: to 64 and 128 in three, 256 in two
    assert len(found) == 7 + 2 * 8
    return found


def memory(line):
    return re.match(r"(global|flat|scratch|buffer)_\w+", line)


def test_no_flat_loads(kernels):
    for name, lines in kernels.items():
        flat = [x for x in lines if x.startswith("flat_")]
        assert not flat, (name, flat[:3], len(flat))


def test_counted_loads_are_the_values(kernels):
    for name, lines in kernels.items():
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
