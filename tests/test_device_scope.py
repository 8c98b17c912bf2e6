"""Calls that run between a program's own leave its current device as it was
(no GPU needed: the runtime's two functions are counted)."""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "vectorstorekit_amd", "csrc")


@pytest.mark.skipif(shutil.which("g++") is None or not os.path.isdir("/opt/rocm/include"),
                    reason="no g++ or no HIP headers")
def test_device_is_set_back(tmp_path):
    exe = tmp_path / "device_scope"
    subprocess.run(["g++", "-std=c++17", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", "-I", CSRC,
                    os.path.join(ROOT, "tests", "device_scope.cpp"), "-o", str(exe)],
                   check=True, capture_output=True, text=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and "device scope ok" in r.stdout


def test_every_queued_call_has_it():
    header = open(os.path.join(ROOT, "include", "vsk_hip.h")).read()
    section = header[header.index("---- key-value cache and attention"):]
    calls = set(re.findall(r"^vsk_status (vsk_\w+)\(", section, re.M))
    assert len(calls) == 10
    text = "".join(open(os.path.join(CSRC, f)).read()
                   for f in ("rotary.hip", "kvcache.hip", "attention.hip"))
    for name in calls:
        body = re.search(r"^vsk_status " + name + r"\(.*?^}", text, re.M | re.S)[0]
        assert "QUEUED_API_BEGIN(ctx);" in body or "DeviceScope scope(" in body, name
