"""The workspace that the query asks for suffices for every gradient that is wanted, whatever number of SMs the device has."""

import os
import subprocess

from see_ai_b200 import backend as B
from see_ai_b200 import build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_no_device_wants_more_than_the_query_says(tmp_path):
    if not os.path.exists(B.LIB_PATH):
        build.build()
    exe, lib_dir = str(tmp_path / "gated_workspace_probe"), os.path.dirname(B.LIB_PATH)
    subprocess.run(["g++"] + build.CXX_FLAGS + [os.path.join(ROOT, "tests", "gated_workspace_probe.cc"), "-o", exe, f"-L{lib_dir}", "-lsee_cuda",
                                                f"-Wl,-rpath,{lib_dir}"], check=True, capture_output=True, text=True)
    lines = [list(map(int, line.split())) for line in subprocess.run([exe], check=True, capture_output=True, text=True).stdout.splitlines()]
    assert {sms for sms, _, _ in lines} >= {2, 132, 148, 160} and all(tried > 4000 for _, tried, _ in lines)
    assert [(sms, short) for sms, _, short in lines if short] == []
