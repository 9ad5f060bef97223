"""Which logit_scale the losses over rows of logits take, without a device."""

import os
import subprocess

import pytest

from see_ai_b200 import backend as B
from see_ai_b200 import build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def said(tmp_path_factory):
    if not os.path.exists(B.LIB_PATH):
        build.build()
    exe = str(tmp_path_factory.mktemp("probe") / "logit_scale_probe")
    lib_dir = os.path.dirname(B.LIB_PATH)
    subprocess.run(["g++"] + build.CXX_FLAGS + [os.path.join(ROOT, "tests", "logit_scale_probe.cc"), "-o", exe, f"-L{lib_dir}", "-lsee_cuda",
                                                f"-Wl,-rpath,{lib_dir}"], check=True, capture_output=True, text=True)
    return [line.split("\t") for line in subprocess.run([exe], check=True, capture_output=True, text=True).stdout.splitlines()]


@pytest.mark.parametrize("loss", ["policy", "preference"])
def test_from_2_to_the_minus_100_to_2_to_the_100(said, loss):
    mine = [(float.fromhex(scale), answer) for which, scale, answer in said if which == loss]
    assert len(mine) == 18
    for scale, answer in mine:
        assert answer == "ok" if 2.0 ** -100 <= scale <= 2.0 ** 100 else "logit_scale" in answer, (scale, answer)
