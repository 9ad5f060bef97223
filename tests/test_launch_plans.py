"""What the host decides before it launches, over many sizes and without a device."""

import os
import subprocess

import pytest

from see_ai_b200 import build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FAMILIES = ["grad tables", "join rings"]


@pytest.fixture(scope="module")
def said(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("probe") / "launch_plans_probe")
    subprocess.run(["g++"] + build.CXX_FLAGS + [os.path.join(ROOT, "tests", "launch_plans_probe.cc"), "-o", exe], check=True, capture_output=True, text=True)
    out = subprocess.run([exe], check=True, capture_output=True, text=True).stdout
    return dict(line.split("\t", 1) for line in out.splitlines())


def test_every_family_is_expected(said):
    assert sorted(said) == sorted(FAMILIES)


@pytest.mark.parametrize("name", FAMILIES)
def test_plans(said, name):
    assert said[name] == "ok", said[name]
