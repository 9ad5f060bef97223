"""A flush of a handle without a plan, as hosts of the operators on caller memory have it: it waits, and reports once what a
kernel raised."""

import os
import subprocess

import pytest
import torch

from see_ai_b200 import backend as B
from see_ai_b200 import build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def probe(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("probe") / "unbound_flush_probe")
    if not os.path.exists(B.LIB_PATH):
        build.build()
    lib_dir = os.path.dirname(B.LIB_PATH)
    subprocess.run(["g++"] + build.CXX_FLAGS + [os.path.join(ROOT, "tests", "unbound_flush_probe.cc"), "-o", exe, f"-L{lib_dir}", "-lsee_cuda",
                                                f"-Wl,-rpath,{lib_dir}"], check=True, capture_output=True, text=True)
    return exe


def test_probe_builds(probe):
    assert os.path.exists(probe)


@pytest.mark.gpu
def test_wait_that_ran_out_is_reported_once(probe):
    said = subprocess.run([probe], check=True, capture_output=True, text=True).stdout.splitlines()
    assert said == ["ok", "cuda: a bounded device-side wait ran out", "ok"]


@pytest.mark.gpu
def test_flush_waits_for_the_stream():
    be, stream = B.CudaBackend(0), torch.cuda.Stream()
    be.set_stream(stream.cuda_stream)
    x, y, rstd = torch.ones(4096, 4096, device="cuda"), torch.zeros(4096, 4096, device="cuda"), torch.zeros(4096, device="cuda")
    gamma = torch.ones(4096, device="cuda")
    torch.cuda.synchronize()
    for _ in range(50):
        be.norm_forward(B.NORM_RMS, 4096, 4096, x.data_ptr(), gamma.data_ptr(), 0, y.data_ptr(), 0, rstd.data_ptr(), eps=0.0)
    be.flush()
    assert stream.query()
    assert (y == 1).all()
    be.close()
