"""Operands that cover no bytes have no address to be checked: an empty batch, as a rank or an expert without tokens has it."""

import os
import subprocess

import pytest
import torch

from see_ai_b200 import backend as B
from see_ai_b200 import build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# None: taken; otherwise a part of the message.
EXPECTED = {
    "norm": None, "norm gamma": "gamma is null", "norm beta": "beta is null", "norm addresses": None, "norm back": None,
    "norm back dgamma": "dgamma is null", "norm back dbeta": "dbeta is null", "norm back work": "workspace is null",
    "norm back no bytes": "workspace is too small", "rms": None, "rms back": None, "norm one row": "x is null",
    "gated": None, "gated weights": "w_up is null", "gated back": None, "gated back half": "together", "gated back nothing": "no output",
    "gated back dx": None, "gated back weights": "w_gate is null", "gated one row": "hidden is null",
    "adamw": None, "adamw copy": None, "adamw type": "unknown type", "adamw one element": "a copy has 16 bits",
}


@pytest.fixture(scope="module")
def said(tmp_path_factory):
    if not os.path.exists(B.LIB_PATH):
        build.build()
    exe = str(tmp_path_factory.mktemp("probe") / "empty_operands_probe")
    lib_dir = os.path.dirname(B.LIB_PATH)
    subprocess.run(["g++"] + build.CXX_FLAGS + [os.path.join(ROOT, "tests", "empty_operands_probe.cc"), "-o", exe, f"-L{lib_dir}", "-lsee_cuda",
                                                f"-Wl,-rpath,{lib_dir}"], check=True, capture_output=True, text=True)
    out = subprocess.run([exe], check=True, capture_output=True, text=True).stdout
    return dict(line.split("\t", 1) for line in out.splitlines())


def test_every_call_is_expected(said):
    assert sorted(said) == sorted(EXPECTED)


@pytest.mark.parametrize("name", sorted(EXPECTED))
def test_empty(said, name):
    want = EXPECTED[name]
    assert said[name] == "ok" if want is None else want in said[name], said[name]


@pytest.mark.gpu
def test_tensors_without_rows():
    be = B.CudaBackend(0)
    be.set_stream(torch.cuda.current_stream().cuda_stream)
    none = lambda *s, t=torch.float32: torch.empty(*s, device="cuda", dtype=t).data_ptr()  # noqa: E731
    d, f = 64, 128
    gamma, beta, dgamma, dbeta = (torch.ones(d, device="cuda") for _ in range(4))
    work = torch.empty(B.norm_backward_workspace(0, d), device="cuda", dtype=torch.uint8)
    assert none(0, d) == 0
    be.norm_forward(B.NORM_LAYER, 0, d, none(0, d), gamma.data_ptr(), beta.data_ptr(), none(0, d), none(0), none(0))
    be.norm_backward(B.NORM_LAYER, 0, d, none(0, d), none(0, d), gamma.data_ptr(), none(0), none(0), none(0, d), dgamma.data_ptr(),
                     dbeta.data_ptr(), work.data_ptr(), work.numel(), addend=none(0, d))
    assert (dgamma == 0).all() and (dbeta == 0).all()
    wg, wu, dwg, dwu = (torch.ones(d, f, device="cuda", dtype=torch.bfloat16) for _ in range(4))
    work = torch.empty(B.gated_backward_workspace(0, d, f), device="cuda", dtype=torch.uint8)
    x, h = none(0, d, t=torch.bfloat16), none(0, f, t=torch.bfloat16)
    be.gated_forward(0, d, f, x, wg.data_ptr(), wu.data_ptr(), h, h, h)
    be.gated_backward(0, d, f, h, x, wg.data_ptr(), wu.data_ptr(), h, h, x, dwg.data_ptr(), dwu.data_ptr(), work.data_ptr(), work.numel())
    assert (dwg == 0).all() and (dwu == 0).all()
    rest = {k: torch.ones(300, device="cuda") for k in ("p", "g", "m", "v")}
    copy = torch.empty(300, device="cuda", dtype=torch.bfloat16)
    table = B.adamw_tensors([dict(p=none(0), g=none(0), m=none(0), v=none(0), copy=none(0, t=torch.bfloat16), n=0, copy_type=B.BF16),
                             dict({k: v.data_ptr() for k, v in rest.items()}, copy=copy.data_ptr(), n=300, copy_type=B.BF16)])
    be.adamw_step(table, B.StepParams(1e-3, 0.9, 0.999, 1e-8, 0.0, 0, 1))
    assert (rest["p"] != 1).all() and torch.equal(copy, rest["p"].bfloat16())
    torch.cuda.synchronize()
    be.close()
