"""What the norm, gated and AdamW operators refuse, without a device: the library's own checks on made-up addresses."""

import os
import subprocess

import pytest

from see_ai_b200 import backend as B
from see_ai_b200 import build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# None: taken; otherwise a part of the message.
EXPECTED = {
    "norm": None, "norm kind": "unknown kind", "norm x_type": "x_type and y_type", "norm types": "x_type and y_type",
    "norm eps": "eps", "norm eps nan": "eps", "norm no columns": "16384 columns", "norm columns": "16384 columns",
    "norm rows": "2^31 - 1 rows", "norm stride": "stride", "norm stride wide": "stride", "norm null": "gamma is null",
    "norm null mean": "mean is null", "norm aligned": "x is not aligned", "norm in place": "x and y overlap",
    "norm behind": None, "norm into": "x and y overlap", "norm side by side": None, "norm side into": "x and y overlap",
    "norm rms beta": "rms has neither", "norm rms": None, "norm empty": None,
    "norm back": None, "norm back addend": None, "norm back addend into": "dx and addend overlap",
    "norm back work": "workspace is too small", "norm back work null": "workspace is null",
    "norm back work aligned": "workspace is not aligned", "norm back work into": "overlap", "norm back dbeta": "dbeta is null",
    "norm back rms dbeta": "rms has neither",
    "gated": None, "gated not kept": None, "gated half kept": "together", "gated type": "bf16 or f16", "gated act": "activation",
    "gated d_in": "multiples of 8", "gated d_hidden": "multiples of 8", "gated no d_in": "multiples of 8", "gated rows": "2^31 - 256",
    "gated rows by widths": "too many rows", "gated stride": "stride", "gated aligned": "w_gate is not aligned", "gated null": "x is null",
    "gated into": "hidden and gate overlap", "gated side by side": None,
    "gated back": None, "gated back dx": None, "gated back dw": None, "gated back half dw": "together",
    "gated back nothing": "no output", "gated back work": "workspace is too small", "gated back work aligned": "workspace is not aligned",
    "gated back into": "x and dx overlap", "gated back weights": "w_gate and dw_gate overlap",
    "adamw": None, "adamw 32": None, "adamw bits": "8 or 32 bits", "adamw step": "count from 1", "adamw beta": "beta1 and beta2",
    "adamw g_type": "tensor 1: unknown type", "adamw copy": "tensor 1: a copy", "adamw no copy": None, "adamw flag": "tensor 2: unknown flag",
    "adamw null": "tensor 2: v is null", "adamw scale null": "tensor 0: m_scale is null", "adamw aligned": "tensor 0: p is not aligned",
    "adamw large": "2^38", "adamw twice": "overlap", "adamw into": "overlap", "adamw p over g": "overlap", "adamw same g": None,
    "adamw descending": None, "adamw interleaved": None, "adamw scale in p": "overlap", "adamw scale": None,
    "adamw scale aligned": "grad_scale is not aligned", "adamw empty tensor": None, "adamw none": None, "adamw no table": "tensors is null",
    "handle": None, "handle gated": None, "handle adamw": None,
}


@pytest.fixture(scope="module")
def said(tmp_path_factory):
    if not os.path.exists(B.LIB_PATH):
        build.build()
    exe = str(tmp_path_factory.mktemp("probe") / "block_checks_probe")
    lib_dir = os.path.dirname(B.LIB_PATH)
    subprocess.run(["g++"] + build.CXX_FLAGS + [os.path.join(ROOT, "tests", "block_checks_probe.cc"), "-o", exe, f"-L{lib_dir}", "-lsee_cuda",
                                                f"-Wl,-rpath,{lib_dir}"], check=True, capture_output=True, text=True)
    out = subprocess.run([exe], check=True, capture_output=True, text=True).stdout
    return dict(line.split("\t", 1) for line in out.splitlines())


def test_every_call_is_expected(said):
    assert sorted(said) == sorted(EXPECTED)


@pytest.mark.parametrize("name", sorted(EXPECTED))
def test_refusal(said, name):
    want = EXPECTED[name]
    assert said[name] == "ok" if want is None else want in said[name], said[name]


def test_workspaces():
    assert B.norm_backward_workspace(0, 16) > 0 and B.norm_backward_workspace(10, 0) == 0 and B.norm_backward_workspace(10, 20000) == 0
    assert B.norm_backward_workspace(10, 64) == 10 * 64 * 8
    assert B.norm_backward_workspace(1 << 20, 64) == B.norm_backward_workspace(4096, 64)
    assert B.gated_backward_workspace(0, 64, 64) > 0 and B.gated_backward_workspace(8, 60, 64) == 0
    assert B.gated_backward_workspace(512, 64, 64) >= 2 * 512 * 64 * 2
