"""What the join, preference, policy and gradient-norm operators refuse, without a device: the library's own checks on made-up addresses."""

import os
import subprocess

import pytest

from see_ai_b200 import backend as B
from see_ai_b200 import build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# None: taken; otherwise a part of the message.
EXPECTED = {
    "join": None, "join rms": None, "join no post": None, "join no gate": None, "join kind": "unknown kind", "join types": "x_type and y_type",
    "join y_type": "x_type and y_type", "join eps": "eps", "join scale": "residual_scale", "join no columns": "16384 columns",
    "join columns": "16384 columns", "join rows": "2^31 - 1 rows", "join stride": "stride", "join stride wide": "stride",
    "join no weights": "weights is null", "join no stats": "stats is null", "join rms beta": "rms has neither", "join rms mean": "rms has neither",
    "join layer beta": "post_beta is null", "join stray beta": "go with post_gamma", "join stray rstd": "go with post_gamma",
    "join pre_gamma": "pre_gamma is null", "join post_rstd": "post_rstd is null", "join null": "block is null", "join aligned": "y is not aligned",
    "join gate aligned": "gate is not aligned", "join in place": "x and x_out overlap", "join y over block": "block and y overlap",
    "join side by side": None, "join empty": None,
    "join back": None, "join back rms": None, "join back no post": None, "join back no gate": None, "join back no dx_out": None,
    "join back no gradients": "gradients is null", "join back stray gate": "not there", "join back stray post": "not there",
    "join back rms beta": "not there", "join back gate null": "gate's gradient is null", "join back dbeta null": "post_beta's gradient is null",
    "join back pre_beta unread": None, "join back work": "workspace is too small", "join back work aligned": "workspace is not aligned",
    "join back dx over dx_out": "overlap", "join back dblock over dy": "overlap", "join back gradient over weight": "overlap", "join back empty": None,
    "preference": None, "preference bare": None, "preference in place": None, "preference into logits": "logits and dlogits overlap",
    "preference type": "unknown type", "preference kind": "unknown kind", "preference scale": "logit_scale", "preference scale nan": "logit_scale",
    "preference no classes": "2^20 classes", "preference classes": "2^20 classes", "preference rows": "2^31 - 1 rows", "preference stride": "stride",
    "preference no pairs": "2^24 pairs", "preference pairs": "2^24 pairs", "preference beta": "beta", "preference smoothing": "smoothing",
    "preference smoothed hinge": "smoothing belongs", "preference margin": "margin is not finite", "preference square margin": "no margin",
    "preference work": "workspace is too small", "preference work aligned": "workspace is not aligned", "preference starts": "starts is null",
    "preference labels aligned": "labels is not aligned", "preference loss into margins": "loss and margins overlap", "preference empty": None,
    "policy": None, "policy bare": None, "policy in place": None, "policy into logits": "logits and dlogits overlap", "policy type": "unknown type",
    "policy scale": "logit_scale", "policy classes": "2^20 classes", "policy stride": "stride", "policy low": "clip_low", "policy low nan": "clip_low",
    "policy high": "clip_high", "policy kl": "kl_coef", "policy kl without": "ref_logp", "policy old": "old_logp is null",
    "policy work": "workspace is too small", "policy logp over old": "overlap", "policy empty": None,
    "grad": None, "grad infinite": None, "grad max": "max_norm", "grad max nan": "max_norm", "grad type": "tensor 1: unknown type",
    "grad null": "tensor 2: g is null", "grad aligned": "tensor 0: g is not aligned", "grad large": "2^38", "grad work": "workspace is too small",
    "grad work aligned": "workspace is not aligned", "grad factor null": "factor is null", "grad norm is factor": "overlap", "grad scale": None,
    "grad scale is factor": "overlap", "grad descending": None, "grad twice": None, "grad in place": None, "grad in place unsaid": None,
    "grad in place twice": None, "grad out over another": None, "grad norm in a tensor": "overlap", "grad empty tensor": None, "grad none": None,
    "clip": None, "clip infinite": None, "clip max": "max_norm", "clip max nan": "max_norm", "clip type": "tensor 1: unknown type",
    "clip null": "tensor 2: g is null", "clip aligned": "tensor 0: g is not aligned", "clip large": "2^38", "clip work": "workspace is too small",
    "clip work aligned": "workspace is not aligned", "clip factor null": "factor is null", "clip norm is factor": "overlap", "clip scale": None,
    "clip scale is factor": "overlap", "clip descending": None, "clip twice": "overlap", "clip in place": None, "clip in place unsaid": None,
    "clip in place twice": "overlap", "clip out over another": "overlap", "clip norm in a tensor": "overlap", "clip empty tensor": None,
    "clip none": None, "grad no table": "tensors is null",
    "handle join": None, "handle join back": None, "handle preference": None, "handle policy": None, "handle grad": None, "handle clip": None,
}


@pytest.fixture(scope="module")
def said(tmp_path_factory):
    if not os.path.exists(B.LIB_PATH):
        build.build()
    exe = str(tmp_path_factory.mktemp("probe") / "step_checks_probe")
    lib_dir = os.path.dirname(B.LIB_PATH)
    subprocess.run(["g++"] + build.CXX_FLAGS + [os.path.join(ROOT, "tests", "step_checks_probe.cc"), "-o", exe, f"-L{lib_dir}", "-lsee_cuda",
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
    assert B.join_backward_workspace(0, 16) > 0 and B.join_backward_workspace(10, 0) == 0 and B.join_backward_workspace(10, 20000) == 0
    assert B.join_backward_workspace(10, 64) == 10 * 64 * 16 and B.join_backward_workspace(1 << 20, 64) == B.join_backward_workspace(4096, 64)
    assert B.preference_workspace(100, 0) == 0 and B.preference_workspace(1 << 31, 1) == 0
    assert B.preference_workspace(100, 3) == 100 * 16 + 32 and B.preference_workspace(0, 1) == 16
    assert B.policy_workspace(100) == B.policy_workspace(0) + 1600 and B.policy_workspace(1 << 31) == 0
    assert B.grad_workspace() > 0
