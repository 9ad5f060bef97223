"""The policy loss where little decides much: ratios at a corner of the clip, policies next to their reference, ratios beyond f32.

Tolerances are logit_reference's, but for two that are narrower or wider there:
- kl = exp(x) - x - 1 of an x that is off by `off`: |exp(x) - 1| off, and 4 roundings of f32 of kl itself (its own, the weight's product,
  the sum's, the result's).  No term in |x|: that would be the digits lost by a subtraction in f32.
- the slope of 16-bit logits may be off by 2^-15 of itself, a sixteenth of f16's half step."""

import math

import pytest
import torch

import logit_reference as R
from see_ai_b200 import backend as B
from test_gpu_policy_loss import Policy

pytestmark = pytest.mark.gpu

# A warp's rows, a group's, a cluster's, streams (f32's and 16 bits').
SIZES = [(1300, 250), (1190, 1003), (200, 5003), (160, 32000), (5, 128003), (2, 300001), (2, 1 << 20)]


@pytest.fixture(scope="module")
def be():
    b = B.CudaBackend(0)
    b.set_stream(torch.cuda.current_stream().cuda_stream)
    yield b
    torch.cuda.synchronize()
    b.close()


def formula(c):
    """R.policy's, at any ratio that is not within what logp may be off of a corner; and with what 16-bit slopes may be off."""
    want = R.policy(c.reference, c.old, c.ref, c.a, c.w, *c.clip, c.kl)
    if c.ref is not None:
        x = torch.where(c.reference.counts, c.ref.double() - c.reference.logp, 0.0)
        off = c.reference.logp_off + 2.0 ** -50 * (c.reference.logp.abs() + x.abs())   # (a double difference)
        kl = torch.where(x.abs() < 1e-3, x * x * (0.5 + x / 6 + x * x / 24 + x ** 3 / 120), torch.expm1(x) - x)
        w = torch.where(c.reference.counts, c.w.double() if c.w is not None else 1.0, 0.0)
        want["kl"], want["kl_off"] = kl * w, (torch.expm1(x).abs() * off + 0.51 * off * off + 4 * R.ULP * kl) * w
    if c.dtype != "f32":
        want["slope_off"] = want["slope_off"] + 2.0 ** -15 * want["slope"].abs()
    return want


@pytest.mark.parametrize("dtype", list(R.DTYPES))
@pytest.mark.parametrize("rows,classes", SIZES)
@pytest.mark.parametrize("clip", [(0.0, 0.0), (0.2, 0.28)])
def test_rows_without_a_gradient_are_those_counted_as_clipped(be, rows, classes, dtype, clip):
    """old_logp of the operator itself, moved to the corners: which side of them a ratio lies on is a rounding's choice, but one."""
    c = Policy(rows, classes, dtype, clip=clip, kl=0.0, weighted=False)
    c(be, None)
    corner = torch.tensor([math.log(1 - clip[0]), math.log(1 + clip[1])], device="cuda")
    c.old = c.logp - corner[torch.arange(rows, device="cuda") % 2] * (1 + 1e-6 * torch.randn(rows, device="cuda"))
    c.a = torch.where(torch.rand(rows, device="cuda") < 0.5, -1.0, 1.0)
    c(be)
    still = (c.d == 0).all(1) & c.reference.counts
    assert float(c.loss[2]) == int(still.sum())


def certain(rows, classes, dtype, lead, seed, **options):
    """Labels that lead by `lead`: their log-probability, next to 0, has digits far below f32's of 1."""
    c = Policy(rows, classes, dtype, seed=seed, spread=0.5, **options)
    z = 0.5 * torch.randn(rows, classes, device="cuda")
    c.labels = torch.randint(classes, (rows,), device="cuda", dtype=torch.int32)
    z.scatter_(1, c.labels.long()[:, None], lead)
    c.logits.copy_(z)
    c.reference = R.Rows(c.logits, c.labels, c.scale)
    c.old = (c.reference.logp + 0.1 * torch.sign(torch.randn(rows, device="cuda"))).float()
    c.a, c.w = torch.randn(rows, device="cuda"), torch.rand(rows, device="cuda") if c.w is not None else None
    return c


def near_reference(c, least, most):
    rows = c.rows
    x = torch.exp(torch.rand(rows, device="cuda") * (math.log(most) - math.log(least)) + math.log(least)) * torch.sign(torch.randn(rows, device="cuda"))
    c.ref = (c.reference.logp + x).float()


@pytest.mark.parametrize("dtype", list(R.DTYPES))
@pytest.mark.parametrize("advantage", ["none", "cancels", "some"])
@pytest.mark.parametrize("rows,classes", [(1300, 250), (33, 250), (200, 5003), (5, 128003)])
def test_gradient_next_to_the_reference(be, rows, classes, dtype, advantage):
    c = certain(rows, classes, dtype, 16.0, 11, kl=0.5)
    near_reference(c, 1e-6, 1e-2)
    if advantage == "none":
        c.a.zero_()
    elif advantage == "cancels":   # what the KL term leaves of the policy's
        x = c.ref.double() - c.reference.logp
        c.a = (-0.5 * torch.expm1(x) / torch.exp(c.reference.logp - c.old.double()) * 1.01).float()
    c(be)
    want = formula(c)
    c.reference.check_dlogits(c.d, want["slope"], want["slope_off"])


@pytest.mark.parametrize("dtype", list(R.DTYPES))
@pytest.mark.parametrize("rows", [1, 40, 3000])
@pytest.mark.parametrize("least,most", [(1e-9, 1e-6), (1e-5, 1e-2), (0.1, 3.0)])
def test_kl_keeps_its_digits(be, rows, dtype, least, most):
    c = certain(rows, 250, dtype, 24.0, 12, kl=0.5)
    near_reference(c, least, most)
    c(be, None)
    want = formula(c)
    total, off = float(want["kl"].sum()), float(want["kl_off"].sum())
    assert abs(float(c.loss[1]) - total) <= off and float(c.loss[1]) >= 0


@pytest.mark.parametrize("dtype", list(R.DTYPES))
@pytest.mark.parametrize("rows,classes", [(1300, 250), (33, 250), (200, 5003), (2, 300001)])
def test_ratios_beyond_f32_times_nothing(be, rows, classes, dtype):
    """exp(logp - old_logp) or exp(ref_logp - logp) overflows f32 where an advantage, a weight or kl_coef is 0: their terms are 0."""
    for what in ("advantages", "weights", "kl_coef", "weights of kl"):
        c = Policy(rows, classes, dtype, seed=13, kl=0.0 if what == "kl_coef" else 0.05)
        far = torch.arange(rows, device="cuda") % 2 == 0
        if what in ("advantages", "weights"):
            c.old = torch.where(far & c.reference.counts, -300.0, c.old)
            (c.a if what == "advantages" else c.w)[far] = 0.0
            c.a = torch.where(far, -c.a.abs(), c.a)   # (below 0: no clip takes them)
        else:
            c.ref = torch.where(far, 300.0, c.reference.logp.float())
            if what != "kl_coef":
                c.w[far] = 0.0
        c(be)
        want = formula(c)
        c.reference.check_dlogits(c.d, want["slope"], want["slope_off"])
        for i, key in enumerate(("loss", "kl", "clipped")):
            total = float(want[key].sum())
            if what == "kl_coef" and key == "kl":   # (beyond f32)
                assert float(c.loss[1]) == math.inf
                continue
            off = float(want[key + "_off"].sum()) if key != "clipped" else 0.0
            assert abs(float(c.loss[i]) - total) <= off + 2 * R.ULP * abs(total), (what, key)


@pytest.mark.parametrize("dtype", list(R.DTYPES))
def test_what_is_not_a_number_is_not_lost_in_a_weight_of_0(be, dtype):
    for rows, classes in ((1300, 250), (20, 5003)):
        c = Policy(rows, classes, dtype, seed=14)
        c.w.zero_()
        c.a.zero_()
        row = int(torch.nonzero(c.reference.counts)[3])
        c.logits[row, 7] = math.nan
        c(be)
        assert torch.isnan(c.loss[0]) and torch.isnan(c.d[row]).all()
        c.d[row] = 0.0
        assert (c.d == 0).all()
