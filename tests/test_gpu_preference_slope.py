"""The preference losses where little of a pair's slope is left, and in place over far rows.  Tolerances are logit_reference's."""

import math

import pytest
import torch

import logit_reference as R
import test_gpu_far_logits as F
from see_ai_b200 import backend as B
from test_gpu_preference_loss import Preference

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be():
    b = B.CudaBackend(0)
    b.set_stream(torch.cuda.current_stream().cuda_stream)
    yield b
    torch.cuda.synchronize()
    b.close()


@pytest.mark.parametrize("dtype", list(R.DTYPES))
@pytest.mark.parametrize("smoothing", [0.01, 0.1, 0.3])
@pytest.mark.parametrize("left", [1e-3, -1e-5, 1e-6])
def test_what_smoothing_leaves(be, left, smoothing, dtype):
    """One pair of rows whose labels are all but certain, so that their log-probabilities have digits to spare; h is where `left` remains."""
    c = Preference([9, 7], 250, dtype, smoothing=smoothing, reference=False)
    z = 0.5 * torch.randn(c.rows, 250, device="cuda")
    c.labels = torch.randint(250, (c.rows,), device="cuda", dtype=torch.int32)
    z.scatter_(1, c.labels.long()[:, None], 24.0)
    c.logits.copy_(z)
    c.reference = R.Rows(c.logits, torch.where(c.outside, -1, c.labels))
    s, beta = float(torch.tensor(smoothing, dtype=torch.float32)), float(torch.tensor(0.1, dtype=torch.float32))
    chance = s - left   # sigmoid(-h)
    h = math.log((1 - chance) / chance)
    c.ref = torch.tensor([-h / beta, 0.0], device="cuda")
    w = c.want()
    assert 0.5 * abs(left) < abs(float(w["slopes"][0])) * 1 / beta < 2 * abs(left) + 1e-6
    c(be)
    c.check(c.d)


@pytest.mark.parametrize("dtype", list(R.DTYPES))
@pytest.mark.parametrize("lengths,classes", [([20, 30, 9, 12], 250), ([700, 601], 251), ([40, 33], 5003), ([200, 170], 50001)])
def test_far_rows_in_place(be, lengths, classes, dtype):
    c = F.fill(Preference(lengths, classes, dtype, seed=25, reference=False))
    c(be)
    want, inside = [t.clone() for t in (c.d, c.loss, c.sums)], ~c.outside
    kept = c.logits[c.outside].clone()
    c(be, "in place")
    assert torch.equal(c.logits[inside], want[0][inside]) and torch.equal(c.loss, want[1]) and torch.equal(c.sums, want[2])
    assert torch.equal(c.logits[c.outside].nan_to_num(7.0), kept.nan_to_num(7.0))
