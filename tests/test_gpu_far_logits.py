"""Losses over rows whose largest logit is far from 0: classes masked with large negative numbers or the type's lowest value, all of them or
all but some, and rows of large positive ones.  What is equal to the largest shares the row; the rest has no chance, or, where logits next to
one another are some units apart, the chance that the formula gives it.  Tolerances are logit_reference's."""

import math

import pytest
import torch

import logit_reference as R
from see_ai_b200 import backend as B
from test_gpu_policy_loss import Policy
from test_gpu_preference_loss import Preference

pytestmark = pytest.mark.gpu

FAR = {"f32": [-5e7, -1e8, 2e8, -1e9, -3e9, -1e10, -1e20, -1e30, -1e37, 3e9, 1e10, 1e25, 1e37, "lowest"],
       "bf16": [-1e8, 3e8, -1e9, -3e9, -1e10, -1e20, -1e37, 1e10, 1e37, "lowest"],
       "f16": [-60000.0, 60000.0, "lowest"]}


@pytest.fixture(scope="module")
def be():
    b = B.CudaBackend(0)
    b.set_stream(torch.cuda.current_stream().cuda_stream)
    yield b
    torch.cuda.synchronize()
    b.close()


def values(dtype):
    return [torch.finfo(R.DTYPES[dtype]).min if v == "lowest" else v for v in FAR[dtype]]


def fill(c):
    """Row by row: all classes at a far value; some of them, among them the label, above others; ordinary ones with far ones in between, and
    with a run of far ones at their end, as a vocabulary is padded."""
    rows, classes = c.logits.shape
    far = values(c.dtype)
    for r in range(rows):
        kind, v = r % 4, far[r // 4 % len(far)]
        label = int(c.labels[r]) if 0 <= int(c.labels[r]) < classes else 0
        if kind == 0:
            c.logits[r] = v
        elif kind == 1:
            c.logits[r] = v if v < 0 else v / 4
            keep = torch.rand(classes, device="cuda") < 0.4
            keep[label] = True
            c.logits[r, keep] = v if v > 0 else v / 4
        else:
            z = float(c.logits[r, label])
            if kind == 2:
                c.logits[r, torch.rand(classes, device="cuda") < 0.5] = -abs(v)
            else:
                c.logits[r, classes // 3:] = -abs(v)
            c.logits[r, label] = z
    return c


SIZES = [(70, 250), (1300, 250), (1250, 1003), (66, 5003), (33, 32000), (33, 50001), (9, 128003)]


@pytest.mark.parametrize("dtype", list(R.DTYPES))
@pytest.mark.parametrize("rows,classes", SIZES + [(9, 300001), (3, 1 << 20)])
def test_policy(be, rows, classes, dtype):
    c = fill(Policy(rows, classes, dtype, seed=21, kl=0.0))
    c.reference = R.Rows(c.logits, c.labels)
    c.old = (c.reference.logp - 0.1).float()
    kept = c.logits.clone()
    c(be)
    c.check(c.d)
    assert torch.equal(c.logits, kept)
    want = c.d.clone()
    c(be, "in place")
    assert torch.equal(c.logits, want)


@pytest.mark.parametrize("dtype", list(R.DTYPES))
@pytest.mark.parametrize("lengths,classes", [([20, 30, 9, 12], 250), ([700, 601], 251), ([40, 33], 5003), ([33, 40], 32000), ([200, 170], 50001),
                                             ([11, 20], 128003)])
def test_preference(be, lengths, classes, dtype):
    c = Preference(lengths, classes, dtype, seed=22, reference=False)
    outside = c.logits[c.outside].clone()
    fill(c)
    inside = torch.where(c.outside, -1, c.labels)
    c.reference = R.Rows(c.logits, inside)
    c.logits[c.outside] = outside
    c(be)
    c.check(c.d)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("scale", [2.0 ** -90, 0.3, 1.0, 1.9, 1000.0])
def test_scaled(be, dtype, scale):
    """Logits up to 2^125 / scale."""
    for rows, classes in ((60, 250), (1300, 250), (40, 5003)):
        c = Policy(rows, classes, dtype, seed=23, kl=0.0, scale=scale)
        top = min(2.0 ** 125 / scale, torch.finfo(R.DTYPES[dtype]).max)
        for r in range(rows):
            v = math.copysign(top ** (0.3 + 0.7 * (r % 12 + 1) / 12), r % 2 - 0.5)
            c.logits[r] = v
            c.logits[r, ::2] = v if r % 3 else v - abs(v) / 2
        c.labels = (torch.arange(rows, device="cuda", dtype=torch.int32) * 2 + 1) % (classes - 1) | 1
        c.reference = R.Rows(c.logits, c.labels, scale)
        c.old = (c.reference.logp - 0.1).float()
        c.a, c.w = torch.randn(rows, device="cuda"), torch.rand(rows, device="cuda")
        c(be)
        c.check(c.d)


@pytest.mark.parametrize("dtype", list(R.DTYPES))
def test_labels_without_a_chance(be, dtype):
    """logp of a label far below the largest logit; infinities and NaN beside far values."""
    for rows, classes in ((1300, 250), (30, 5003)):
        c = Policy(rows, classes, dtype, seed=24, kl=0.0)
        top = 60000.0 if dtype == "f16" else 1e12
        c.labels = torch.arange(rows, device="cuda", dtype=torch.int32) % classes
        c.logits.copy_(torch.randn(rows, classes, device="cuda"))
        c.logits[:, 0] = top
        c.logits[1, int(c.labels[1])] = -top
        c.logits[2, int(c.labels[2])] = -math.inf
        c.logits[3, 5] = math.nan
        c.logits[4, 7] = math.inf
        c(be, None)
        want = torch.log_softmax(c.logits.double(), 1).gather(1, c.labels.long()[:, None])[:, 0]
        assert c.logp[2] == -math.inf and torch.isnan(c.logp[3:5]).all()
        rest = torch.ones(rows, device="cuda", dtype=torch.bool)
        rest[2:5] = False
        assert ((c.logp.double() - want).abs() <= 4 * R.ULP * want.abs())[rest].all()


@pytest.mark.parametrize("scale", [1.0, 1e-3, 0.25])
@pytest.mark.parametrize("rows,classes", [(1300, 250), (64, 250), (64, 5003), (9, 128003), (9, 300001)])
def test_neighbours(be, rows, classes, scale):
    """Rows of one far value and the three f32 numbers below it."""
    at = [v / scale for v in (1.2e7, -4e7, 5e7, -1e8, 2e8, 7e8, -7.5e8, 1.4e9, -3e9)]

    def fill(logits):
        for r in range(rows):
            steps = [torch.tensor(at[r % len(at)], dtype=torch.float32)]
            for _ in range(3):
                steps.append(torch.nextafter(steps[-1], torch.tensor(-math.inf)))
            logits[r] = torch.stack(steps).cuda()[(torch.arange(classes, device="cuda") * 7 + r) % 4]

    c = Policy(rows, classes, "f32", seed=26, kl=0.0, scale=scale)
    fill(c.logits)
    c.labels = torch.randint(classes, (rows,), device="cuda", dtype=torch.int32)
    c.reference = R.Rows(c.logits, c.labels, scale)
    c.old = (c.reference.logp - 0.1).float()
    c.a, c.w = torch.randn(rows, device="cuda"), torch.rand(rows, device="cuda")
    c(be)
    c.check(c.d)
    half = rows // 2
    q = Preference([half, rows - half], classes, "f32", seed=27, reference=False, scale=scale, behind=0)
    fill(q.logits)
    q.reference = R.Rows(q.logits, q.labels, scale)
    q(be)
    q.check(q.d)


@pytest.mark.parametrize("dtype", list(R.DTYPES))
@pytest.mark.parametrize("rows,classes,stride,begin,d_begin", [(1300, 250, 251, 3, 3), (60, 250, 251, 1, 2), (40, 5003, 5011, 5, 0), (9, 32000, 33001, 7, 7),
                                                              (9, 128003, 128003, 1, 5)])
def test_strides_and_alignments(be, rows, classes, stride, begin, d_begin, dtype):
    c = fill(Policy(rows, classes, dtype, seed=28, kl=0.0, stride=stride, begin=begin, d_begin=d_begin))
    c.reference = R.Rows(c.logits, c.labels)
    c.old = (c.reference.logp - 0.1).float()
    before = c.buf.clone()
    c(be)
    c.check(c.d)
    assert torch.equal(c.buf, before)
    c.d[:] = 9.0
    assert (c.d_buf == 9).all()
