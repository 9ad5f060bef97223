"""The clipped policy loss with its KL term and the gradient of the logits, against the formulas in 64 bits and against differences.
The tolerances are logit_reference's."""

import math

import pytest
import torch

import logit_reference as R
from see_ai_b200 import backend as B

pytestmark = pytest.mark.gpu

DTYPES = R.DTYPES


@pytest.fixture(scope="module")
def be():
    b = B.CudaBackend(0)
    b.set_stream(torch.cuda.current_stream().cuda_stream)
    yield b
    torch.cuda.synchronize()
    b.close()


def matrix(rows, cols, dtype, stride, begin=0):
    """A view of rows x cols that begins `begin` elements into a buffer, and the buffer."""
    buf = torch.full((begin + rows * stride + 64,), 9.0, device="cuda", dtype=dtype)
    return buf[begin:begin + rows * stride].view(rows, stride)[:, :cols], buf


class Policy:
    """Rows of a trained model's logits; every fifth label does not count."""

    def __init__(self, rows, classes, dtype, seed=0, stride=0, begin=0, d_begin=None, spread=2.0, clip=(0.2, 0.28), kl=0.05, scale=1.0, weighted=True):
        torch.manual_seed(seed * 1000 + rows + classes)
        self.rows, self.classes, self.clip, self.kl, self.scale = rows, classes, clip, kl, scale
        self.stride = stride or classes
        self.logits, self.buf = matrix(rows, classes, DTYPES[dtype], self.stride, begin)
        self.d, self.d_buf = matrix(rows, classes, DTYPES[dtype], self.stride, begin if d_begin is None else d_begin)
        self.labels = torch.randint(classes, (rows,), device="cuda", dtype=torch.int32)
        z = torch.randn(rows, classes, device="cuda") * spread
        z.scatter_add_(1, self.labels.long()[:, None], torch.rand(rows, 1, device="cuda") * math.log(classes + 1) * 1.6)
        self.logits.copy_(z)
        self.labels[3::5] = torch.tensor([-1, -100, classes, 2 ** 31 - 1], device="cuda", dtype=torch.int32).repeat(rows)[:self.labels[3::5].numel()]
        self.a = torch.randn(rows, device="cuda")
        self.w = torch.rand(rows, device="cuda") if weighted else None
        self.dtype = dtype
        self.loss = torch.full((3,), 7.0, device="cuda")
        self.logp = torch.full((rows,), 7.0, device="cuda")
        self.work = torch.full((B.policy_workspace(rows),), 0xFF, device="cuda", dtype=torch.uint8)
        self.loss_grad = None
        self.reference = R.Rows(self.logits, self.labels, scale)
        ratio = torch.exp(0.2 * torch.randn(rows, device="cuda")).double()
        for border in (1 - clip[0], 1 + clip[1]):
            ratio = torch.where((ratio - border).abs() < 1e-4, border + 2e-4, ratio)
        self.old = (self.reference.logp - ratio.log()).float()
        self.ref = (self.reference.logp + 0.3 * torch.randn(rows, device="cuda")).float() if kl else None
        for t in (self.old, self.ref, self.a, self.w):   # of rows that do not count nothing is read
            if t is not None:
                t[~self.reference.counts] = math.nan

    def __call__(self, be, d="apart"):
        p = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
        d = {"apart": p(self.d), "in place": p(self.logits), None: 0}[d]
        be.policy_loss(self.rows, self.classes, p(self.logits), p(self.labels), p(self.old), p(self.a), p(self.loss), p(self.logp), p(self.work),
                       self.work.numel(), ref_logp=p(self.ref), weights=p(self.w), loss_grad=p(self.loss_grad), dlogits=d, type=B.TYPES[self.dtype],
                       logit_scale=self.scale, clip_low=self.clip[0], clip_high=self.clip[1], kl_coef=self.kl, stride=self.stride)

    def check(self, d, loss_grad=1.0):
        want = R.policy(self.reference, self.old, self.ref, self.a, self.w, *self.clip, self.kl)
        self.reference.check_logp(self.logp)
        for got, key in zip(self.loss.tolist(), ("loss", "kl", "clipped")):
            total = float(want[key].sum())
            off = float(want[key + "_off"].sum()) if key != "clipped" else 0.0
            assert abs(got - total) <= off + 2 * R.ULP * abs(total), (key, got, total)
        if d is not None:
            self.reference.check_dlogits(d, want["slope"] * loss_grad, want["slope_off"] * abs(loss_grad))


SIZES = [(1, 1), (5, 2), (3, 7), (40, 8), (33, 33), (1, 250), (300, 250), (17, 1000), (9, 4096), (200, 5003), (1, 32000), (160, 32000), (3, 50001),
         (2, 128003), (155, 100000), (2, 300001), (1, 1 << 20),
         (1300, 1), (1500, 55), (2400, 250), (1190, 511), (1185, 1003)]


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,classes", SIZES)
def test_formula(be, rows, classes, dtype):
    c = Policy(rows, classes, dtype)
    before = c.buf.clone()
    c(be)
    c.check(c.d)
    assert torch.equal(c.buf, before)
    want = c.loss.clone(), c.logp.clone()
    c.loss.fill_(7.0)
    c(be, None)
    assert torch.equal(c.loss, want[0]) and torch.equal(c.logp, want[1])
    kept = c.d.clone()
    c(be, "in place")
    assert torch.equal(c.logits, kept) and torch.equal(c.loss, want[0])


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,classes,stride,begin,d_begin", [(7, 33, 40, 8, 8), (7, 33, 37, 3, 3), (50, 250, 251, 1, 2), (6, 5003, 5011, 5, 0),
                                                              (3, 32000, 32008, 8, 1), (5, 32000, 33001, 7, 7), (2, 128003, 128003, 1, 5),
                                                              (2, 300001, 300001, 3, 4), (4, 1, 1, 0, 0), (9, 3, 5, 2, 1), (1300, 250, 251, 3, 3),
                                                              (1300, 1003, 1016, 8, 1)])
def test_strides_and_alignments(be, rows, classes, stride, begin, d_begin, dtype):
    c = Policy(rows, classes, dtype, stride=stride, begin=begin, d_begin=d_begin)
    c(be)
    c.check(c.d)
    c.d[:] = 9.0
    assert (c.d_buf == 9).all()   # what lies around is as it was


@pytest.mark.parametrize("options", [dict(kl=0.0), dict(kl=0.0, weighted=False), dict(clip=(0.0, 0.0)), dict(clip=(1.0, 3.0)), dict(scale=0.7),
                                     dict(scale=1.6, spread=8.0), dict(spread=0.0)])
def test_options(be, options):
    for dtype in DTYPES:
        c = Policy(130, 1003, dtype, seed=2, **options)
        c(be)
        c.check(c.d)


def test_loss_scale(be):
    c = Policy(64, 777, "f16", seed=3)
    c.loss_grad = torch.full((1,), 1024.0, device="cuda")
    c(be)
    c.check(c.d, 1024.0)


def test_nothing_counts(be):
    for rows, classes in ((20, 300), (5, 32000)):
        c = Policy(rows, classes, "bf16")
        c.labels.fill_(-1)
        c.logits.fill_(math.nan)
        c(be)
        assert (c.d == 0).all() and (c.logp == 0).all() and (c.loss == 0).all()


def test_no_rows(be):
    loss = torch.full((3,), 7.0, device="cuda")
    work = torch.empty(B.policy_workspace(0), device="cuda", dtype=torch.uint8)
    be.policy_loss(0, 100, 0, 0, 0, 0, loss.data_ptr(), 0, work.data_ptr(), work.numel())
    assert (loss == 0).all()


def test_certain_labels_keep_their_digits(be):
    """A chance of 1 - 1e-9: logp and the label's gradient are what the others leave, not 0."""
    c = Policy(10, 4000, "f32", spread=0.5, kl=0.0)
    z = torch.randn(10, 4000, device="cuda")
    c.labels.copy_(torch.arange(10, device="cuda") * 400)
    z.scatter_(1, c.labels.long()[:, None], 30.0)
    c.logits.copy_(z)
    c.reference = R.Rows(c.logits, c.labels)
    c.old, c.a, c.w = c.reference.logp.float(), torch.randn(10, device="cuda"), torch.rand(10, device="cuda")
    c(be)
    assert (c.logp < 0).all()
    c.check(c.d)


def test_masked_classes(be):
    """Logits of -inf have no chance and no gradient; one class left: nothing to learn."""
    for dtype in DTYPES:
        c = Policy(40, 515, dtype, kl=0.0)
        keep = torch.rand(40, 515, device="cuda") < 0.3
        keep[0] = False
        keep.scatter_(1, c.labels.long().clamp(0, 514)[:, None], True)
        c.logits.copy_(torch.where(keep, c.logits, -math.inf))
        c.reference = R.Rows(c.logits, c.labels)
        c.old = (c.reference.logp - 0.05).float()
        c(be)
        c.check(c.d)
        assert (c.d[~keep] == 0).all() and (c.d[0] == 0).all()


def test_what_is_not_a_number_stays_in_its_row(be):
    for classes in (300, 32000):
        for bad in (math.nan, math.inf, "all"):
            c = Policy(12, classes, "bf16", kl=0.0)
            rows = [0, 5, 11]
            for r in rows:
                if bad == "all":
                    c.logits[r] = -math.inf
                else:
                    c.logits[r, (r * 7) % classes] = bad
                    c.logits[r, int(c.labels[r])] = bad if r == 5 else c.logits[r, int(c.labels[r])]
            c(be)
            assert torch.isnan(c.loss[0]) and torch.isnan(c.d[rows]).all() and torch.isnan(c.logp[rows]).all()
            rest = [r for r in range(12) if r not in rows]
            assert torch.isfinite(c.d[rest]).all()


def test_gradient_against_differences(be):
    """The loss of f32 logits, moved along random directions."""
    c = Policy(12, 50, "f32", seed=5, kl=0.1)
    c(be)
    grad, base = c.d.double().clone(), c.logits.clone()
    for seed in range(4):
        torch.manual_seed(seed)
        step = torch.randn_like(base)
        step[~c.reference.counts] = 0.0
        losses = []
        for eps in (1e-3, -1e-3):
            moved = base.double() + eps * step.double()
            c.logits.copy_(moved)
            rows = R.Rows(moved, c.labels)
            losses.append(float(R.policy(rows, c.old, c.ref, c.a, c.w, *c.clip, c.kl)["loss"].sum()))
            c(be, None)
            assert abs(float(c.loss[0]) - losses[-1]) <= 1e-5 * (1 + abs(losses[-1]))
        slope, want = (losses[0] - losses[1]) / 2e-3, float((grad * step).sum())
        # Third derivatives of 12 rows, each of a size of 1 to 10, times 1e-6 / 6; the gradient's own roundings.
        assert abs(slope - want) <= 1e-4 * (1 + abs(want))


@pytest.mark.parametrize("rows,classes", [(200, 5003), (3, 128003), (1300, 250), (400, 50001), (2, 300001)])
def test_same_bits_replayed_and_two_at_once(be, rows, classes):
    c = Policy(rows, classes, "bf16", seed=7)
    c(be)
    want = c.d.clone(), c.loss.clone(), c.logp.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    try:
        with torch.cuda.graph(graph, stream=side):
            be.set_stream(side.cuda_stream)
            c(be)
    finally:
        be.set_stream(torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        c.d.zero_()
        graph.replay()
        assert torch.equal(c.d, want[0]) and torch.equal(c.loss, want[1]) and torch.equal(c.logp, want[2])
    torch.cuda.synchronize()
    others = [(B.CudaBackend(0), Policy(rows, classes, "bf16", seed=7)) for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        for b, o in others:
            o(b)
    torch.cuda.synchronize()
    for b, o in others:
        assert torch.equal(o.d, want[0]) and torch.equal(o.loss, want[1])
        b.close()
