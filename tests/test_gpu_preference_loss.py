"""The preference losses of paired sequences and the gradient of the logits, against the formulas in 64 bits and against differences.
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


class Preference:
    """lengths: of the sequences; `before` and `behind` rows belong to none; every fourth label does not count."""

    def __init__(self, lengths, classes, dtype, kind="sigmoid", beta=0.1, smoothing=0.0, margin=0.0, average=False, scale=1.0, before=0, behind=3,
                 stride=0, begin=0, d_begin=None, seed=0, reference=True):
        torch.manual_seed(seed * 1000 + sum(lengths) + classes)
        self.pairs, self.classes, self.dtype, self.kind = len(lengths) // 2, classes, dtype, kind
        self.options = dict(beta=beta, smoothing=smoothing, margin=margin, average=average)
        self.scale, self.stride = scale, stride or classes
        starts = [before]
        for n in lengths:
            starts.append(starts[-1] + n)
        self.rows = starts[-1] + behind
        self.starts = torch.tensor(starts, device="cuda", dtype=torch.int32)
        new = lambda at: torch.full((at + self.rows * self.stride + 64,), 9.0, device="cuda", dtype=DTYPES[dtype])  # noqa: E731
        view = lambda buf, at: buf[at:at + self.rows * self.stride].view(self.rows, self.stride)[:, :classes]  # noqa: E731
        d_begin = begin if d_begin is None else d_begin
        self.buf, self.d_buf = new(begin), new(d_begin)
        self.logits, self.d = view(self.buf, begin), view(self.d_buf, d_begin)
        self.labels = torch.randint(classes, (self.rows,), device="cuda", dtype=torch.int32)
        z = torch.randn(self.rows, classes, device="cuda") * 2
        z.scatter_add_(1, self.labels.long()[:, None], torch.rand(self.rows, 1, device="cuda") * math.log(classes + 1) * 1.6)
        self.logits.copy_(z)
        self.labels[2::4] = torch.tensor([-1, -100, classes], device="cuda", dtype=torch.int32).repeat(self.rows)[:self.labels[2::4].numel()]
        self.outside = torch.ones(self.rows, device="cuda", dtype=torch.bool)
        self.outside[before:starts[-1]] = False
        inside = torch.where(self.outside, -1, self.labels)
        self.reference = R.Rows(self.logits, inside, scale)
        self.ref = None
        if reference:
            sums = R.preference(self.reference, self.starts, None, "square", beta, 0.0, 0.0, average)["sums"]
            self.ref = (sums + torch.randn(2 * self.pairs).double() * (0.5 if average else 3.0)).float().cuda()
        self.logits[self.outside] = math.nan   # not read
        self.loss, self.margins, self.sums = (torch.full((n,), 7.0, device="cuda") for n in (1, self.pairs, 2 * self.pairs))
        self.work = torch.full((B.preference_workspace(self.rows, self.pairs),), 0xFF, device="cuda", dtype=torch.uint8)
        self.loss_grad = None

    def __call__(self, be, d="apart"):
        p = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
        d = {"apart": p(self.d), "in place": p(self.logits), None: 0}[d]
        be.preference_loss(self.rows, self.classes, self.pairs, p(self.logits), p(self.labels), p(self.starts), p(self.loss), p(self.margins),
                           p(self.sums), p(self.work), self.work.numel(), ref_logp=p(self.ref), loss_grad=p(self.loss_grad), dlogits=d,
                           type=B.TYPES[self.dtype], kind=B.PREFERENCES[self.kind], logit_scale=self.scale, stride=self.stride, **self.options)

    def want(self):
        return R.preference(self.reference, self.starts, self.ref, self.kind, **self.options)

    def check(self, d, loss_grad=1.0):
        w = self.want()
        assert ((self.sums.double().cpu() - w["sums"]).abs() <= w["sums_off"]).all()
        assert ((self.margins.double().cpu() - w["margins"]).abs() <= w["margins_off"]).all()
        assert abs(float(self.loss) - w["loss"]) <= w["loss_off"]
        if d is None:
            return
        outside = self.outside
        assert (d[outside] == 9).all()   # as they were
        d = torch.where(outside[:, None], 0.0, d)
        self.reference.check_dlogits(d, w["slopes"] * loss_grad, w["slopes_off"] * abs(loss_grad))


LISTS = {"shortest": [1, 1], "one empty": [0, 5], "both empty": [0, 0, 3, 4], "ragged": [3, 17, 40, 1, 9, 9], "long": [300, 211], "many": [2, 3] * 70}


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("classes", [1, 7, 33, 250, 5003, 32000])
@pytest.mark.parametrize("name", list(LISTS))
def test_formula(be, name, classes, dtype):
    c = Preference(LISTS[name], classes, dtype, before=2)
    c(be)
    c.check(c.d)
    outputs = [t.clone() for t in (c.loss, c.margins, c.sums)]
    for t in (c.loss, c.margins, c.sums):
        t.fill_(7.0)
    c(be, None)
    assert all(torch.equal(a, b) for a, b in zip(outputs, (c.loss, c.margins, c.sums)))
    inside = ~c.outside
    kept = c.d[inside].clone()
    c(be, "in place")
    assert torch.equal(c.logits[inside], kept) and torch.isnan(c.logits[c.outside]).all()


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("lengths,classes", [([3, 2], 128003), ([90, 70], 50001), ([1, 2], 300001), ([700, 900], 2000), ([160, 150], 70001),
                                             ([700, 600, 9, 0], 251), ([800, 500], 40)])
def test_wide_and_long(be, lengths, classes, dtype):
    c = Preference(lengths, classes, dtype, average=True)
    c(be)
    c.check(c.d)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("lengths,classes,stride,begin,d_begin", [([150, 170], 20000, 20000, 0, 0), ([40, 60] * 4, 20011, 20013, 3, 3),
                                                                 ([301, 0, 1, 20], 33001, 33001, 5, 2), ([0, 310], 20481, 20488, 7, 7),
                                                                 ([200, 220], 45056, 45056, 1, 1)])
def test_many_wide_rows(be, lengths, classes, stride, begin, d_begin, dtype):
    """Rows that single warps' rings walk, where a block lists those that count: chunks of 256 units that end beside a row's end, too."""
    c = Preference(lengths, classes, dtype, before=5, stride=stride, begin=begin, d_begin=d_begin)
    c(be)
    c.check(c.d)
    outputs = [t.clone() for t in (c.loss, c.margins, c.sums)]
    c(be, None)
    assert all(torch.equal(a, b) for a, b in zip(outputs, (c.loss, c.margins, c.sums)))
    c.d[:] = 9.0
    assert (c.d_buf == 9).all()


def test_many_wide_rows_of_which_none_counts(be):
    c = Preference([200, 200], 20000, "bf16", reference=False)
    c.labels.fill_(-1)
    c.logits.fill_(math.nan)
    c(be)
    assert (c.sums == 0).all() and (c.margins == 0).all() and abs(float(c.loss) - math.log(2)) < 1e-6
    assert (c.d[:400] == 0).all()


def test_rows_that_count_far_apart(be):
    """More rows than are counted at a time, most of which do not count and hold NaN: the same as those that count alone.  A row's
    log-probability is the same there; their sums in double are in another order, and each output is rounded once to f32."""
    few = Preference([230, 170], 20000, "bf16", behind=0)
    few(be)
    few.check(few.d)
    rows, split = 33100, 16500
    logits = torch.full((rows, 20000), math.nan, device="cuda", dtype=torch.bfloat16)
    labels = torch.full((rows,), -1, device="cuda", dtype=torch.int32)
    generator = torch.Generator().manual_seed(1)
    at = torch.cat([torch.randperm(split, generator=generator)[:230].sort().values,
                    split + torch.randperm(rows - split, generator=generator)[:170].sort().values])
    at[-1], at[0] = rows - 1, 0
    at = at.cuda()
    logits[at], labels[at] = few.logits, few.labels
    starts = torch.tensor([0, split, rows], device="cuda", dtype=torch.int32)
    loss, margins, sums = (torch.full((n,), 7.0, device="cuda") for n in (1, 1, 2))
    work = torch.full((B.preference_workspace(rows, 1),), 0xFF, device="cuda", dtype=torch.uint8)
    be.preference_loss(rows, 20000, 1, logits.data_ptr(), labels.data_ptr(), starts.data_ptr(), loss.data_ptr(), margins.data_ptr(), sums.data_ptr(),
                       work.data_ptr(), work.numel(), ref_logp=few.ref.data_ptr(), type=B.TYPES["bf16"], kind=B.PREFERENCES["sigmoid"], **few.options)
    for got, want in ((loss, few.loss), (margins, few.margins), (sums, few.sums)):
        assert ((got - want).abs() <= 2.0 ** -23 * want.abs() + 1e-12).all()


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("lengths,classes", [([700, 10], 2000), ([9, 600], 20000), ([1500, 3], 250)])
def test_what_is_off_alike_does_not_add_up(be, lengths, classes, dtype):
    """A margin of many rows against few.  A row's log-probability is off by a rounding or two of its sum, 2^-24 each, in either direction:
    6e-9 on the average of 500 rows and more.  ex2.approx's average is known to 1e-9.  3e-8 leaves room for neither's 2^-24 in one direction."""
    c = Preference(lengths, classes, dtype, beta=0.1)
    c(be)
    want = float(c.want()["margins"])
    assert abs(float(c.margins) - want) <= 0.1 * sum(lengths) * 3e-8 + 2.0 ** -24 * abs(want)


OPTIONS = [dict(kind="sigmoid", smoothing=0.1), dict(kind="sigmoid", margin=0.5, average=True), dict(kind="hinge"), dict(kind="hinge", margin=-0.4, average=True),
           dict(kind="square"), dict(kind="square", beta=2.0, average=True), dict(reference=False, beta=0.01), dict(reference=False, average=True, beta=2.0),
           dict(scale=0.7), dict(scale=1.6)]


@pytest.mark.parametrize("options", OPTIONS)
def test_options(be, options):
    for dtype in DTYPES:
        c = Preference(LISTS["ragged"], 1003, dtype, seed=1, **options)
        c(be)
        c.check(c.d)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("classes,stride,begin,d_begin", [(33, 40, 8, 8), (33, 37, 3, 3), (250, 251, 1, 2), (5003, 5011, 5, 0), (32000, 32008, 8, 1),
                                                         (50001, 50001, 7, 7), (3, 5, 2, 1)])
def test_strides_and_alignments(be, classes, stride, begin, d_begin, dtype):
    c = Preference([4, 7, 2, 5], classes, dtype, stride=stride, begin=begin, d_begin=d_begin)
    c(be)
    c.check(c.d)
    c.d[:] = 9.0
    assert (c.d_buf == 9).all()


def test_loss_scale(be):
    c = Preference([30, 41], 777, "f16")
    c.loss_grad = torch.full((1,), 512.0, device="cuda")
    c(be)
    c.check(c.d, 512.0)


def test_large_margins(be):
    """Far from the corner a sigmoid's loss is the margin or next to nothing, and neither overflows."""
    c = Preference([20, 20, 20, 20], 300, "f32", beta=1.0)
    c.ref += torch.tensor([3000.0, 0.0, -3000.0, 0.0], device="cuda")
    c(be)
    c.check(c.d)
    assert abs(float(c.loss) - 1500.0) < 20 and (c.d[40:60] == 0).all()


def test_no_rows_and_nothing_that_counts(be):
    c = Preference([0, 0], 100, "f32", behind=0, reference=False)
    c(be)
    assert float(c.loss) == pytest.approx(math.log(2.0), rel=1e-6) and (c.sums == 0).all() and (c.margins == 0).all()
    c = Preference([4, 6], 100, "bf16", average=True, reference=False)
    c.labels.fill_(-1)
    c.logits.fill_(math.nan)
    c(be)
    assert (c.sums == 0).all() and (c.d[:10] == 0).all() and (c.d[10:] == 9).all()


@pytest.mark.parametrize("kind", list(B.PREFERENCES))
def test_what_is_not_a_number_stays_in_its_pair(be, kind):
    c = Preference([5, 6, 7, 8], 300, "bf16", kind=kind)
    c.logits[1, 5] = math.nan
    c(be)
    counted = c.reference.counts
    assert torch.isnan(c.loss).all() and torch.isnan(c.margins[0]) and torch.isfinite(c.margins[1])
    assert torch.isnan(c.d[:11][counted[:11]]).all() and torch.isfinite(c.d[11:26]).all()


def test_starts_outside_the_rows(be):
    """Row numbers outside the matrix lead nowhere."""
    c = Preference([4, 4], 64, "f32", behind=0, reference=False)
    c.starts.copy_(torch.tensor([-5, 4, 1000], device="cuda", dtype=torch.int32))
    c(be)
    assert torch.isfinite(c.d).all() and torch.isfinite(c.loss).all()


@pytest.mark.parametrize("kind", list(B.PREFERENCES))
def test_gradient_against_differences(be, kind):
    c = Preference([4, 5, 3, 6], 40, "f32", kind=kind, beta=0.3, seed=5, behind=0)
    c(be)
    grad, base = c.d.double().clone(), c.logits.clone()
    for seed in range(4):
        torch.manual_seed(seed)
        step = torch.randn_like(base).double()
        losses = []
        for eps in (1e-3, -1e-3):
            rows = R.Rows(base.double() + eps * step, c.labels)
            losses.append(R.preference(rows, c.starts, c.ref, kind, **c.options)["loss"])
        slope, want = (losses[0] - losses[1]) / 2e-3, float((grad * step).sum())
        # Third derivatives of 18 rows' logp (of a size of 1) and of the square in them, times 1e-6 / 6; the gradient's own roundings.
        assert abs(slope - want) <= 1e-4 * (1 + abs(want))


@pytest.mark.parametrize("lengths,classes", [([100, 90, 3, 50], 5003), ([4, 3], 128003), ([700, 650], 250), ([160, 150], 50001)])
def test_same_bits_replayed_and_two_at_once(be, lengths, classes):
    c = Preference(lengths, classes, "bf16", seed=7)
    c(be)
    inside = ~c.outside
    want = c.d.clone(), c.loss.clone(), c.sums.clone()
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
        c.d[inside] = 0.0
        graph.replay()
        assert torch.equal(c.d, want[0]) and torch.equal(c.loss, want[1]) and torch.equal(c.sums, want[2])
    torch.cuda.synchronize()
    others = [(B.CudaBackend(0), Preference(lengths, classes, "bf16", seed=7)) for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        for b, o in others:
            o(b)
    torch.cuda.synchronize()
    for b, o in others:
        assert torch.equal(o.d, want[0]) and torch.equal(o.loss, want[1])
        b.close()
