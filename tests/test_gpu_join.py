"""A block's join to the residual stream, forward and backward with the weights' gradients, against the formulas in 64 bits and against
differences.

Tolerances count roundings of f32 (2^-24 each, relative) along the longest chain of a result, and half a step of the output type.  A sum
over a row is a chain of at most 32 additions in a thread and 21 between threads, 64 with the terms' own roundings; what multiplies it is
the sum of the terms' magnitudes.  What a stage is off is carried through the next one by its formula."""

import pytest
import torch

from see_ai_b200 import backend as B

pytestmark = pytest.mark.gpu

ULP = 2.0 ** -24
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
PAIRS = [("f32", "f32"), ("f32", "bf16"), ("f32", "f16"), ("bf16", "bf16"), ("f16", "f16")]


@pytest.fixture(scope="module")
def be():
    b = B.CudaBackend(0)
    b.set_stream(torch.cuda.current_stream().cuda_stream)
    yield b
    torch.cuda.synchronize()
    b.close()


def ptr(t):
    return 0 if t is None else t.data_ptr()


def rounding(dtype, value):
    if dtype == torch.float32:
        return ULP * value.abs() + 2.0 ** -149
    f = torch.finfo(dtype)
    return f.eps / 2 * value.abs() + f.smallest_normal * f.eps / 2


def strided(rows, cols, dtype, stride, begin=0):
    buf = torch.full((begin + rows * stride,), -3.0, device="cuda", dtype=dtype)
    return buf[begin:].view(rows, stride)[:, :cols], buf


class Join:
    def __init__(self, kind, rows, cols, xt, yt, post=True, gate=True, scale=0.9, x_stride=0, y_stride=0, begin=0, seed=0, eps=1e-5, dx_out=True):
        torch.manual_seed(seed * 1000 + rows * 31 + cols)
        self.kind, self.layer, self.rows, self.cols, self.xt, self.yt, self.eps, self.scale = kind, kind == B.NORM_LAYER, rows, cols, xt, yt, eps, scale
        self.post, self.x_stride, self.y_stride = post, x_stride or cols, y_stride or cols
        new_x = lambda: strided(rows, cols, DTYPES[xt], self.x_stride, begin)  # noqa: E731
        new_y = lambda: strided(rows, cols, DTYPES[yt], self.y_stride, begin)  # noqa: E731
        (self.x, _), (self.block, _), (self.x_out, self.x_buf), (self.y, self.y_buf) = new_x(), new_y(), new_x(), new_y()
        (self.dy, _), (self.dx_out, _), (self.dx, self.dx_buf), (self.dblock, self.db_buf) = new_y(), new_x(), new_x(), new_y()
        rand = lambda *s: torch.randn(*s, device="cuda")  # noqa: E731
        self.x.copy_(rand(rows, cols) * 2 + 0.5)
        self.block.copy_(rand(rows, cols) * torch.exp(0.3 * rand(cols)) + 0.3)
        self.dy.copy_(rand(rows, cols))
        self.dx_out.copy_(rand(rows, cols))
        if not dx_out:
            self.dx_out = None
        vector = lambda there, v: v if there else None  # noqa: E731
        self.w = dict(pre_gamma=1 + 0.1 * rand(cols), pre_beta=vector(self.layer, rand(cols)), gate=vector(gate, 0.5 + 0.3 * rand(cols)),
                      post_gamma=vector(post, 1 + 0.1 * rand(cols)), post_beta=vector(post and self.layer, rand(cols)))
        full = lambda n: torch.full((n,), 7.0, device="cuda")  # noqa: E731
        self.g = {k: None if v is None else full(cols) for k, v in self.w.items()}
        self.stats = dict(pre_rstd=full(rows), pre_mean=vector(self.layer, full(rows)), post_rstd=vector(post, full(rows)),
                          post_mean=vector(post and self.layer, full(rows)))
        self.work = torch.full((B.join_backward_workspace(rows, cols),), 0xFF, device="cuda", dtype=torch.uint8)   # (NaNs)
        self.types = dict(x_type=B.TYPES[xt], y_type=B.TYPES[yt], residual_scale=scale, x_stride=self.x_stride, y_stride=self.y_stride)

    def table(self, tensors, make):
        return make(**{k: ptr(v) for k, v in tensors.items()})

    def forward(self, be):
        be.join_forward(self.kind, self.rows, self.cols, ptr(self.x), ptr(self.block), self.table(self.w, B.join_weights), ptr(self.x_out),
                        ptr(self.y), self.table(self.stats, B.join_stats), eps=self.eps, **self.types)

    def backward(self, be):
        be.join_backward(self.kind, self.rows, self.cols, ptr(self.dy), ptr(self.dx_out), ptr(self.x_out), ptr(self.block),
                         self.table(self.w, B.join_weights), self.table(self.stats, B.join_stats), ptr(self.dx), ptr(self.dblock),
                         self.table(self.g, B.join_weights), ptr(self.work), self.work.numel(), **self.types)

    def wide(self, name):
        return None if self.w[name] is None else self.w[name].double()

    def norm(self, v, off, gamma, beta):
        """N(v), what it may be off, and mean and rstd with theirs; v is off by `off`."""
        n = self.cols
        m = v.mean(1, keepdim=True) if self.layer else torch.zeros_like(v[:, :1])
        reach = v.abs().amax(1, keepdim=True) if self.layer else torch.zeros_like(m)
        d = v - m
        r = (d.square().sum(1, keepdim=True) / n + self.eps).rsqrt()
        off_mean = (2 * ULP * m.abs() + 64 * ULP * d.abs().mean(1, keepdim=True) + off.mean(1, keepdim=True)) if self.layer else torch.zeros_like(m)
        off_var = 64 * ULP * d.square().mean(1, keepdim=True) + off_mean.square() + 2 * ULP * reach * d.abs().mean(1, keepdim=True) + \
            2 * (d.abs() * (off + off_mean)).mean(1, keepdim=True)
        off_r = 4 * ULP + 0.5 * off_var * r.square()
        want = d * r * gamma + (0.0 if beta is None else beta)
        allowed = (d * r * gamma).abs() * (off_r + 4 * ULP) + (off + off_mean + 2 * ULP * reach) * r * gamma.abs() + 2 * ULP * want.abs()
        return want, allowed, (m[:, 0], (off_mean + 4 * ULP * ULP * reach)[:, 0]), (r[:, 0], (off_r * r)[:, 0])

    def formula(self):
        u, off = self.block.double(), torch.zeros(self.rows, self.cols, device="cuda", dtype=torch.float64)
        kept = {}
        if self.post:
            u, off, kept["post_mean"], kept["post_rstd"] = self.norm(u, off, self.wide("post_gamma"), self.wide("post_beta"))
        if self.w["gate"] is not None:
            u, off = u * self.wide("gate"), off * self.wide("gate").abs()
        scaled = float(torch.tensor(self.scale, dtype=torch.float32)) * self.x.double()
        x_out, off = scaled + u, off + 3 * ULP * (scaled.abs() + u.abs())
        y, off_y, kept["pre_mean"], kept["pre_rstd"] = self.norm(x_out, off, self.wide("pre_gamma"), self.wide("pre_beta"))
        return (x_out, off), (y, off_y), kept

    def check_forward(self):
        (x_out, off), (y, off_y), kept = self.formula()
        for got, want, allowed in ((self.x_out, x_out, off), (self.y, y, off_y)):
            ok = (got.double() - want).abs() <= allowed * 1.001 + rounding(got.dtype, want.abs() + allowed)
            assert ok.all(), float(((got.double() - want).abs() / (allowed + rounding(got.dtype, want))).max())
        for name, t in self.stats.items():
            if t is not None:
                want, allowed = kept[name]
                assert ((t.double() - want).abs() <= allowed + ULP * want.abs()).all(), name

    def check_backward(self):
        column = lambda name: self.stats[name].double()[:, None]  # noqa: E731
        mean = lambda t: t.mean(1, keepdim=True)  # noqa: E731
        zero = torch.zeros(1, 1, device="cuda", dtype=torch.float64)

        def through(q, e, unit, r):
            """The gradient through a norm of q, which is off by e."""
            shift = mean(q) if self.layer else zero
            want = r * (q - shift - unit * mean(q * unit))
            size = q.abs() + (mean(q.abs()) if self.layer else zero) + unit.abs() * mean((q * unit).abs())
            return want, r * (e + mean(e) + unit.abs() * mean(e * unit.abs()) + 64 * ULP * size)

        dy, r2 = self.dy.double(), column("pre_rstd")
        unit2 = (self.x_out.double() - (column("pre_mean") if self.layer else zero)) * r2
        d, off = through(dy * self.wide("pre_gamma"), torch.zeros_like(dy), unit2, r2)
        if self.dx_out is not None:
            d = d + self.dx_out.double()
        off = off + 2 * ULP * d.abs()
        scale = float(torch.tensor(self.scale, dtype=torch.float32))
        close = lambda got, want, allowed: ((got.double() - want).abs() <= allowed * 1.001 + rounding(got.dtype, want.abs() + allowed)).all()  # noqa: E731
        assert close(self.dx, scale * d, abs(scale) * (off + ULP * d.abs()))
        unit1, r1 = self.block.double(), torch.ones_like(r2)
        if self.post:
            r1 = column("post_rstd")
            unit1 = (unit1 - (column("post_mean") if self.layer else zero)) * r1
        gate = self.wide("gate") if self.w["gate"] is not None else torch.ones(self.cols, device="cuda", dtype=torch.float64)
        by = gate * (self.wide("post_gamma") if self.post else 1.0)
        want, allowed = d * by, off * by.abs() + 3 * ULP * (d * by).abs()
        if self.post:
            want, allowed = through(want, allowed, unit1, r1)
        assert close(self.dblock, want, allowed)
        # A thread's rows (one row a block at the least), 16 groups, 10 + 5 in the fold, a term's own roundings.
        chain = (self.rows / 148 + 1) + 35
        total = lambda t, e, other: ((t * other).sum(0), (e * other.abs() + chain * ULP * (t * other).abs()).sum(0))  # noqa: E731
        one = torch.ones_like(dy)
        p1, p2 = total(dy, torch.zeros_like(dy), unit2), total(dy, torch.zeros_like(dy), one)
        s1, s2 = total(d, off, unit1), total(d, off, one)
        want = dict(pre_gamma=p1, pre_beta=p2)
        scaled = lambda s, by: (s[0] * by, s[1] * by.abs() + 2 * ULP * (s[0] * by).abs())  # noqa: E731
        if self.post:
            want.update(post_gamma=scaled(s1, gate), post_beta=scaled(s2, gate))
            a, b = scaled(s1, self.wide("post_gamma")), scaled(s2, self.wide("post_beta")) if self.layer else (0.0, 0.0)
            want["gate"] = (a[0] + b[0], a[1] + b[1] + 2 * ULP * (a[0] + b[0]).abs())
        else:
            want["gate"] = s1
        for name, got in self.g.items():
            if got is not None:
                assert ((got.double() - want[name][0]).abs() <= want[name][1] + ULP * want[name][0].abs()).all(), name


SIZES = [(1, 1), (1, 768), (3, 7), (17, 33), (257, 256), (64, 1000), (33, 1029), (5, 4096), (9, 4104), (2, 8200), (3, 12001), (2, 16384), (1, 16383),
         (700, 64), (5000, 64), (1500, 256), (2500, 768), (1300, 1000), (700, 1544), (400, 4096), (301, 8192), (1700, 3), (950, 55), (800, 333),
         (700, 1029), (350, 5003)]


@pytest.mark.parametrize("xt,yt", PAIRS)
@pytest.mark.parametrize("kind", [B.NORM_LAYER, B.NORM_RMS])
@pytest.mark.parametrize("rows,cols", SIZES)
def test_formula(be, kind, rows, cols, xt, yt):
    j = Join(kind, rows, cols, xt, yt)
    j.forward(be)
    j.check_forward()
    j.backward(be)
    j.check_backward()


@pytest.mark.parametrize("kind", [B.NORM_LAYER, B.NORM_RMS])
@pytest.mark.parametrize("post,gate,scale,dx_out", [(True, False, 1.0, True), (False, True, 0.5, True), (False, False, 1.0, False), (True, True, 0.0, False),
                                                    (True, False, -1.5, False)])
@pytest.mark.parametrize("rows,cols", [(4, 9), (40, 768), (700, 768), (130, 1029), (1400, 256), (33, 4096), (2, 12008)])
def test_parts(be, rows, cols, post, gate, scale, dx_out, kind):
    for xt, yt in PAIRS:
        j = Join(kind, rows, cols, xt, yt, post=post, gate=gate, scale=scale, dx_out=dx_out, seed=1)
        j.forward(be)
        j.check_forward()
        j.backward(be)
        j.check_backward()


@pytest.mark.parametrize("x_stride,y_stride,begin", [(1024, 1032, 0), (771, 769, 0), (1024, 800, 1), (2048, 768, 8), (768, 776, 4)])
@pytest.mark.parametrize("rows", [5, 1500])
def test_strided_rows_and_odd_addresses(be, rows, x_stride, y_stride, begin):
    """Rows inside wider buffers; what lies between them stays."""
    for kind, (xt, yt) in ((B.NORM_LAYER, PAIRS[3]), (B.NORM_RMS, PAIRS[1]), (B.NORM_RMS, PAIRS[4])):
        j = Join(kind, rows, 768, xt, yt, x_stride=x_stride, y_stride=y_stride, begin=begin, seed=2)
        j.forward(be)
        j.check_forward()
        j.backward(be)
        j.check_backward()
        for t, buf in ((j.x_out, j.x_buf), (j.y, j.y_buf), (j.dx, j.dx_buf), (j.dblock, j.db_buf)):
            t.fill_(-3.0)
            assert (buf == -3.0).all()


def test_rows_far_from_zero(be):
    """A mean a thousand times the spread, and rows without any spread."""
    for rows in (50, 2000):
        j = Join(B.NORM_LAYER, rows, 1024, "f32", "f32", scale=1.0)
        j.x += 1000.0
        j.block -= 500.0
        j.block[7], j.x[7] = 3.0, 5.0
        j.forward(be)
        j.check_forward()


def test_what_is_not_finite_stays_in_its_row(be):
    for rows in (8, 1500):
        for kind in (B.NORM_LAYER, B.NORM_RMS):
            j = Join(kind, rows, 304, "f32", "bf16")
            j.x[2, 5], j.block[4, 299], j.x[6, 0] = float("nan"), float("nan"), float("nan")
            j.forward(be)
            bad = torch.zeros(rows, device="cuda", dtype=torch.bool)
            bad[[2, 4, 6]] = True
            assert torch.isnan(j.y[bad]).all() and torch.isfinite(j.y[~bad]).all() and torch.isfinite(j.x_out[~bad]).all()
            j.backward(be)
            assert torch.isfinite(j.dx[~bad]).all() and torch.isfinite(j.dblock[~bad]).all() and torch.isnan(j.dx[bad]).all()


def test_no_rows(be):
    cols = 16
    w = {k: torch.ones(cols, device="cuda") for k in ("post_gamma", "post_beta", "gate", "pre_gamma", "pre_beta")}
    g = {k: torch.ones(cols, device="cuda") for k in w}
    work = torch.empty(B.join_backward_workspace(0, cols), device="cuda", dtype=torch.uint8)
    weights, grads = (B.join_weights(**{k: ptr(v) for k, v in t.items()}) for t in (w, g))
    be.join_forward(B.NORM_LAYER, 0, cols, 0, 0, weights, 0, 0, B.join_stats(0))
    be.join_backward(B.NORM_LAYER, 0, cols, 0, 0, 0, 0, weights, B.join_stats(0), 0, 0, grads, ptr(work), work.numel())
    assert all((v == 0).all() for v in g.values())


def test_as_the_norm_alone(be):
    """Without a gate and a norm after the block, of zeros that join: the norm operator's results."""
    for kind in (B.NORM_LAYER, B.NORM_RMS):
        j = Join(kind, 300, 768, "f32", "bf16", post=False, gate=False, scale=1.0)
        j.block.zero_()
        j.forward(be)
        j.backward(be)
        y, mean, rstd = torch.empty_like(j.y), torch.empty(300, device="cuda"), torch.empty(300, device="cuda")
        be.norm_forward(kind, 300, 768, ptr(j.x), ptr(j.w["pre_gamma"]), ptr(j.w["pre_beta"]), ptr(y), ptr(mean) if j.layer else 0, ptr(rstd),
                        y_type=B.BF16)
        assert torch.equal(j.x_out, j.x) and (j.y.float() - y.float()).abs().max() <= 2.0 ** -7 * y.float().abs().max()


@pytest.mark.parametrize("kind", [B.NORM_LAYER, B.NORM_RMS])
def test_gradient_against_differences(be, kind):
    """<dy, y> + <dx_out, x_out> moved along random directions of every input, in 64 bits."""
    j = Join(kind, 6, 40, "f32", "f32", scale=0.8)
    j.forward(be)
    j.backward(be)
    inputs = dict(x=j.x, block=j.block, **{k: v for k, v in j.w.items() if v is not None})
    grads = dict(x=j.dx, block=j.dblock, **{k: v for k, v in j.g.items() if v is not None})

    def value(moved):
        norm = lambda v, gamma, beta: ((v - v.mean(1, keepdim=True)) if j.layer else v) * ((v - v.mean(1, keepdim=True) if j.layer else v).square()  # noqa: E731
                                                                                        .mean(1, keepdim=True) + j.eps).rsqrt() * gamma + (beta if beta is not None else 0.0)
        u = norm(moved["block"], moved["post_gamma"], moved.get("post_beta"))
        x_out = float(torch.tensor(0.8)) * moved["x"] + moved["gate"] * u
        y = norm(x_out, moved["pre_gamma"], moved.get("pre_beta"))
        return float((j.dy.double() * y).sum() + (j.dx_out.double() * x_out).sum())

    for name in inputs:
        torch.manual_seed(len(name))
        step = torch.randn(inputs[name].shape, device="cuda", dtype=torch.float64)
        values = []
        for eps in (1e-4, -1e-4):
            moved = {k: v.double() for k, v in inputs.items()}
            moved[name] = moved[name] + eps * step
            values.append(value(moved))
        slope, want = (values[0] - values[1]) / 2e-4, float((grads[name].double() * step).sum())
        # The third derivative's 1e-8 / 6 and f32's roundings (and x_out's, kept in f32) over 240 terms.
        assert abs(slope - want) <= 1e-5 * float((grads[name].double() * step).abs().sum()) + 1e-5, name


def test_same_bits_replayed_and_two_at_once(be):
    for rows, cols in ((40, 768), (1500, 768), (700, 1029)):
        make = lambda: Join(B.NORM_LAYER, rows, cols, "f32", "bf16", seed=5)  # noqa: E731
        outputs = lambda j: [j.x_out, j.y, j.dx, j.dblock] + [t for t in list(j.stats.values()) + list(j.g.values()) if t is not None]  # noqa: E731
        one, other = make(), make()
        one.forward(be)
        one.backward(be)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        try:
            with torch.cuda.graph(graph, stream=side):
                be.set_stream(side.cuda_stream)
                other.forward(be)
                other.backward(be)
        finally:
            be.set_stream(torch.cuda.current_stream().cuda_stream)
        for _ in range(3):
            for t in outputs(other):
                t.zero_()
            graph.replay()
            assert all(torch.equal(a, b) for a, b in zip(outputs(one), outputs(other)))
        torch.cuda.synchronize()
        pair = [(B.CudaBackend(0), make()) for _ in range(2)]
        torch.cuda.synchronize()
        for _ in range(5):
            for b, j in pair:
                j.forward(b)
                j.backward(b)
        torch.cuda.synchronize()
        for b, j in pair:
            assert all(torch.equal(a, b) for a, b in zip(outputs(one), outputs(j)))
            b.close()
