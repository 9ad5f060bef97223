"""Layer norm and root-mean-square norm with the weights' gradients, against the formulas in 64 bits.

Tolerances count roundings of f32 (2^-24 each, relative) along the longest chain of a result, and half a step of the output
type, finfo.eps / 2 of the value.  A sum over n terms is a chain of at most ceil(n / threads) additions in a thread (32 at
most) and a dozen between threads; what multiplies it is the sum of the terms' magnitudes.
"""

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


def rounding(t, value):
    """Half a step of type t around `value`, its smallest step included."""
    if t == "f32":
        return ULP * value.abs()
    f = torch.finfo(DTYPES[t])
    return f.eps / 2 * value.abs() + f.smallest_normal * f.eps / 2


def matrix(rows, cols, dtype, stride, fill):
    buf = torch.full((rows, stride), fill, device="cuda", dtype=dtype)
    return buf, buf[:, :cols]


def forward(be, kind, x, gamma, beta, eps, yt, y=None):
    rows, cols = x.shape
    layer = kind == B.NORM_LAYER
    xt = {v: k for k, v in DTYPES.items()}[x.dtype]
    if y is None:
        y = torch.empty(rows, cols, device="cuda", dtype=DTYPES[yt])
    mean = torch.full((rows,), 7.0, device="cuda") if layer else None
    rstd = torch.full((rows,), 7.0, device="cuda")
    be.norm_forward(kind, rows, cols, ptr(x), ptr(gamma), ptr(beta) if layer else 0, ptr(y), ptr(mean), ptr(rstd),
                    x_type=B.TYPES[xt], y_type=B.TYPES[yt], eps=eps, x_stride=x.stride(0) if rows > 1 else 0,
                    y_stride=y.stride(0) if rows > 1 else 0)
    return y, mean, rstd


def check_forward(kind, x, gamma, beta, eps, yt, y, mean, rstd):
    xd, g = x.double(), gamma.double()
    if kind == B.NORM_LAYER:
        m = xd.mean(1, keepdim=True)
        reach = xd.abs().amax(1, keepdim=True)
        assert ((mean.double() - m[:, 0]).abs() <= 2 * ULP * m[:, 0].abs() + 64 * ULP * (xd - m).abs().mean(1) + 4 * ULP * ULP * reach[:, 0]).all()
    else:
        m, reach = torch.zeros_like(xd[:, :1]), torch.zeros_like(xd[:, :1])
    d = xd - m
    r = (d.square().mean(1, keepdim=True) + eps).rsqrt()
    # The variance: squares and their chain, half of which the root keeps; an f32 mean is off by ULP of itself.
    off_mean = 2 * ULP * m.abs() + 64 * ULP * d.abs().mean(1, keepdim=True)
    off_var = 64 * ULP * d.square().mean(1, keepdim=True) + off_mean.square() + 2 * ULP * reach * d.abs().mean(1, keepdim=True)
    off_r = 4 * ULP + 0.5 * off_var * r.square()
    assert ((rstd.double()[:, None] - r).abs() <= off_r * r).all()
    want = d * r * g + (beta.double() if kind == B.NORM_LAYER else 0.0)
    allowed = (d * r * g).abs() * (off_r + 4 * ULP) + (off_mean + 2 * ULP * reach) * r * g.abs() + 2 * ULP * want.abs()
    assert ((y.double() - want).abs() <= allowed + rounding(yt, want) * 1.001).all()


@pytest.mark.parametrize("xt,yt", PAIRS)
@pytest.mark.parametrize("kind", [B.NORM_LAYER, B.NORM_RMS])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 768), (3, 7), (17, 33), (257, 256), (64, 1000), (33, 1029), (5, 4096), (9, 4104),
                                       (2, 8200), (3, 12001), (2, 16384), (1, 16383), (700, 64), (5000, 64), (4800, 256),
                                       (5001, 768), (7100, 1000), (4737, 1024), (2500, 1544), (1200, 4096), (700, 8192), (9600, 1), (9500, 3),
                                       (9501, 55), (6000, 333), (2400, 1029), (700, 5003), (593, 8191)])
def test_forward(be, kind, rows, cols, xt, yt):
    torch.manual_seed(rows * 31 + cols)
    x = (torch.randn(rows, cols, device="cuda") * 2 + 0.5).to(DTYPES[xt])
    gamma, beta = 1 + 0.1 * torch.randn(cols, device="cuda"), torch.randn(cols, device="cuda")
    y, mean, rstd = forward(be, kind, x, gamma, beta, 1e-5, yt)
    check_forward(kind, x, gamma, beta, 1e-5, yt, y, mean, rstd)


def backward(be, kind, dy, x, gamma, mean, rstd, addend, dx=None):
    rows, cols = x.shape
    layer = kind == B.NORM_LAYER
    names = {v: k for k, v in DTYPES.items()}
    if dx is None:
        dx = torch.empty(rows, cols, device="cuda", dtype=x.dtype)
    dgamma = torch.full((cols,), 7.0, device="cuda")
    dbeta = torch.full((cols,), 7.0, device="cuda") if layer else None
    work = torch.empty(B.norm_backward_workspace(rows, cols), device="cuda", dtype=torch.uint8)
    be.norm_backward(kind, rows, cols, ptr(dy), ptr(x), ptr(gamma), ptr(mean) if layer else 0, ptr(rstd), ptr(dx), ptr(dgamma),
                     ptr(dbeta), ptr(work), work.numel(), addend=ptr(addend), x_type=B.TYPES[names[x.dtype]],
                     y_type=B.TYPES[names[dy.dtype]], x_stride=x.stride(0) if rows > 1 else 0,
                     y_stride=dy.stride(0) if rows > 1 else 0)
    return dx, dgamma, dbeta


def check_backward(kind, dy, x, gamma, mean, rstd, addend, dx, dgamma, dbeta):
    names = {v: k for k, v in DTYPES.items()}
    rows = x.shape[0]
    layer = kind == B.NORM_LAYER
    d, r = dy.double(), rstd.double()[:, None]
    u = (x.double() - (mean.double()[:, None] if layer else 0.0)) * r
    q = d * gamma.double()
    mq, mqu = (q.mean(1, keepdim=True) if layer else torch.zeros_like(r)), (q * u).mean(1, keepdim=True)
    want = r * (q - mq - u * mqu) + (addend.double() if addend is not None else 0.0)
    size = r * (q.abs() + q.abs().mean(1, keepdim=True) + u.abs() * (q * u).abs().mean(1, keepdim=True))
    assert ((dx.double() - want).abs() <= 64 * ULP * size + ULP * want.abs() + rounding(names[x.dtype], want) * 1.001).all()
    # A thread's rows (at most rows / 148 + 1 with one row a block), 16 groups, 10 + 5 in the fold, 4 roundings a term.
    chain = (rows / 148 + 1) + 35
    assert ((dgamma.double() - (d * u).sum(0)).abs() <= chain * ULP * (d * u).abs().sum(0)).all()
    if layer:
        assert ((dbeta.double() - d.sum(0)).abs() <= chain * ULP * d.abs().sum(0)).all()


def stats(kind, x, eps=1e-5):
    xd = x.double()
    m = xd.mean(1) if kind == B.NORM_LAYER else torch.zeros_like(xd[:, 0])
    return m.float(), ((xd - m[:, None]).square().mean(1) + eps).rsqrt().float()


@pytest.mark.parametrize("xt,yt", PAIRS)
@pytest.mark.parametrize("kind", [B.NORM_LAYER, B.NORM_RMS])
@pytest.mark.parametrize("rows,cols,add", [(1, 1, True), (1, 768, False), (3, 7, True), (17, 33, False), (2500, 256, True),
                                           (4097, 768, True), (640, 1000, True), (777, 1029, True), (333, 4096, False),
                                           (9, 4104, True), (20, 8200, False), (3, 12001, True), (302, 16384, True),
                                           (155, 16383, False), (700, 64, False), (9600, 1, True), (9500, 3, False),
                                           (9501, 55, True), (6000, 333, True), (2400, 1029, False), (700, 5003, True), (593, 8191, True)])
def test_backward(be, kind, rows, cols, add, xt, yt):
    torch.manual_seed(rows * 31 + cols)
    x = (torch.randn(rows, cols, device="cuda") * 2 + 0.5).to(DTYPES[xt])
    dy = torch.randn(rows, cols, device="cuda").to(DTYPES[yt])
    addend = torch.randn(rows, cols, device="cuda").to(DTYPES[xt]) if add else None
    gamma = 1 + 0.1 * torch.randn(cols, device="cuda")
    mean, rstd = stats(kind, x)
    out = backward(be, kind, dy, x, gamma, mean, rstd, addend)
    check_backward(kind, dy, x, gamma, mean, rstd, addend, *out)
    again = backward(be, kind, dy, x, gamma, mean, rstd, addend)
    assert all(a is None or torch.equal(a, b) for a, b in zip(out, again))


def test_gradients_against_differences(be):
    """(L(w + h) - L(w - h)) / 2h of L = sum(y dy), in 64 bits, against the kernel's gradients: the difference quotient is
    off by h^2 times third derivatives, far below the f32 tolerance here."""
    torch.manual_seed(3)
    rows, cols, eps, h = 3, 40, 1e-5, 1e-5
    x, dy = torch.randn(rows, cols, device="cuda"), torch.randn(rows, cols, device="cuda")
    gamma, beta = torch.rand(cols, device="cuda") + 0.5, torch.randn(cols, device="cuda")
    for kind in (B.NORM_LAYER, B.NORM_RMS):
        def loss(x, gamma, beta):
            d = x - x.mean(1, keepdim=True) if kind == B.NORM_LAYER else x
            y = d * (d.square().mean(1, keepdim=True) + eps).rsqrt() * gamma + (beta if kind == B.NORM_LAYER else 0.0)
            return (y * dy.double()).sum()

        mean, rstd = stats(kind, x, eps)
        dx, dgamma, dbeta = backward(be, kind, dy, x, gamma, mean, rstd, None)
        at = [x.double(), gamma.double(), beta.double()]
        for k, got in enumerate((dx, dgamma, dbeta)):
            if got is None:
                continue
            for i in range(0, got.numel(), 7):
                step = torch.zeros_like(at[k])
                step.view(-1)[i] = h
                plus, minus = list(at), list(at)
                plus[k], minus[k] = at[k] + step, at[k] - step
                want = (loss(*plus) - loss(*minus)) / (2 * h)
                assert abs(got.view(-1)[i].item() - want.item()) <= 1e-4


@pytest.mark.parametrize("x_stride,y_stride,offset", [(1024, 1032, 0), (771, 769, 0), (1024, 800, 1), (2048, 768, 8)])
def test_strided_rows_and_odd_addresses(be, x_stride, y_stride, offset):
    """Rows inside wider buffers; what lies between them stays."""
    torch.manual_seed(5)
    rows, cols = 37, 768
    def strided(dtype, stride, value):
        buf = torch.full((rows * stride + offset,), value, device="cuda", dtype=dtype)
        return buf, buf[offset:].view(rows, stride)[:, :cols] if stride >= cols else None
    _, x = strided(torch.bfloat16, x_stride, 1.0)
    x.copy_(torch.randn(rows, cols))
    ybuf, y = strided(torch.bfloat16, y_stride, -3.0)
    gamma, beta = 1 + 0.1 * torch.randn(cols, device="cuda"), torch.randn(cols, device="cuda")
    y, mean, rstd = forward(be, B.NORM_LAYER, x, gamma, beta, 1e-5, "bf16", y)
    check_forward(B.NORM_LAYER, x, gamma, beta, 1e-5, "bf16", y, mean, rstd)
    kept = ybuf.clone()
    y.fill_(-3.0)
    assert (ybuf == -3.0).all() and not (kept == -3.0).all()
    y.copy_(torch.randn(rows, cols))
    dxbuf, dx = strided(torch.bfloat16, x_stride, -3.0)
    dx, dgamma, dbeta = backward(be, B.NORM_LAYER, y, x, gamma, mean, rstd, None, dx)
    check_backward(B.NORM_LAYER, y, x, gamma, mean, rstd, None, dx, dgamma, dbeta)
    dx.fill_(-3.0)
    assert (dxbuf == -3.0).all()


def test_rows_far_from_zero(be):
    """A mean a thousand times the spread: deviations keep f32 accuracy."""
    torch.manual_seed(6)
    x = torch.randn(50, 1024, device="cuda") + 1000.0
    x[7] = 5.0            # no spread at all
    gamma, beta = torch.ones(1024, device="cuda"), torch.zeros(1024, device="cuda")
    y, mean, rstd = forward(be, B.NORM_LAYER, x, gamma, beta, 1e-5, "f32")
    check_forward(B.NORM_LAYER, x, gamma, beta, 1e-5, "f32", y, mean, rstd)
    assert (y[7] == 0).all()


def test_what_is_not_finite_stays_in_its_row(be):
    x = torch.randn(8, 300, device="cuda")
    x[2, 5], x[4, 299], x[6, 0] = float("nan"), float("inf"), -float("inf")
    gamma, beta = torch.ones(300, device="cuda"), torch.zeros(300, device="cuda")
    y, mean, rstd = forward(be, B.NORM_LAYER, x, gamma, beta, 1e-5, "f32")
    bad = torch.tensor([False, False, True, False, True, False, True, False], device="cuda")
    assert torch.isnan(y[bad]).all() and torch.isfinite(y[~bad]).all()
    y, _, rstd = forward(be, B.NORM_RMS, x, gamma, beta, 1e-5, "f32")
    assert torch.isfinite(y[~bad]).all() and torch.isnan(y[2]).all() and torch.isnan(y[4, 299]) and (y[4, :299] == 0).all()


def test_no_rows(be):
    gamma = torch.ones(16, device="cuda")
    dummy = torch.empty(16, device="cuda")
    be.norm_forward(B.NORM_RMS, 0, 16, ptr(dummy), ptr(gamma), 0, ptr(torch.empty(16, device="cuda")), 0, ptr(torch.empty(16, device="cuda")))
    dgamma, dbeta = torch.ones(16, device="cuda"), torch.ones(16, device="cuda")
    work = torch.empty(B.norm_backward_workspace(0, 16), device="cuda", dtype=torch.uint8)
    be.norm_backward(B.NORM_LAYER, 0, 16, ptr(dummy), ptr(dummy), ptr(gamma), ptr(dummy), ptr(dummy), ptr(torch.empty(16, device="cuda")),
                     ptr(dgamma), ptr(dbeta), ptr(work), work.numel())
    assert (dgamma == 0).all() and (dbeta == 0).all()


def test_captured_and_replayed_on_another_stream(be):
    torch.manual_seed(8)
    rows, cols = 300, 512
    x, dy = torch.randn(rows, cols, device="cuda"), torch.randn(rows, cols, device="cuda")
    gamma = torch.ones(cols, device="cuda")
    mean, rstd = stats(B.NORM_LAYER, x)
    want = backward(be, B.NORM_LAYER, dy, x, gamma, mean, rstd, None)
    out = [torch.zeros_like(w) for w in want]
    work = torch.empty(B.norm_backward_workspace(rows, cols), device="cuda", dtype=torch.uint8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    try:
        with torch.cuda.graph(graph, stream=side):
            be.set_stream(side.cuda_stream)
            be.norm_backward(B.NORM_LAYER, rows, cols, ptr(dy), ptr(x), ptr(gamma), ptr(mean), ptr(rstd), *(ptr(o) for o in out),
                             ptr(work), work.numel())
    finally:
        be.set_stream(torch.cuda.current_stream().cuda_stream)
    for _ in range(2):
        for o in out:
            o.zero_()
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.parametrize("cols,x_stride,y_stride,offset", [(33, 37, 41, 1), (3, 3, 5, 1), (250, 251, 250, 3)])
def test_odd_rows_in_wider_buffers(be, cols, x_stride, y_stride, offset):
    """Many rows of odd widths, strides and addresses: copied with what lies beside them, which neither shows nor changes."""
    torch.manual_seed(9)
    rows = 9601
    def strided(stride, value):
        buf = torch.full(((rows - 1) * stride + cols + offset,), value, device="cuda", dtype=torch.bfloat16)
        return buf, torch.as_strided(buf, (rows, cols), (stride, 1), offset)
    xbuf, x = strided(x_stride, float("nan"))
    x.copy_(torch.randn(rows, cols))
    _, dy = strided(y_stride, float("nan"))
    dy.copy_(torch.randn(rows, cols))
    _, add = strided(x_stride, float("nan"))
    add.copy_(torch.randn(rows, cols))
    dxbuf, dx = strided(x_stride, -3.0)
    gamma = 1 + 0.1 * torch.randn(cols, device="cuda")
    mean, rstd = stats(B.NORM_LAYER, x)
    out = backward(be, B.NORM_LAYER, dy, x, gamma, mean, rstd, add, dx)
    check_backward(B.NORM_LAYER, dy, x, gamma, mean, rstd, add, *out)
    dx.fill_(-3.0)
    assert (dxbuf == -3.0).all()
    ybuf, y = strided(y_stride, -3.0)
    beta = torch.randn(cols, device="cuda")
    check_forward(B.NORM_LAYER, x, gamma, beta, 1e-5, "bf16", *forward(be, B.NORM_LAYER, x, gamma, beta, 1e-5, "bf16", y))
    y.fill_(-3.0)
    assert (ybuf == -3.0).all()
