"""Layer norm of rows whose mean is far larger than their spread, at sizes that reach each forward kernel: a row's mean, rstd and
result do not depend on how many rows there are.

An f32 sum of a thread's at most 32 values leaves the mean off by c, up to 33 * 2^-24 of it; the deviations of such rows are exact
differences, their squares' average lies c^2 above the variance, and c is known from the deviations' own average.  What is left of
either is the roundings of a chain of 64 terms of that size.
"""

import pytest
import torch

from see_ai_b200 import backend as B

pytestmark = pytest.mark.gpu

ULP = 2.0 ** -24
EPS = 1e-5


@pytest.fixture(scope="module")
def be():
    b = B.CudaBackend(0)
    b.set_stream(torch.cuda.current_stream().cuda_stream)
    yield b
    torch.cuda.synchronize()
    b.close()


@pytest.mark.parametrize("rows,cols", [(12, 768), (12, 1029), (12, 5000), (5001, 64), (5001, 256), (5001, 768), (4800, 1000), (1300, 4096), (700, 8192),
                                       (9600, 55), (6000, 333), (2400, 1029)])
def test_rows_with_little_or_no_spread(be, rows, cols):
    torch.manual_seed(cols)
    centre = torch.tensor([3000.7, 10000.1, 65000.7, -10000.1, 0.3, 20000.3], device="cuda")[torch.arange(rows, device="cuda") % 6]
    x = centre[:, None].repeat(1, cols)
    step = torch.nextafter(x, torch.full_like(x, 1e9)) - x
    spread = (torch.arange(rows, device="cuda") // 6 % 2 == 1)[:, None]   # every other six: two neighbours, of which the mean lies between
    x = x + step * (torch.rand(rows, cols, device="cuda") < 0.5) * spread
    gamma, beta = torch.ones(cols, device="cuda"), torch.zeros(cols, device="cuda")
    y, mean, rstd = torch.empty_like(x), torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    be.norm_forward(B.NORM_LAYER, rows, cols, x.data_ptr(), gamma.data_ptr(), beta.data_ptr(), y.data_ptr(), mean.data_ptr(), rstd.data_ptr(),
                    eps=EPS)
    xd = x.double()
    m = xd.mean(1, keepdim=True)
    d = xd - m
    var, spread = d.square().mean(1), d.abs().mean(1)
    r = (var + EPS).rsqrt()
    c = 33 * ULP * m[:, 0].abs()
    off_var = 64 * ULP * (var + c * c) + 2 * c * 64 * ULP * (c + spread) + 64 * ULP * var
    off_r = 4 * ULP + 0.5 * off_var / (var + EPS)
    assert ((rstd.double() - r).abs() <= off_r * r * 1.01).all()
    # The mean: its own rounding, and the average of the deviations, whose chain is of terms of c.
    off_mean = ULP * m[:, 0].abs() + 64 * ULP * (c + spread)
    assert ((mean.double() - m[:, 0]).abs() <= off_mean * 1.01).all()
    want = d * r[:, None]
    assert ((y.double() - want).abs() <= want.abs() * (off_r + 4 * ULP)[:, None] + (off_mean * r)[:, None] * 1.01).all()
