"""Many narrow rows, as a norm of each head has them, by the checks of the other widths."""

import pytest
import torch

from see_ai_b200 import backend as B
from test_gpu_norm import DTYPES, PAIRS, backward, check_backward, check_forward, forward, stats

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be():
    b = B.CudaBackend(0)
    b.set_stream(torch.cuda.current_stream().cuda_stream)
    yield b
    torch.cuda.synchronize()
    b.close()


@pytest.mark.parametrize("xt,yt", PAIRS)
@pytest.mark.parametrize("kind", [B.NORM_LAYER, B.NORM_RMS])
@pytest.mark.parametrize("rows,cols,stride", [(5001, 8, 8), (20001, 16, 16), (70000, 64, 64), (30001, 64, 192), (40000, 128, 128), (30000, 96, 104), (12000, 80, 81)])
def test_both_directions(be, kind, rows, cols, stride, xt, yt):
    torch.manual_seed(rows)
    wide = lambda t: torch.full((rows, stride), float("nan"), device="cuda", dtype=DTYPES[t])[:, :cols]  # noqa: E731
    x, dy, addend, y, dx = wide(xt), wide(yt), wide(xt), wide(yt), wide(xt)
    x.copy_(torch.randn(rows, cols, device="cuda") * 2 + 0.5)
    dy.copy_(torch.randn(rows, cols, device="cuda"))
    addend.copy_(torch.randn(rows, cols, device="cuda"))
    gamma, beta = 1 + 0.1 * torch.randn(cols, device="cuda"), torch.randn(cols, device="cuda")
    check_forward(kind, x, gamma, beta, 1e-5, yt, *forward(be, kind, x, gamma, beta, 1e-5, yt, y))
    mean, rstd = stats(kind, x)
    check_backward(kind, dy, x, gamma, mean, rstd, addend, *backward(be, kind, dy, x, gamma, mean, rstd, addend, dx))
