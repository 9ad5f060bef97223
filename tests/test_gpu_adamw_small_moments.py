"""AdamW with 8-bit moments where second moments lie below the smallest normal number: their roots, and what the weights move by."""

import numpy as np
import pytest
import torch

from see_ai_b200 import backend as B

pytestmark = pytest.mark.gpu

LR, BETA1, BETA2, EPS = 1e-3, 0.9, 0.999, 1e-30


@pytest.mark.parametrize("offset", [0, 1])   # through the ring, and where the operands lie
def test_roots_of_subnormal_second_moments(offset):
    be = B.CudaBackend(0)
    be.set_stream(torch.cuda.current_stream().cuda_stream)
    n = 4 * 256 + 7
    g = torch.zeros(n + offset, device="cuda")[offset:]
    g[:256] = torch.logspace(-21, -17, 256, device="cuda")    # second moments from 1e-45 to 1e-37
    g[256:512] = 1e-20
    g[512:768] = torch.logspace(-20, -3, 256, device="cuda")  # beside ordinary ones
    g[768:1024:3] = 3e-19                                     # and beside none
    g[1024:] = -2e-19
    p = torch.zeros(n + offset, device="cuda")[offset:]
    m, v = (torch.zeros(n + offset, device="cuda", dtype=torch.uint8)[offset:] for _ in range(2))
    ms, vs = torch.zeros(5, device="cuda"), torch.zeros(5, device="cuda")
    table = B.adamw_tensors([dict(p=p.data_ptr(), g=g.data_ptr(), m=m.data_ptr(), v=v.data_ptr(), m_scale=ms.data_ptr(), v_scale=vs.data_ptr(), n=n)])
    be.adamw_step(table, B.StepParams(LR, BETA1, BETA2, EPS, 0.0, 0, 1), state_bits=8)
    f = lambda x: float(np.float32(x))  # noqa: E731
    gd = g.double()
    m64, v64 = (1 - f(BETA1)) * gd, (1 - f(BETA2)) * gd * gd
    want = -f(LR) * (m64 / (1 - f(BETA1))) / ((v64 / (1 - f(BETA2))).sqrt() + f(EPS))
    # A second moment is a multiple of 2^-149: off by half of that, of which the root keeps half.  Step 1's corrections, rounded
    # to f32, are off by 2^-24 / (1 - beta2) = 1000 * 2^-24; the roots, quotients and products by a few 2^-22.
    off = 0.5 * 2.0 ** -150 / v64.clamp(min=1e-300) + 1100 * 2.0 ** -24
    seen = v64 >= 2.0 ** -145   # (below, the roundings leave little of the moment)
    assert seen.sum() > 700
    assert ((p.double() - want).abs() <= want.abs() * off * 1.01 + 1e-30)[seen].all()
    assert (p[gd == 0] == 0).all()
    # The blocks' scales: the largest root on 448.
    root = v64.sqrt()
    largest = torch.nn.functional.pad(root, (0, 5 * 256 - n)).view(5, 256).amax(1)
    least = torch.nn.functional.pad(v64, (0, 5 * 256 - n)).view(5, 256).amax(1)
    assert ((vs.double() - largest / 448).abs() <= (8 * 2.0 ** -24 + 0.5 * 2.0 ** -150 / least) * 1.01 * largest / 448).all()
    torch.cuda.synchronize()
    be.close()
