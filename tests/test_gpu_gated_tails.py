"""The gated block's activations far from zero, relative to their own size: negative gates, whose GELU and SiLU are small, and
gates that are not finite.

Each hidden column has a gate of its own and an up of one, exact in f32: one input column of ones times a row of gates.  With
2u the exponent's argument and s = 1 / (1 + E), E = e^-2u: E is off by the roundings of its argument, 7 of them and its
constants, times |2u|, and the hardware's 2^-22; s by (1 - s) of that, the sum's rounding and the reciprocal's 2^-23.  The value is
one product more, the slope's second term four.  Below 2^-126 the reciprocal is zero.
"""

import pytest
import torch

from see_ai_b200 import backend as B

pytestmark = pytest.mark.gpu

ULP = 2.0 ** -24
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
GELU_C, GELU_A = 0.7978845608028654, 0.044715
COLS = 4096


@pytest.fixture(scope="module")
def be():
    b = B.CudaBackend(0)
    b.set_stream(torch.cuda.current_stream().cuda_stream)
    yield b
    torch.cuda.synchronize()
    b.close()


def gates(t):
    g = torch.linspace(-13.0, 13.0, COLS, dtype=torch.float64)
    g[:64] = -torch.logspace(1, 4, 64, dtype=torch.float64)
    return g.to(t).cuda()


def exact(kind, g):
    """Value, slope, and how far each may be off before its rounding."""
    if kind == "silu":
        arg, inner = g, torch.ones_like(g)
    else:
        arg, inner = 2 * GELU_C * (g + GELU_A * g ** 3), 2 * GELU_C * (1 + 3 * GELU_A * g * g)
    s, rest = torch.sigmoid(arg), torch.sigmoid(-arg)
    off_e = (7 * arg.abs() + 4) * ULP
    off_s = rest * off_e + 4 * ULP
    value, tail = g * s, g * inner * s * rest
    least = 2.0 ** -126
    # (SiLU takes 1 - s as it stands: a rounding of s there is as large as one of its own)
    off_tail = tail.abs() * (2 * off_s + off_e + 6 * ULP) + (g.abs() * s * (off_s * s + ULP) if kind == "silu" else 0.0)
    return value, s + tail, value.abs() * (off_s + ULP) + g.abs() * least, s * (off_s + ULP) + off_tail + (1 + (g * inner).abs()) * least


def half_step(t, value):
    f = torch.finfo(t)
    return value.abs() * f.eps / 2 + f.smallest_normal * f.eps / 2


def operands(rows, t):
    x = torch.zeros(rows, 16, device="cuda", dtype=t)
    x[:, 0] = x[:, 1] = 1
    x[:, 2] = 4
    wg, wu = (torch.zeros(16, COLS, device="cuda", dtype=t) for _ in range(2))
    wg[0], wu[1] = gates(t), 1
    return x, wg, wu


@pytest.mark.parametrize("t", list(DTYPES))
@pytest.mark.parametrize("kind", ["silu", "gelu"])
@pytest.mark.parametrize("rows", [1, 3, 300])
def test_forward(be, rows, kind, t):
    t = DTYPES[t]
    x, wg, wu = operands(rows, t)
    hidden, gate, up = (torch.empty(rows, COLS, device="cuda", dtype=t) for _ in range(3))
    be.gated_forward(rows, 16, COLS, x.data_ptr(), wg.data_ptr(), wu.data_ptr(), hidden.data_ptr(), gate.data_ptr(), up.data_ptr(),
                     type=B.BF16 if t is torch.bfloat16 else B.F16, act=B.ACTS[kind])
    assert (up == 1).all() and torch.equal(gate, wg[0].expand(rows, COLS))
    want, _, off, _ = exact(kind, wg[0].double())
    assert ((hidden.double() - want).abs() <= off + half_step(t, want.abs() + off)).all()


@pytest.mark.parametrize("t", list(DTYPES))
@pytest.mark.parametrize("kind", ["silu", "gelu"])
def test_backward(be, kind, t):
    """One row whose inputs are ones: dw_gate and dw_up are dgate and dup."""
    t = DTYPES[t]
    x, wg, wu = torch.ones(1, 8, device="cuda", dtype=t), *(torch.zeros(8, COLS, device="cuda", dtype=t) for _ in range(2))
    gate, ones = gates(t), torch.ones(COLS, device="cuda", dtype=t)
    dwg, dwu = torch.empty_like(wg), torch.empty_like(wu)
    work = torch.empty(B.gated_backward_workspace(1, 8, COLS), device="cuda", dtype=torch.uint8)
    be.gated_backward(1, 8, COLS, ones.data_ptr(), x.data_ptr(), wg.data_ptr(), wu.data_ptr(), gate.data_ptr(), ones.data_ptr(), 0,
                      dwg.data_ptr(), dwu.data_ptr(), work.data_ptr(), work.numel(), type=B.BF16 if t is torch.bfloat16 else B.F16,
                      act=B.ACTS[kind])
    value, slope, off_value, off_slope = exact(kind, gate.double())
    for got, want, off in ((dwg, slope, off_slope), (dwu, value, off_value)):
        # (and the product with one, stored: the same 16 bits again)
        assert ((got.double() - want).abs() <= off + half_step(t, want.abs() + off)).all()


@pytest.mark.parametrize("kind", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("rows", [1, 3])
def test_a_gate_beyond_f32_is_infinite(be, rows, kind):
    x, wg, wu = operands(rows, torch.bfloat16)
    wg[2, 5] = 2.0 ** 127
    hidden = torch.empty(rows, COLS, device="cuda", dtype=torch.bfloat16)
    be.gated_forward(rows, 16, COLS, x.data_ptr(), wg.data_ptr(), wu.data_ptr(), hidden.data_ptr(), act=B.ACTS[kind])
    assert (hidden[:, 5] == float("inf")).all() and torch.isfinite(hidden[:, 6:]).all()


def test_slope_of_a_gate_that_is_not_finite(be):
    """GELU's is 1 and 0 at either end; a NaN stays one."""
    x, w = torch.ones(1, 8, device="cuda", dtype=torch.bfloat16), torch.zeros(8, 8, device="cuda", dtype=torch.bfloat16)
    gate = torch.tensor([float("inf"), -float("inf"), float("nan"), 3e38, -3e38, 1e15, -1e15, 0.0], device="cuda").bfloat16()
    ones, dwg, dwu = torch.ones(8, device="cuda", dtype=torch.bfloat16), torch.empty_like(w), torch.empty_like(w)
    work = torch.empty(B.gated_backward_workspace(1, 8, 8), device="cuda", dtype=torch.uint8)
    be.gated_backward(1, 8, 8, ones.data_ptr(), x.data_ptr(), w.data_ptr(), w.data_ptr(), gate.data_ptr(), ones.data_ptr(), 0, dwg.data_ptr(),
                      dwu.data_ptr(), work.data_ptr(), work.numel(), act=B.ACT_GELU)
    got = dwg[0].float().tolist()
    assert got[:2] == [1.0, 0.0] and got[2] != got[2] and got[3:] == [1.0, 0.0, 1.0, 0.0, 0.5]
