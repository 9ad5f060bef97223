"""The gated feed-forward block and its backward pass against the formulas in 64 bits.

Tolerances: the tensor cores add 16 products at a time to an f32 accumulator and cut at its magnitude, at most 2^-22 of the
sum of magnitudes each time; the activations are good to 2^-20; each 16-bit result, and dgate and dup before their products,
is off by half a step, finfo.eps / 2 of its value (and half the smallest step, where f16 runs out of exponents).
"""

import pytest
import torch

from see_ai_b200 import backend as B

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
NAMES = {v: k for k, v in DTYPES.items()}
GELU_C, GELU_A = 0.7978845608028654, 0.044715


@pytest.fixture(scope="module")
def be():
    b = B.CudaBackend(0)
    b.set_stream(torch.cuda.current_stream().cuda_stream)
    yield b
    torch.cuda.synchronize()
    b.close()


def act(kind, g):
    """The activation and its slope."""
    if kind == "relu":
        return g.clamp(min=0), (g > 0).double()
    if kind == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    t = torch.tanh(GELU_C * (g + GELU_A * g ** 3))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * GELU_C * (1 + 3 * GELU_A * g * g)


def half_step(t, value):
    f = torch.finfo(t)
    return value.abs() * f.eps / 2 + f.smallest_normal * f.eps / 2


def sum_error(terms, magnitudes):
    return (terms / 16 + 4) * 2.0 ** -22 * magnitudes


def inputs(rows, d_in, d_hidden, t, seed=0, x_stride=None):
    torch.manual_seed(seed + rows * 7 + d_in)
    x = torch.randn(rows, x_stride or d_in, device="cuda").to(t)[:, :d_in]
    wg, wu = ((torch.randn(d_in, d_hidden, device="cuda") * d_in ** -0.5).to(t) for _ in range(2))
    return x, wg, wu


def forward(be, x, wg, wu, kind, keep=True, hidden_stride=None):
    rows, d_in = x.shape
    f = wg.shape[1]
    stride = hidden_stride or f
    outs = [torch.full((rows, stride), 7.0, device="cuda", dtype=x.dtype) for _ in range(3 if keep else 1)]
    be.gated_forward(rows, d_in, f, x.data_ptr(), wg.data_ptr(), wu.data_ptr(), *(o.data_ptr() for o in outs),
                     type=B.TYPES[NAMES[x.dtype]], act=B.ACTS[kind], x_stride=x.stride(0) if rows > 1 else 0,
                     hidden_stride=hidden_stride or 0)
    for o in outs:
        assert (o[:, f:] == 7.0).all()
    return [o[:, :f] for o in outs]


def check_forward(x, wg, wu, kind, hidden, gate=None, up=None):
    t, d_in = x.dtype, x.shape[1]
    xd, g64, u64 = x.double(), wg.double(), wu.double()
    g, u = xd @ g64, xd @ u64
    eg, eu = (sum_error(d_in, xd.abs() @ w.abs()) for w in (g64, u64))
    value, _ = act(kind, g)
    want = value * u
    # |act'| <= 1.13 for GELU and 1.1 for SiLU
    allowed = 1.13 * eg * (u.abs() + eu) + (value.abs() + 2.0 ** -20 * g.abs()) * eu + 2.0 ** -20 * g.abs() * u.abs()
    assert ((hidden.double() - want).abs() <= allowed + half_step(t, want.abs() + allowed)).all()
    if gate is not None:
        assert ((gate.double() - g).abs() <= eg + half_step(t, g.abs() + eg)).all()
        assert ((up.double() - u).abs() <= eu + half_step(t, u.abs() + eu)).all()


SHAPES = [(1, 64, 64), (1, 8, 8), (3, 72, 200), (1, 768, 2048), (2, 4096, 1032), (8, 512, 1376), (17, 136, 264), (127, 64, 128), (128, 256, 512),
          (129, 768, 2048), (257, 1000, 1096), (600, 512, 1376), (1029, 264, 4104), (5000, 192, 520)]


@pytest.mark.parametrize("t", list(DTYPES))
@pytest.mark.parametrize("kind", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("rows,d_in,d_hidden", SHAPES)
def test_forward(be, rows, d_in, d_hidden, kind, t):
    x, wg, wu = inputs(rows, d_in, d_hidden, DTYPES[t])
    check_forward(x, wg, wu, kind, *forward(be, x, wg, wu, kind))
    check_forward(x, wg, wu, kind, *forward(be, x, wg, wu, kind, keep=False))


def backward(be, dh, x, wg, wu, gate, up, kind, want=(True, True)):
    rows, d_in = x.shape
    f = wg.shape[1]
    dx = torch.full((rows, x.stride(0) if rows > 1 else d_in), 7.0, device="cuda", dtype=x.dtype) if want[0] else None
    dwg, dwu = (torch.full_like(wg, 7.0) if want[1] else None for _ in range(2))
    work = torch.empty(B.gated_backward_workspace(rows, d_in, f), device="cuda", dtype=torch.uint8)
    p = lambda v: 0 if v is None else v.data_ptr()  # noqa: E731
    be.gated_backward(rows, d_in, f, dh.data_ptr(), x.data_ptr(), wg.data_ptr(), wu.data_ptr(), gate.data_ptr(), up.data_ptr(), p(dx),
                      p(dwg), p(dwu), work.data_ptr(), work.numel(), type=B.TYPES[NAMES[x.dtype]], act=B.ACTS[kind],
                      x_stride=x.stride(0) if rows > 1 else 0, hidden_stride=dh.stride(0) if rows > 1 else 0)
    if dx is not None:
        assert (dx[:, d_in:] == 7.0).all()
        dx = dx[:, :d_in]
    return dx, dwg, dwu


def check_backward(dh, x, wg, wu, gate, up, kind, dx, dwg, dwu):
    t, rows, f = x.dtype, x.shape[0], wg.shape[1]
    value, slope = act(kind, gate.double())
    d = dh.double()
    dg, du = d * up.double() * slope, d * value
    near = 2.0 ** -19 * (d * up.double()).abs() + half_step(t, dg), 2.0 ** -19 * (d * gate.double()).abs() + half_step(t, du)
    if dx is not None:
        want = dg @ wg.double().T + du @ wu.double().T
        size = dg.abs() @ wg.double().abs().T + du.abs() @ wu.double().abs().T
        allowed = near[0] @ wg.double().abs().T + near[1] @ wu.double().abs().T + sum_error(2 * f, 1.01 * size)
        assert ((dx.double() - want).abs() <= allowed + half_step(t, want.abs() + allowed)).all()
    if dwg is not None:
        for got, v, n in ((dwg, dg, near[0]), (dwu, du, near[1])):
            want = x.double().T @ v
            allowed = x.double().abs().T @ n + sum_error(rows, 1.01 * (x.double().abs().T @ v.abs()))
            assert ((got.double() - want).abs() <= allowed + half_step(t, want.abs() + allowed)).all()


def gradients(rows, f, t, x, wg, wu, stride=None):
    gate, up = ((x.float() @ w.float()).to(t) for w in (wg, wu))
    dh = torch.randn(rows, f, device="cuda").to(t)
    if stride:
        gate, up, dh = (torch.nn.functional.pad(v, (0, stride - f), value=3.0)[:, :f] for v in (gate, up, dh))
    return dh, gate, up


@pytest.mark.parametrize("t", list(DTYPES))
@pytest.mark.parametrize("kind", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("rows,d_in,d_hidden", SHAPES)
def test_backward(be, rows, d_in, d_hidden, kind, t):
    x, wg, wu = inputs(rows, d_in, d_hidden, DTYPES[t])
    dh, gate, up = gradients(rows, d_hidden, DTYPES[t], x, wg, wu)
    out = backward(be, dh, x, wg, wu, gate, up, kind)
    check_backward(dh, x, wg, wu, gate, up, kind, *out)
    again = backward(be, dh, x, wg, wu, gate, up, kind)
    assert all(torch.equal(a, b) for a, b in zip(out, again))


@pytest.mark.parametrize("want", [(True, False), (False, True)])
def test_backward_of_what_is_wanted(be, want):
    x, wg, wu = inputs(300, 128, 320, torch.bfloat16)
    dh, gate, up = gradients(300, 320, torch.bfloat16, x, wg, wu)
    check_backward(dh, x, wg, wu, gate, up, "silu", *backward(be, dh, x, wg, wu, gate, up, "silu", want))


def test_gradients_against_differences(be):
    """(L(w + h) - L(w - h)) / 2h of L = sum(hidden dhidden) in 64 bits, at inputs that 16 bits hold and with the gate and up
    that belong to them; off by h^2 times third derivatives, against the roundings that check_backward allows."""
    t, rows, d_in, f, h = torch.float16, 5, 16, 24, 1e-4
    x, wg, wu = inputs(rows, d_in, f, t, seed=9)
    dh = torch.randn(rows, f, device="cuda").to(t)
    for kind in ("silu", "gelu"):
        _, gate, up = forward(be, x, wg, wu, kind)
        out = backward(be, dh, x, wg, wu, gate, up, kind)
        at = [x.double(), wg.double(), wu.double()]

        def loss(x, wg, wu):
            return (act(kind, x @ wg)[0] * (x @ wu) * dh.double()).sum()

        for k, got in enumerate(out):
            for i in range(0, got.numel(), 5):
                step = torch.zeros_like(at[k])
                step.view(-1)[i] = h
                plus, minus = list(at), list(at)
                plus[k], minus[k] = at[k] + step, at[k] - step
                want = ((loss(*plus) - loss(*minus)) / (2 * h)).item()
                # terms of up to 24 * |3 * 3 * 3| with 2^-11 each of gate, up, dgate and the result
                assert abs(got.reshape(-1)[i].item() - want) <= 48 * 27 * 4 * 2.0 ** -11 / 8


def test_strided_rows(be):
    rows, d_in, f = 333, 136, 264
    x, wg, wu = inputs(rows, d_in, f, torch.bfloat16, x_stride=160)
    check_forward(x, wg, wu, "silu", *forward(be, x, wg, wu, "silu", hidden_stride=280))
    dh, gate, up = gradients(rows, f, torch.bfloat16, x, wg, wu, stride=272)
    check_backward(dh, x, wg, wu, gate, up, "silu", *backward(be, dh, x, wg, wu, gate, up, "silu"))


def test_gate_and_up_side_by_side(be):
    """Two halves of one buffer's rows."""
    rows, d_in, f = 200, 64, 128
    x, wg, wu = inputs(rows, d_in, f, torch.bfloat16)
    both = torch.empty(rows, 2 * f, device="cuda", dtype=torch.bfloat16)
    hidden = torch.empty_like(both)
    be.gated_forward(rows, d_in, f, x.data_ptr(), wg.data_ptr(), wu.data_ptr(), hidden.data_ptr(), both.data_ptr(),
                     both.data_ptr() + 2 * f, hidden_stride=2 * f)
    check_forward(x, wg, wu, "silu", hidden[:, :f], both[:, :f], both[:, f:])


def test_not_finite_stays_in_its_row(be):
    x, wg, wu = inputs(300, 64, 192, torch.bfloat16)
    x[7, 3], x[140, 0] = float("nan"), float("inf")
    hidden, gate, up = forward(be, x, wg, wu, "relu")
    fine = torch.ones(300, dtype=torch.bool, device="cuda")
    fine[7] = fine[140] = False
    assert torch.isnan(hidden[7]).all() and torch.isnan(gate[7]).all() and not torch.isfinite(gate[140]).any()
    check_forward(x[fine], wg, wu, "relu", hidden[fine], gate[fine], up[fine])


def test_no_rows(be):
    x, wg, wu = inputs(1, 64, 64, torch.bfloat16)
    hidden = torch.full((1, 64), 7.0, device="cuda", dtype=torch.bfloat16)
    be.gated_forward(0, 64, 64, x.data_ptr(), wg.data_ptr(), wu.data_ptr(), hidden.data_ptr())
    assert (hidden == 7.0).all()
    dwg, dwu = torch.ones_like(wg), torch.ones_like(wu)
    work = torch.empty(B.gated_backward_workspace(0, 64, 64), device="cuda", dtype=torch.uint8)
    be.gated_backward(0, 64, 64, hidden.data_ptr(), x.data_ptr(), wg.data_ptr(), wu.data_ptr(), hidden.data_ptr(), hidden.data_ptr(), 0,
                      dwg.data_ptr(), dwu.data_ptr(), work.data_ptr(), work.numel())
    assert (dwg == 0).all() and (dwu == 0).all()


def test_captured_and_replayed(be):
    x, wg, wu = inputs(700, 192, 448, torch.bfloat16)
    dh, gate, up = gradients(700, 448, torch.bfloat16, x, wg, wu)
    want_h = forward(be, x, wg, wu, "gelu", keep=False)[0]
    want = backward(be, dh, x, wg, wu, gate, up, "gelu")
    hidden, out = torch.zeros_like(want_h), [torch.zeros_like(v) for v in want]
    work = torch.empty(B.gated_backward_workspace(700, 192, 448), device="cuda", dtype=torch.uint8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    try:
        with torch.cuda.graph(graph, stream=side):
            be.set_stream(side.cuda_stream)
            be.gated_forward(700, 192, 448, x.data_ptr(), wg.data_ptr(), wu.data_ptr(), hidden.data_ptr(), act=B.ACT_GELU)
            be.gated_backward(700, 192, 448, dh.data_ptr(), x.data_ptr(), wg.data_ptr(), wu.data_ptr(), gate.data_ptr(), up.data_ptr(),
                              *(o.data_ptr() for o in out), work.data_ptr(), work.numel(), act=B.ACT_GELU)
    finally:
        be.set_stream(torch.cuda.current_stream().cuda_stream)
    for _ in range(2):
        hidden.zero_()
        for o in out:
            o.zero_()
        graph.replay()
        assert torch.equal(hidden, want_h) and all(torch.equal(a, b) for a, b in zip(out, want))
