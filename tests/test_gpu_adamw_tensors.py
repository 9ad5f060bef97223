"""AdamW over many tensors at once, moments in 32 bits and in 8, against the formulas in 64 bits and the kAdamWStep instruction."""

import numpy as np
import pytest
import torch

from see_ai_b200 import backend as B
from see_ai_b200 import plan as P

pytestmark = pytest.mark.gpu

ULP = 2.0 ** -24
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
E4M3 = torch.float8_e4m3fn
PARAMS = dict(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.01)


@pytest.fixture(scope="module")
def be():
    b = B.CudaBackend(0)
    b.set_stream(torch.cuda.current_stream().cuda_stream)
    yield b
    torch.cuda.synchronize()
    b.close()


def params(step, **over):
    v = dict(PARAMS, **over)
    return B.StepParams(v["lr"], v["beta1"], v["beta2"], v["eps"], v["weight_decay"], 0, step)


def at(buf, offset):
    return buf.data_ptr() + offset * buf.element_size()


class Tensors:
    """`sizes` tensors, `gap` elements apart in common buffers, of a run's middle."""

    def __init__(self, sizes, bits, grad="f32", copy="f32", gap=0, seed=0, zero=False):
        torch.manual_seed(seed)
        self.bits, self.sizes, self.offsets = bits, sizes, []
        total = gap
        for n in sizes:
            self.offsets.append(total)
            total += n + gap
        self.blocks, self.block_at = 0, []
        for n in sizes:
            self.block_at.append(self.blocks)
            self.blocks += (n + 255) // 256
        r = lambda: torch.randn(total, device="cuda")  # noqa: E731
        self.p, self.g = r() * 0.02, (r() * 1e-3).to(DTYPES[grad])
        self.copy = torch.full((total,), 9.0, device="cuda", dtype=DTYPES[copy]) if copy != "f32" else None
        self.m, self.v, self.ms, self.vs = r() * 3e-4 * (not zero), r().square() * 1e-6 * (not zero), None, None
        if bits == 8:
            self.m, self.v = (self.m / 1e-5).clamp(-448, 448).to(E4M3), (self.v.sqrt() / 1e-5).clamp(0, 448).to(E4M3)
            self.ms, self.vs = (torch.rand(self.blocks + 1, device="cuda") * 1e-5 for _ in range(2))
        self.grad, self.copy_type = grad, copy

    def buffers(self):
        return [b for b in (self.p, self.m, self.v, self.ms, self.vs, self.copy) if b is not None]

    def table(self, no_decay=()):
        return B.adamw_tensors([
            dict(p=at(self.p, o), g=at(self.g, o), m=at(self.m, o), v=at(self.v, o), m_scale=at(self.ms, b) if self.bits == 8 else 0,
                 v_scale=at(self.vs, b) if self.bits == 8 else 0, copy=at(self.copy, o) if self.copy is not None else 0, n=n,
                 g_type=B.TYPES[self.grad], copy_type=B.TYPES[self.copy_type], no_decay=i in no_decay)
            for i, (n, o, b) in enumerate(zip(self.sizes, self.offsets, self.block_at))])

    def values(self, i):
        """p, g, m, second moment of tensor i in 64 bits."""
        n, o, b = self.sizes[i], self.offsets[i], self.block_at[i]
        cut = lambda t: t[o:o + n].double()  # noqa: E731
        if self.bits == 32:
            return cut(self.p), cut(self.g), cut(self.m), cut(self.v)
        wide = lambda s: s[b:b + (n + 255) // 256].double().repeat_interleave(256)[:n]  # noqa: E731
        return cut(self.p), cut(self.g), cut(self.m.float()) * wide(self.ms), (cut(self.v.float()) * wide(self.vs)).square()


def formula(p, g, m, v, step, decay=True, scale=1.0):
    f = {k: float(np.float32(x)) for k, x in PARAMS.items()}
    g = g * scale
    m, v = f["beta1"] * m + (1 - f["beta1"]) * g, f["beta2"] * v + (1 - f["beta2"]) * g * g
    mh, vh = m / (1 - f["beta1"] ** step), v / (1 - f["beta2"] ** step)
    return p - f["lr"] * (mh / (vh.sqrt() + f["eps"]) + (f["weight_decay"] if decay else 0.0) * p), m, v


def check_p(got, before, want):
    # The update is lr times a quotient of at most ~1/sqrt(1 - beta2): a score of f32 roundings in it, corrections off by
    # 2^-24 / (1 - beta^step) <= 1000 * 2^-24 at step 1, and one rounding of p.
    update = (want - before).abs()
    assert ((got.double() - want).abs() <= ULP * (want.abs() + before.abs()) + 1100 * ULP * update + 1e-12).all()


SIZES = [[1], [255], [256], [257], [2048 * 3 + 5], [1, 2, 3, 4, 5], [768 * 16] * 5, [5, 0, 4096, 0, 300], [33] * 61, [70000, 3, 2500]]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{s[0]}")
@pytest.mark.parametrize("grad,copy,gap", [("f32", "f32", 0), ("bf16", "bf16", 3), ("f16", "f16", 8), ("bf16", "f32", 1)])
def test_step(be, bits, sizes, grad, copy, gap):
    t = Tensors(sizes, bits, grad, copy, gap, seed=len(sizes))
    before = [b.clone() for b in t.buffers()]
    start = [t.values(i) for i in range(len(sizes))]
    be.adamw_step(t.table(no_decay={1}), params(17), state_bits=bits)
    touched = torch.zeros(t.p.numel(), dtype=torch.bool, device="cuda")
    for i, n in enumerate(sizes):
        if n == 0:
            continue
        o, b = t.offsets[i], t.block_at[i]
        touched[o:o + n] = True
        want, m, v = formula(*start[i], 17, decay=i != 1)
        check_p(t.p[o:o + n], start[i][0], want)
        if t.copy is not None:
            assert torch.equal(t.copy[o:o + n], t.p[o:o + n].to(t.copy.dtype))
        _, _, got_m, got_v = t.values(i)
        if bits == 32:
            assert ((got_m - m).abs() <= 3 * ULP * (m.abs() + start[i][2].abs() + start[i][1].abs())).all()
            assert ((got_v - v).abs() <= 5 * ULP * v).all()
            continue
        for got, exact, scale in ((got_m, m, t.ms), (got_v.sqrt(), v.sqrt(), t.vs)):
            blocks = (n + 255) // 256
            largest = torch.nn.functional.pad(exact.abs(), (0, blocks * 256 - n)).view(blocks, 256).amax(1)
            assert ((scale[b:b + blocks].double() - largest / 448).abs() <= 8 * ULP * largest / 448).all()
            unit = (largest / 448).repeat_interleave(256)[:n]
            # A cut goes to one of the two neighbours: closer than their distance, 1/8 of the power of two below (from 2^-6 on).
            code = exact.abs() / unit
            distance = 2.0 ** (torch.floor(torch.log2(code.clamp(min=2.0 ** -6) * (1 + 1e-6))) - 3)
            assert ((got - exact).abs() <= (distance * (1 + 1e-5) + code * 2e-6) * unit).all()
            assert ((got.abs() > 0) | (exact.abs() < unit * 2.0 ** -9 * (1 + 1e-5))).all()
        assert ((got_v > 0) | (v == 0)).all()
    for was, now in zip(before, t.buffers()):   # what lies between the tensors
        if now.numel() == touched.numel():
            assert torch.equal(was.view(torch.uint8).view(touched.numel(), -1)[~touched], now.view(torch.uint8).view(touched.numel(), -1)[~touched])
    if bits == 8:
        assert t.ms[-1] == before[3][-1] and t.vs[-1] == before[4][-1]


@pytest.mark.parametrize("n", [1, 300, 768 * 16 + 3])
def test_f32_moments_have_the_instructions_bits(be, n):
    t = Tensors([n], 32, seed=3)
    arena = np.concatenate([b.cpu().numpy() for b in (t.p, t.g, t.m, t.v)]).view(np.uint8).copy()
    host = B.CudaBackend(0)
    host.bind(arena, None)
    host.run([P.Instr(P.Op.ADAMW_STEP, 0, 0, (0, 4 * n, 8 * n, 12 * n), (n, 0, 0))], params(5))
    host.close()
    be.adamw_step(t.table(), params(5))
    want = arena.view(np.float32).reshape(4, n)
    for row, got in ((0, t.p), (2, t.m), (3, t.v)):
        assert want[row].tobytes() == got.cpu().numpy().tobytes()


@pytest.mark.parametrize("bits", [32, 8])
def test_first_step_from_zero_bytes_and_gradient_scale(be, bits):
    t = Tensors([1000], bits, "bf16", zero=True)
    if bits == 8:
        for b in (t.m, t.v):
            b.view(torch.uint8).zero_()
        t.ms.zero_(), t.vs.zero_()
    p, g, m, v = t.values(0)
    scale = torch.tensor([0.25], device="cuda")
    be.adamw_step(t.table(), params(1), state_bits=bits, grad_scale=scale.data_ptr())
    want, _, _ = formula(p, g, m, v, 1, scale=0.25)
    check_p(t.p, p, want)


def test_zero_gradients_leave_zero_moments_and_only_decay(be):
    t = Tensors([600], 8, zero=True)
    t.g.zero_()
    for b in (t.m, t.v):
        b.view(torch.uint8).zero_()
    p = t.p.double()
    be.adamw_step(t.table(), params(3), state_bits=8)
    assert (t.m.view(torch.uint8) == 0).all() and (t.v.view(torch.uint8) == 0).all() and (t.ms[:3] == 0).all()
    assert ((t.p.double() - p * (1 - 1e-5)).abs() <= 2 * ULP * p.abs()).all()


def test_cut_is_even_over_elements_and_steps(be):
    """The cut's offsets are multiples of the golden section plus multiples of sqrt(2), modulo 1: over N consecutive elements
    or steps their share below any point is off by less than 3 log(N) / N (bounded partial quotients).  So the values held
    for one number average to it within that share of the distance between its neighbours."""
    n = 65536
    t = Tensors([n], 8, zero=True)
    t.g.fill_(3.1e-3)
    t.g[::256] = 1e-2                       # the blocks' largest
    for step in (1, 2, 1000):
        for b in (t.m, t.v):
            b.view(torch.uint8).zero_()
        be.adamw_step(t.table(), params(step), state_bits=8)
        _, _, m, v = t.values(0)
        keep = torch.ones(n, dtype=torch.bool, device="cuda")
        keep[::256] = False
        for got, exact in ((m, 3.1e-4), (v.sqrt(), 3.1e-3 * (1 - float(np.float32(0.999))) ** 0.5)):
            assert abs((got[keep].mean() / exact).item() - 1) <= 0.125 * 3 * np.log(n) / n * 256
            assert got[keep].unique().numel() == 2
    held = []
    for step in range(1, 257):
        for b in (t.m, t.v):
            b.view(torch.uint8).zero_()
        be.adamw_step(t.table(), params(step), state_bits=8)
        held.append(t.values(0)[2][5])
    mean = torch.stack(held).mean().item()
    assert abs(mean / 3.1e-4 - 1) <= 0.125 * 3 * np.log(256) / 256


def test_not_finite_gradients(be):
    """f32 moments: the element alone.  8 bits: its block's moments, and of the weights the element alone at this step."""
    for bits in (32, 8):
        t = Tensors([1024], bits)
        t.g[300] = float("nan")
        t.g[800] = float("inf")
        be.adamw_step(t.table(), params(9), state_bits=bits)
        assert torch.isnan(t.p[300]) and torch.isnan(t.p[800])
        fine = torch.ones(1024, dtype=torch.bool, device="cuda")
        fine[300] = fine[800] = False
        assert torch.isfinite(t.p[fine]).all()
        if bits == 8:
            assert torch.isnan(t.ms[[1, 3]]).all() and torch.isfinite(t.ms[[0, 2]]).all() and torch.isnan(t.vs[[1, 3]]).all()
            _, _, m, v = t.values(0)
            assert torch.isnan(m[256:512]).all() and torch.isnan(v[768:]).all() and torch.isfinite(m[:256]).all()


def test_captured_table_is_the_graphs_own(be):
    """Two graphs of one backend, tables freed after capture, replayed in turn."""
    sets = [Tensors([700, 5], 8, seed=1), Tensors([3000], 8, seed=2)]
    twins = [Tensors([700, 5], 8, seed=1), Tensors([3000], 8, seed=2)]
    for w in twins:
        be.adamw_step(w.table(), params(4), state_bits=8)
        be.adamw_step(w.table(), params(4), state_bits=8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    try:
        for t in sets:
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1], stream=side):
                be.set_stream(side.cuda_stream)
                be.adamw_step(t.table(), params(4), state_bits=8)
    finally:
        be.set_stream(torch.cuda.current_stream().cuda_stream)
    for _ in range(2):
        for g in graphs:
            g.replay()
    for t, w in zip(sets, twins):
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(t.buffers(), w.buffers()))
