"""The norm over all gradients, the factor that clips them and the clipped gradients, against the formulas in 64 bits.

Tolerances: a thread adds at most 64 f32 squares, eight at a time and the eights after that: 8 + 8 roundings and the square's own,
each at most 2^-24 of the sum; beyond that sums are double.  The root halves the error; the result's rounding adds one."""

import math

import pytest
import torch

from see_ai_b200 import backend as B

pytestmark = pytest.mark.gpu

ULP = 2.0 ** -24
OFF = 17 / 2 * ULP + 2 * ULP   # relative, of norm and factor
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


@pytest.fixture(scope="module")
def be():
    b = B.CudaBackend(0)
    b.set_stream(torch.cuda.current_stream().cuda_stream)
    yield b
    torch.cuda.synchronize()
    b.close()


class Call:
    def __init__(self, be, max_norm, scale=None):
        self.be, self.max_norm = be, max_norm
        self.norm, self.factor = (torch.full((1,), 7.0, device="cuda") for _ in range(2))
        self.scale = None if scale is None else torch.full((1,), scale, device="cuda")
        self.work = torch.full((B.grad_workspace(),), 0xFF, device="cuda", dtype=torch.uint8)   # (NaNs)

    def __call__(self, tensors, outs=None, clip=False):
        names = {v: B.TYPES[k] for k, v in DTYPES.items()}
        table = B.grad_tensors([dict(g=t.data_ptr(), out=0 if outs is None else outs[i].data_ptr(), n=t.numel(), type=names[t.dtype])
                                for i, t in enumerate(tensors)])
        (self.be.grad_clip if clip else self.be.grad_norm)(table, self.max_norm, self.norm.data_ptr(), self.factor.data_ptr(), self.work.data_ptr(),
                                                           self.work.numel(), 0 if self.scale is None else self.scale.data_ptr())
        return float(self.norm), float(self.factor)


def formula(tensors, max_norm, scale=1.0):
    norm = math.sqrt(sum(float(t.double().square().sum()) for t in tensors)) * abs(scale)
    return norm, scale * (1.0 if norm <= max_norm or norm == 0 else max_norm / norm)


def near(a, b, off=OFF):
    return abs(a - b) <= off * abs(b)


def check_out(t, out, factor):
    want = t.double() * factor
    step = torch.finfo(out.dtype)
    allowed = (ULP if out.dtype == torch.float32 else step.eps / 2 * (1 + 2 ** -12)) * want.abs() + step.smallest_normal * step.eps
    assert ((out.double() - want).abs() <= allowed).all()


LISTS = {"one element": [1], "one": [1000], "a chunk": [8192], "and one": [8193, 16385], "many": [1, 7, 0, 4096, 100003, 12, 1 << 20],
         "adapters": [768 * 16] * 96, "hundreds": [33] * 700, "large": [9000001]}


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("name", list(LISTS))
def test_norm_and_factor(be, name, dtype):
    torch.manual_seed(3)
    tensors = [(torch.randn(n, device="cuda") * math.exp(i % 5 - 2)).to(DTYPES[dtype]) for i, n in enumerate(LISTS[name])]
    for max_norm, scale in ((1e-3, None), (0.5, 0.25), (1e6, None), (1e6, -2.0), (math.inf, 4.0)):
        norm, factor = Call(be, max_norm, scale)(tensors)
        want_norm, want_factor = formula(tensors, max_norm, scale or 1.0)
        assert near(norm, want_norm) and near(factor, want_factor)
        if max_norm >= 1e6:
            assert factor == (scale or 1.0)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("where", ["in place", "apart", "unlike"])
@pytest.mark.parametrize("name", ["one element", "and one", "many", "hundreds"])
def test_clipped(be, name, where, dtype):
    torch.manual_seed(5)
    tensors = [torch.randn(n, device="cuda").to(DTYPES[dtype]) for n in LISTS[name]]
    kept = [t.clone() for t in tensors]
    outs = None
    if where != "in place":   # unlike: not aligned as the gradients are, and what lies around is left alone
        shift = 8 if where == "apart" else 3
        whole = [torch.full((t.numel() + 16,), 9.0, device="cuda", dtype=t.dtype) for t in tensors]
        outs = [w[shift:shift + t.numel()] for w, t in zip(whole, tensors)]
    call = Call(be, 0.5, 0.75)
    norm, factor = call(tensors, outs, clip=True)
    want_norm, want_factor = formula(kept, 0.5, 0.75)
    assert near(norm, want_norm) and near(factor, want_factor)
    for t, o in zip(kept, tensors if outs is None else outs):
        check_out(t, o, factor)
    if outs is not None:
        assert all(torch.equal(a, b) for a, b in zip(kept, tensors))
        for w, t in zip(whole, tensors):
            assert (w[:shift] == 9).all() and (w[shift + t.numel():] == 9).all()


def test_views_that_begin_anywhere(be):
    torch.manual_seed(7)
    for dtype in DTYPES.values():
        buf = torch.randn(70000, device="cuda").to(dtype)
        buf[:9], buf[-9:] = 1e4, 1e4
        for begin in range(9, 18):
            for n in (1, 3, 8, 9, 40, 8200, 60001):
                t = buf[begin:begin + n]
                norm, _ = Call(be, 1.0)([t])
                assert near(norm, formula([t], 1.0)[0])


def test_below_the_limit_nothing_is_written(be):
    t = torch.randn(5000, device="cuda")
    kept = t.clone()
    out = torch.zeros_like(t)
    assert Call(be, 1e4)([t], clip=True)[1] == 1.0 and torch.equal(t, kept)
    Call(be, 1e4)([t], [out], clip=True)
    assert torch.equal(out, kept)


def test_no_elements(be):
    for tensors in ([], [torch.empty(0, device="cuda")]):
        for clip in (False, True):
            assert Call(be, 1.0)(tensors, clip=clip) == (0.0, 1.0)
            assert Call(be, 1.0, 0.5)(tensors, clip=clip) == (0.0, 0.5)
    zeros = torch.zeros(100000, device="cuda", dtype=torch.bfloat16)
    assert Call(be, 1.0)([zeros], clip=True) == (0.0, 1.0)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("size", [1e-38, 1e-30, 1e-22, 1e-18, 1e18, 1e25, 3e34])
def test_sizes_whose_squares_f32_does_not_hold(be, size, dtype):
    torch.manual_seed(9)
    t = (torch.randn(50000, device="cuda").double() * size).to(DTYPES[dtype])
    norm, factor = Call(be, size)([t])
    want_norm, want_factor = formula([t], float(torch.tensor(size).float()))
    assert near(norm, want_norm, OFF + 2.0 ** -149 / want_norm) and near(factor, want_factor, OFF + 2.0 ** -149 / want_norm)
    # A few large ones among them.
    t[::1000] = 1.0
    assert near(Call(be, 1.0)([t])[0], formula([t], 1.0)[0])


def test_what_is_not_finite_shows(be):
    t = torch.randn(50000, device="cuda")
    t[777] = math.inf
    assert Call(be, 1.0)([t]) == (math.inf, 0.0)
    t[778] = math.nan
    norm, factor = Call(be, 1.0)([t])
    assert math.isnan(norm) and math.isnan(factor)


def test_same_bits_and_replayed(be):
    torch.manual_seed(11)
    tensors = [torch.randn(n, device="cuda").bfloat16() for n in LISTS["many"] + LISTS["hundreds"]]
    outs = [torch.empty_like(t) for t in tensors]
    call = Call(be, 0.5)
    want = call(tensors, outs, clip=True)
    kept = [o.clone() for o in outs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    again = Call(be, 0.5)
    names = {v: B.TYPES[k] for k, v in DTYPES.items()}
    table = B.grad_tensors([dict(g=t.data_ptr(), out=o.data_ptr(), n=t.numel(), type=names[t.dtype]) for t, o in zip(tensors, outs)])
    try:
        with torch.cuda.graph(graph, stream=side):
            be.set_stream(side.cuda_stream)
            be.grad_clip(table, 0.5, again.norm.data_ptr(), again.factor.data_ptr(), again.work.data_ptr(), again.work.numel())
    finally:
        be.set_stream(torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        for o in outs:
            o.zero_()
        graph.replay()
        assert (float(again.norm), float(again.factor)) == want and all(torch.equal(a, b) for a, b in zip(kept, outs))


def test_factor_is_what_adamw_takes(be):
    """Clipped gradients and the factor as AdamW's grad_scale give the same weights but for the gradients' second rounding."""
    torch.manual_seed(13)
    w = torch.randn(5000, device="cuda")
    g = torch.randn(5000, device="cuda")
    results = []
    for clip in (False, True):
        p, grad, m, v = w.clone(), g.clone(), torch.zeros_like(w), torch.zeros_like(w)
        call = Call(be, 0.25)
        call([grad], clip=clip)
        table = B.adamw_tensors([dict(p=p.data_ptr(), g=grad.data_ptr(), m=m.data_ptr(), v=v.data_ptr(), n=5000)])
        be.adamw_step(table, B.StepParams(1e-3, 0.9, 0.999, 1e-8, 0.0, 0, 1), grad_scale=0 if clip else call.factor.data_ptr())
        results.append((p, m, v))
    assert all(torch.equal(a, b) for a, b in zip(*results))
