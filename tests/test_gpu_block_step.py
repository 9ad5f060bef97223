"""The operators together, as a training step of a block's own weights uses them: norm, gated feed-forward, their backward passes
and AdamW, whose 16-bit copies are the next forward pass's weights.  Each stage against its formula at the inputs that it got
(the other files' checks and tolerances); the whole captured and replayed, and two of them at once, by bits."""

import pytest
import torch

from see_ai_b200 import backend as B
from test_gpu_adamw_tensors import check_p, formula, params
from test_gpu_gated import check_backward as check_gated_backward
from test_gpu_gated import check_forward as check_gated_forward
from test_gpu_norm import check_backward as check_norm_backward
from test_gpu_norm import check_forward as check_norm_forward

pytestmark = pytest.mark.gpu


class Block:
    """x [rows, d] f32 -> norm -> gated -> hidden [rows, f], weights in f32 with bf16 copies, moments in `bits`."""

    def __init__(self, be, kind, rows, d, f, bits, act, seed=0):
        self.be, self.kind, self.rows, self.d, self.f, self.bits, self.act = be, kind, rows, d, f, bits, act
        torch.manual_seed(seed)
        self.layer = kind == B.NORM_LAYER
        new = lambda *s, t=torch.float32: torch.zeros(*s, device="cuda", dtype=t)  # noqa: E731
        self.x, self.dh = torch.randn(rows, d, device="cuda"), torch.randn(rows, f, device="cuda").bfloat16()
        self.residual = torch.randn(rows, d, device="cuda")
        self.weights = dict(gamma=1 + 0.1 * torch.randn(d, device="cuda"), wg=torch.randn(d, f, device="cuda") * d ** -0.5,
                            wu=torch.randn(d, f, device="cuda") * d ** -0.5)
        if self.layer:
            self.weights["beta"] = 0.1 * torch.randn(d, device="cuda")
        self.copies = {k: self.weights[k].bfloat16() for k in ("wg", "wu")}
        self.grads = {k: new(*v.shape, t=torch.bfloat16 if k in self.copies else torch.float32) for k, v in self.weights.items()}
        state = torch.float8_e4m3fn if bits == 8 else torch.float32
        self.m, self.v = ({k: torch.zeros(v.numel(), device="cuda").to(state) for k, v in self.weights.items()} for _ in range(2))
        self.ms, self.vs = ({k: new((v.numel() + 255) // 256) for k, v in self.weights.items()} for _ in range(2))
        self.y, self.mean, self.rstd = new(rows, d, t=torch.bfloat16), new(rows), new(rows)
        self.hidden, self.gate, self.up = (new(rows, f, t=torch.bfloat16) for _ in range(3))
        self.dy, self.dx = new(rows, d, t=torch.bfloat16), new(rows, d)
        self.norm_work = new(B.norm_backward_workspace(rows, d), t=torch.uint8)
        self.gated_work = new(B.gated_backward_workspace(rows, d, f), t=torch.uint8)
        p = lambda t: t.data_ptr()  # noqa: E731
        self.table = B.adamw_tensors([
            dict(p=p(w), g=p(self.grads[k]), m=p(self.m[k]), v=p(self.v[k]), m_scale=p(self.ms[k]) if bits == 8 else 0,
                 v_scale=p(self.vs[k]) if bits == 8 else 0, copy=p(self.copies[k]) if k in self.copies else 0, n=w.numel(),
                 g_type=B.BF16 if k in self.copies else B.F32, copy_type=B.BF16 if k in self.copies else B.F32, no_decay=k not in self.copies)
            for k, w in self.weights.items()])

    def forward(self):
        p = lambda t: t.data_ptr()  # noqa: E731
        self.be.norm_forward(self.kind, self.rows, self.d, p(self.x), p(self.weights["gamma"]), p(self.weights["beta"]) if self.layer else 0,
                             p(self.y), p(self.mean) if self.layer else 0, p(self.rstd), y_type=B.BF16)
        self.be.gated_forward(self.rows, self.d, self.f, p(self.y), p(self.copies["wg"]), p(self.copies["wu"]), p(self.hidden), p(self.gate),
                              p(self.up), act=B.ACTS[self.act])

    def backward(self):
        p = lambda t: t.data_ptr()  # noqa: E731
        self.be.gated_backward(self.rows, self.d, self.f, p(self.dh), p(self.y), p(self.copies["wg"]), p(self.copies["wu"]), p(self.gate),
                               p(self.up), p(self.dy), p(self.grads["wg"]), p(self.grads["wu"]), p(self.gated_work), self.gated_work.numel(),
                               act=B.ACTS[self.act])
        self.be.norm_backward(self.kind, self.rows, self.d, p(self.dy), p(self.x), p(self.weights["gamma"]), p(self.mean) if self.layer else 0,
                              p(self.rstd), p(self.dx), p(self.grads["gamma"]), p(self.grads["beta"]) if self.layer else 0,
                              p(self.norm_work), self.norm_work.numel(), addend=p(self.residual), y_type=B.BF16)

    def step(self, step):
        self.forward()
        self.backward()
        self.be.adamw_step(self.table, params(step), state_bits=self.bits)

    def everything(self):
        out = [self.y, self.rstd, self.hidden, self.gate, self.up, self.dy, self.dx]
        for group in (self.weights, self.copies, self.grads, self.m, self.v, self.ms, self.vs):
            out += list(group.values())
        return [t.view(torch.uint8) for t in out]


@pytest.fixture()
def be():
    b = B.CudaBackend(0)
    b.set_stream(torch.cuda.current_stream().cuda_stream)
    yield b
    torch.cuda.synchronize()
    b.close()


SIZES = [(1, 64, 128), (100, 256, 688), (1000, 768, 2048)]


@pytest.mark.parametrize("kind,bits,act", [(B.NORM_LAYER, 8, "silu"), (B.NORM_RMS, 32, "gelu"), (B.NORM_RMS, 8, "relu")])
@pytest.mark.parametrize("rows,d,f", SIZES)
def test_every_stage_of_three_steps(be, rows, d, f, kind, bits, act):
    b = Block(be, kind, rows, d, f, bits, act)
    for step in (1, 2, 3):
        b.forward()
        beta = b.weights.get("beta", b.weights["gamma"])
        check_norm_forward(kind, b.x, b.weights["gamma"], beta, 1e-5, "bf16", b.y, b.mean, b.rstd)
        check_gated_forward(b.y, b.copies["wg"], b.copies["wu"], act, b.hidden, b.gate, b.up)
        b.backward()
        check_gated_backward(b.dh, b.y, b.copies["wg"], b.copies["wu"], b.gate, b.up, act, b.dy, b.grads["wg"], b.grads["wu"])
        check_norm_backward(kind, b.dy, b.x, b.weights["gamma"], b.mean, b.rstd, b.residual, b.dx, b.grads["gamma"], b.grads.get("beta"))
        before = {}
        for k, w in b.weights.items():
            wide = lambda s: s.double().repeat_interleave(256)[:w.numel()]  # noqa: E731
            m, v = b.m[k].double(), b.v[k].double()
            if bits == 8:
                m, v = b.m[k].float().double() * wide(b.ms[k]), (b.v[k].float().double() * wide(b.vs[k])).square()
            before[k] = (w.double().reshape(-1), b.grads[k].double().reshape(-1), m, v)
        be.adamw_step(b.table, params(step), state_bits=bits)
        for k, w in b.weights.items():
            want, _, _ = formula(*before[k], step, decay=k in b.copies)
            check_p(w.reshape(-1), before[k][0], want)
            assert k not in b.copies or torch.equal(b.copies[k], w.bfloat16())


@pytest.mark.parametrize("rows,d,f", SIZES)
def test_captured_and_replayed(be, rows, d, f):
    eager, other = (Block(be, B.NORM_LAYER, rows, d, f, 8, "silu") for _ in range(2))
    for _ in range(3):
        eager.step(5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    try:
        with torch.cuda.graph(graph, stream=side):
            be.set_stream(side.cuda_stream)
            other.step(5)
    finally:
        be.set_stream(torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(eager.everything(), other.everything()))


def test_two_at_once(be):
    """Two backends on two streams: neither waits for what the other holds, and both have the bits of one alone."""
    alone = Block(be, B.NORM_LAYER, 700, 512, 1376, 8, "gelu")
    for step in (1, 2, 3):
        alone.step(step)
    torch.cuda.synchronize()
    pair = []
    for _ in range(2):
        b = B.CudaBackend(0)   # (each on its own stream)
        pair.append(Block(b, B.NORM_LAYER, 700, 512, 1376, 8, "gelu"))
    torch.cuda.synchronize()
    for step in (1, 2, 3):
        for block in pair:
            block.step(step)
    torch.cuda.synchronize()
    for block in pair:
        assert all(torch.equal(a, b) for a, b in zip(alone.everything(), block.everything()))
        block.be.close()


def test_a_refused_call_does_nothing_and_says_why(be):
    b = Block(be, B.NORM_LAYER, 10, 64, 64, 8, "silu")
    before = [t.clone() for t in b.everything()]
    launches = be.counters().kernel_launches
    with pytest.raises(B.BackendError, match="norm forward: x and y overlap"):
        be.norm_forward(B.NORM_LAYER, 10, 64, b.x.data_ptr(), b.weights["gamma"].data_ptr(), b.weights["beta"].data_ptr(), b.x.data_ptr(),
                        b.mean.data_ptr(), b.rstd.data_ptr())
    with pytest.raises(B.BackendError, match="gated forward: d_in and d_hidden"):
        be.gated_forward(10, 60, 64, b.y.data_ptr(), b.copies["wg"].data_ptr(), b.copies["wu"].data_ptr(), b.hidden.data_ptr())
    with pytest.raises(B.BackendError, match="adamw: steps count from 1"):
        be.adamw_step(b.table, params(0), state_bits=8)
    assert be.counters().kernel_launches == launches
    torch.cuda.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(before, b.everything()))
