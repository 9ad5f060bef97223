"""The operators together, as a step that learns from preferences uses them: a block joins the residual stream, a head makes logits of the next
norm's output, the preference loss turns them into their gradient in place, the join's backward pass, the norm of all gradients and AdamW with its
factor.  Each stage against its formula at the inputs that it got (the other files' checks and tolerances); the whole captured and replayed, and two of
them at once, by bits."""

import pytest
import torch

import logit_reference as R
from see_ai_b200 import backend as B
from test_gpu_adamw_tensors import check_p, formula, params
from test_gpu_grad_norm import formula as norm_formula
from test_gpu_grad_norm import near
from test_gpu_join import Join

pytestmark = pytest.mark.gpu

MAX_NORM = 0.01


class Step:
    def __init__(self, be, kind, lengths, d, classes, gate=True, seed=0):
        self.be, self.classes, self.pairs = be, classes, len(lengths) // 2
        starts = [0]
        for n in lengths:
            starts.append(starts[-1] + n)
        rows = starts[-1] + 2
        self.starts = torch.tensor(starts, device="cuda", dtype=torch.int32)
        self.join = Join(kind, rows, d, "f32", "bf16", gate=gate, seed=seed)
        self.join.dy.zero_()
        torch.manual_seed(seed + 7)
        self.labels = torch.randint(classes, (rows,), device="cuda", dtype=torch.int32)
        self.labels[::3] = -1
        self.ref = torch.randn(2 * self.pairs, device="cuda") - 10.0
        self.head = torch.randn(classes, d, device="cuda") * d ** -0.5
        self.head16, self.dhead = self.head.bfloat16(), torch.zeros(classes, d, device="cuda", dtype=torch.bfloat16)
        self.logits = torch.zeros(rows, classes, device="cuda", dtype=torch.bfloat16)
        self.loss, self.norm, self.factor = (torch.zeros(1, device="cuda") for _ in range(3))
        self.margins, self.sums = torch.zeros(self.pairs, device="cuda"), torch.zeros(2 * self.pairs, device="cuda")
        self.work = torch.zeros(B.preference_workspace(rows, self.pairs), device="cuda", dtype=torch.uint8)
        self.grad_work = torch.zeros(B.grad_workspace(), device="cuda", dtype=torch.uint8)
        self.weights = dict({k: v for k, v in self.join.w.items() if v is not None}, head=self.head)
        self.grads = dict({k: v for k, v in self.join.g.items() if v is not None}, head=self.dhead)
        self.m, self.v = ({k: torch.zeros_like(w) for k, w in self.weights.items()} for _ in range(2))
        types = {torch.float32: B.F32, torch.bfloat16: B.BF16}
        p = lambda t: t.data_ptr()  # noqa: E731
        self.grad_table = B.grad_tensors([dict(g=p(g), n=g.numel(), type=types[g.dtype]) for g in self.grads.values()])
        self.table = B.adamw_tensors([
            dict(p=p(w), g=p(self.grads[k]), m=p(self.m[k]), v=p(self.v[k]), copy=p(self.head16) if k == "head" else 0, n=w.numel(),
                 g_type=types[self.grads[k].dtype], copy_type=B.BF16 if k == "head" else B.F32, no_decay=k != "head") for k, w in self.weights.items()])

    def forward(self):
        self.join.forward(self.be)
        torch.mm(self.join.y, self.head16.T, out=self.logits)

    def loss_and_gradient(self):
        p = lambda t: t.data_ptr()  # noqa: E731
        self.be.preference_loss(self.join.rows, self.classes, self.pairs, p(self.logits), p(self.labels), p(self.starts), p(self.loss), p(self.margins),
                                p(self.sums), p(self.work), self.work.numel(), ref_logp=p(self.ref), dlogits=p(self.logits), type=B.BF16)

    def backward(self):
        self.logits[int(self.starts_end):].zero_()   # rows behind the last sequence are still logits
        torch.mm(self.logits.T, self.join.y, out=self.dhead)
        torch.mm(self.logits, self.head16, out=self.join.dy)
        self.join.backward(self.be)
        p = lambda t: t.data_ptr()  # noqa: E731
        self.be.grad_norm(self.grad_table, MAX_NORM, p(self.norm), p(self.factor), p(self.grad_work), self.grad_work.numel())

    @property
    def starts_end(self):
        return self.join.rows - 2

    def update(self, step):
        self.be.adamw_step(self.table, params(step), grad_scale=self.factor.data_ptr())

    def step(self, step):
        self.forward()
        self.loss_and_gradient()
        self.backward()
        self.update(step)

    def everything(self):
        out = [self.join.x_out, self.join.y, self.join.dx, self.join.dblock, self.logits, self.loss, self.margins, self.sums, self.norm, self.factor,
               self.head16]
        for group in (self.weights, self.grads, self.m, self.v):
            out += list(group.values())
        return out


@pytest.fixture()
def be():
    b = B.CudaBackend(0)
    b.set_stream(torch.cuda.current_stream().cuda_stream)
    yield b
    torch.cuda.synchronize()
    b.close()


SIZES = [([1, 2], 64, 33), ([20, 31, 7, 12], 256, 1000), ([150, 120, 90, 201], 768, 5003)]


@pytest.mark.parametrize("kind,gate", [(B.NORM_LAYER, True), (B.NORM_RMS, True), (B.NORM_RMS, False)])
@pytest.mark.parametrize("lengths,d,classes", SIZES)
def test_every_stage_of_three_steps(be, lengths, d, classes, kind, gate):
    s = Step(be, kind, lengths, d, classes, gate)
    for step in (1, 2, 3):
        s.forward()
        s.join.check_forward()
        inside = s.labels.clone()
        inside[s.starts_end:] = -1
        rows = R.Rows(s.logits, inside)
        behind = s.logits[s.starts_end:].clone()
        s.loss_and_gradient()
        want = R.preference(rows, s.starts, s.ref, "sigmoid", 0.1, 0.0, 0.0, False)
        assert abs(float(s.loss) - want["loss"]) <= want["loss_off"]
        assert torch.equal(s.logits[s.starts_end:], behind)
        rows.check_dlogits(torch.cat([s.logits[:s.starts_end], torch.zeros_like(behind)]), want["slopes"], want["slopes_off"])
        s.backward()
        s.join.check_backward()
        norm, factor = norm_formula(list(s.grads.values()), float(torch.tensor(MAX_NORM)))
        assert near(float(s.norm), norm) and near(float(s.factor), factor)
        before = {k: (w.double().reshape(-1), s.grads[k].double().reshape(-1) * float(s.factor), s.m[k].double().reshape(-1), s.v[k].double().reshape(-1))
                  for k, w in s.weights.items()}
        s.update(step)
        for k, w in s.weights.items():
            check_p(w.reshape(-1), before[k][0], formula(*before[k], step, decay=k == "head")[0])
        assert torch.equal(s.head16, s.head.bfloat16())


@pytest.mark.parametrize("lengths,d,classes", SIZES)
def test_captured_and_replayed(be, lengths, d, classes):
    eager, other = (Step(be, B.NORM_LAYER, lengths, d, classes) for _ in range(2))
    for _ in range(3):
        eager.step(5)
    warm = Step(be, B.NORM_LAYER, lengths, d, classes)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):   # (the library's products set themselves up on a stream)
        be.set_stream(side.cuda_stream)
        warm.step(5)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    try:
        with torch.cuda.graph(graph, stream=side):
            other.step(5)
    finally:
        be.set_stream(torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(eager.everything(), other.everything()))


def test_two_at_once(be):
    """Two steps on two streams: neither waits for what the other holds, and both have the bits of one alone."""
    lengths, d, classes = SIZES[2]
    alone = Step(be, B.NORM_RMS, lengths, d, classes)
    for step in (1, 2):
        alone.step(step)
    torch.cuda.synchronize()
    pair = []
    for _ in range(2):
        stream, b = torch.cuda.Stream(), B.CudaBackend(0)
        b.set_stream(stream.cuda_stream)
        pair.append((stream, Step(b, B.NORM_RMS, lengths, d, classes)))
    torch.cuda.synchronize()
    for step in (1, 2):
        for stream, s in pair:
            with torch.cuda.stream(stream):
                s.step(step)
    torch.cuda.synchronize()
    for _, s in pair:
        assert all(torch.equal(a, b) for a, b in zip(alone.everything(), s.everything()))
        s.be.close()


def test_a_refused_call_does_nothing_and_says_why(be):
    s = Step(be, B.NORM_LAYER, [3, 4], 64, 50)
    s.forward()
    before = [t.clone() for t in s.everything()]
    launches = be.counters().kernel_launches
    p = lambda t: t.data_ptr()  # noqa: E731
    with pytest.raises(B.BackendError, match="preference loss: the workspace is too small"):
        be.preference_loss(9, 50, 1, p(s.logits), p(s.labels), p(s.starts), p(s.loss), p(s.margins), p(s.sums), p(s.work), 8, type=B.BF16)
    with pytest.raises(B.BackendError, match="policy loss: clip_low"):
        be.policy_loss(9, 50, p(s.logits), p(s.labels), p(s.ref), p(s.ref), p(s.loss), p(s.sums), p(s.work), 1 << 20, clip_low=2.0, type=B.BF16)
    with pytest.raises(B.BackendError, match="join forward: x and x_out overlap"):
        be.join_forward(B.NORM_RMS, 9, 64, p(s.join.x), p(s.join.block), B.join_weights(p(s.join.w["pre_gamma"])), p(s.join.x), p(s.join.y),
                        B.join_stats(p(s.join.stats["pre_rstd"])), y_type=B.BF16)
    with pytest.raises(B.BackendError, match="grad norm: max_norm"):
        be.grad_norm(s.grad_table, -1.0, p(s.norm), p(s.factor), p(s.grad_work), s.grad_work.numel())
    assert be.counters().kernel_launches == launches
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(before, s.everything()))
