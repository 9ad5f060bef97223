"""Norm and clipping over lists with empty tensors in any place, around the sizes at which a launch's table is full.  Tolerances are
test_gpu_grad_norm's."""

import pytest
import torch

from see_ai_b200 import backend as B
from test_gpu_grad_norm import DTYPES, Call, check_out, formula, near

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be():
    b = B.CudaBackend(0)
    b.set_stream(torch.cuda.current_stream().cuda_stream)
    yield b
    torch.cuda.synchronize()
    b.close()


@pytest.mark.parametrize("empty", [(0, 0, 1), (0, 0, 200), (3, 0, 0), (0, 170, 0), (2, 1, 160)])
@pytest.mark.parametrize("count", [159, 160, 161, 320])
def test_empty_tensors_anywhere(be, count, empty):
    torch.manual_seed(count + sum(empty))
    types = list(DTYPES.values())
    full = [(torch.randn(17 + 331 * (i % 40), device="cuda") * 3).to(types[i % 3]) for i in range(count)]
    none = torch.empty(0, device="cuda", dtype=torch.bfloat16)
    front, between, behind = empty
    tensors = [none] * front + full[:count // 2] + [none] * between + full[count // 2:] + [none] * behind
    want = formula(tensors, 0.5)
    c = Call(be, 0.5)
    norm, factor = c(tensors)
    assert near(norm, want[0]) and near(factor, want[1])
    outs = [torch.full_like(t, 9.0) for t in tensors]
    assert c(tensors, outs, clip=True) == (norm, factor)
    for t, out in zip(tensors, outs):
        check_out(t, out, factor)
