"""The join over many rows of a few hundred columns, where a thread block has the most groups and slots.  Tolerances are test_gpu_join's."""

import pytest
import torch

from see_ai_b200 import backend as B
from test_gpu_join import PAIRS, Join

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be():
    b = B.CudaBackend(0)
    b.set_stream(torch.cuda.current_stream().cuda_stream)
    yield b
    torch.cuda.synchronize()
    b.close()


@pytest.mark.parametrize("kind", [B.NORM_LAYER, B.NORM_RMS])
@pytest.mark.parametrize("cols,stride", [(257, 257), (314, 314), (315, 320), (317, 317), (320, 321), (384, 387), (511, 511)])
def test_every_slot_of_24_groups(be, cols, stride, kind):
    for xt, yt in PAIRS:
        j = Join(kind, 30000, cols, xt, yt, x_stride=stride, y_stride=stride)
        j.forward(be)
        j.check_forward()
        j.backward(be)
        j.check_backward()
