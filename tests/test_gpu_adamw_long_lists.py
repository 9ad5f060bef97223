"""AdamW over lists long enough that a thread block sweeps a range of its own, fills its slots again and again and moves over the ends
of tensors of many blocks and of one; over more tensors than one launch takes; and the evenness of the 8-bit cut over elements."""

import numpy as np
import pytest
import torch

from see_ai_b200 import backend as B
from test_gpu_adamw_tensors import Tensors, params
from test_gpu_adamw_tensors import test_step as check_step

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be():
    b = B.CudaBackend(0)
    b.set_stream(torch.cuda.current_stream().cuda_stream)
    yield b
    torch.cuda.synchronize()
    b.close()


# 17000 blocks, five for each warp of 148 SMs.  Sizes of whole 16-byte runs up to the last but one, so that every tensor goes
# through the copies; the same with one element more each, so that few do.
MIXED = [2_000_016] + [112] * 150 + [1_500_000] + [304, 0, 16] * 10 + [900_016, 17]
# 417 tensors that are not empty, 192 to a launch, some empty where the list is split.
MANY = [704] * 190 + [0, 0, 0] + [256 * 40 + 16] * 2 + [0] + [528] * 220 + [30000] * 5


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("sizes,launches", [(MIXED, 1), ([n + 1 if n else 0 for n in MIXED], 1), (MANY, 3)], ids=["mixed", "odd", "many"])
@pytest.mark.parametrize("grad,copy", [("bf16", "bf16"), ("f32", "f32")])
def test_long_list(be, bits, sizes, launches, grad, copy):
    before = be.counters().kernel_launches
    check_step(be, bits, sizes, grad, copy, 0)
    assert be.counters().kernel_launches - before == launches


def test_list_in_one_call_and_tensor_by_tensor(be):
    """Two steps; every stored byte the same, the scales too."""
    for bits in (32, 8):
        whole, single = (Tensors(MIXED, bits, "f16", "f16", seed=4) for _ in range(2))
        for step in (7, 8):
            be.adamw_step(whole.table(no_decay={0, 200}), params(step), state_bits=bits)
            table = single.table(no_decay={0, 200})
            for i in range(len(table)):
                be.adamw_step((B.AdamWTensor * 1)(table[i]), params(step), state_bits=bits)
        for a, b in zip(whole.buffers(), single.buffers()):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_cut_is_even_over_elements(be):
    """Element i's offset is i phi mod 1 (and a constant of the step).  Of N consecutive multiples of a number whose partial quotients
    are at most K, the count in any interval is off by at most 3 + (1 / log phi + K / log(K + 1)) log N (Kuipers and Niederreiter,
    Uniform Distribution of Sequences, theorem 2.3.4): K = 1 for phi, to 32 bits, up to denominators of 28657, 2 at 75025; 7 for
    256 phi, every 256th element, up to 443.  The elements between the blocks' largest are off by the sum of both.  A value is a
    cut 1/8 of it from its neighbour at most; the cut's last place is 2^-20 of that, the value's own roundings a few 2^-22."""
    n = 65536
    count_off = sum(3 + (1 / np.log((1 + 5 ** 0.5) / 2) + k / np.log(k + 1)) * np.log(terms) for k, terms in ((1, n), (7, n // 256)))
    t = Tensors([n], 8, zero=True)
    keep = torch.ones(n, dtype=torch.bool, device="cuda")
    keep[::256] = False
    kept = n - n // 256
    for value in (3.1e-3, 7.77e-4, 1.03e-3):
        t.g.fill_(value)
        t.g[::256] = 1e-2                       # the blocks' largest
        g = t.g[1].item()
        for step in (1, 2, 1000):
            for b in (t.m, t.v):
                b.view(torch.uint8).zero_()
            be.adamw_step(t.table(), params(step), state_bits=8)
            _, _, m, v = t.values(0)
            for got, exact in ((m, (1 - float(np.float32(0.9))) * g), (v.sqrt(), g * (1 - float(np.float32(0.999))) ** 0.5)):
                assert abs(got[keep].mean().item() / exact - 1) <= 0.125 * (count_off / kept + 2.0 ** -20) + 16 * 2.0 ** -24
                assert got[keep].unique().numel() == 2
