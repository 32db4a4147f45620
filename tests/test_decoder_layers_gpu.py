"""The decoder layers against a plain form of a layer, and what a step keeps and takes."""
import gc

import pytest
import torch

from test_decoder_gpu import BF, _decoder, _lens, _x

pytestmark = pytest.mark.gpu


def test_a_step_keeps_no_memory(dip):
    """Steps of ever new lengths leave nothing behind on the GPU."""
    dec = _decoder()
    rel = torch.ones(3, dtype=torch.bool, device="cuda")
    x = _x(150, 1)

    def steps(counts):
        for n in counts:
            dec.step(x[:n], _lens(n, 0, 0), n)
            dec.release(rel)
        torch.cuda.synchronize()
        gc.collect()
        return torch.cuda.memory_allocated()

    steps([1, 8, 40, 150])
    before = steps([1])
    assert steps(list(range(2, 150, 9)) + [1]) == before   # (the cache holds the last step's slots)


def test_norm_is_the_inputs_own(dip):
    """To the bit what a residual of zeros gives."""
    from dip_b200.stack import RMS_EPS
    dec = _decoder()
    for size in (1.0, 1e-4, 2.0 ** 60, 2.0 ** -60):
        x = (_x(9, 4).float() * size).to(BF)
        want = torch.ops.dip_b200.residual_rmsnorm(x, torch.zeros_like(x), RMS_EPS)
        assert torch.equal(dec._norm(x), want)


def test_first_step_of_a_length_inside_a_capture(dip):
    """A length that a graph capture sees first is served outside it as any other."""
    x0, x = _x(40, 2), _x(21, 3)
    want = _decoder()
    want.step(x0, _lens(40, 0, 0), 40)
    y = want.step(x, _lens(0, 21, 0), 21)
    dec = _decoder()
    dec.step(x0, _lens(40, 0, 0), 40)
    new = _lens(0, 21, 0)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        dec.step(x, new, 21)
    assert torch.equal(dec.step(x, new, 21), y)
