"""CPU: calls that the operators refuse are refused before anything is launched (no GPU is needed to see it)."""
import ctypes

import pytest
import torch

from neat_amd import lib, ops
from neat_amd.optim import MultiTensorAdamW


def _arr(kind, *v):
    return (kind * len(v))(*v)


def _adamw(count=1, p=64, g=64, n=10, block=0, step=1, dtype=0, m=64, v=64, ms=64, vs=64, bits=32):
    return lib.load().neat_adamw_multi(count, _arr(ctypes.c_void_p, p), _arr(ctypes.c_void_p, g), _arr(ctypes.c_int64, n),
                                       _arr(ctypes.c_int64, block), _arr(ctypes.c_int32, step), dtype, m, v, ms, vs, bits, 1e-3,
                                       0.9, 0.999, 1e-8, 0.0, None)


@pytest.mark.parametrize("bad, rc, says", [
    (dict(count=-1), -1, "count"), (dict(p=None), -2, "null"), (dict(g=None), -2, "null"), (dict(m=None), -2, "null"),
    (dict(n=-1), -1, "n=-1"), (dict(n=1 << 40), -1, "too large"), (dict(block=-1), -1, "state_block"),
    (dict(block=1 << 32), -1, "too large"), (dict(step=0), -1, "step=0"), (dict(dtype=7), -2, "dtype"),
    (dict(bits=4), -2, "state_bits"), (dict(bits=8, ms=None), -2, "scales"), (dict(m=68), -2, "aligned"),
    (dict(p=66), -2, "aligned"), (dict(p=65, dtype=1), -2, "aligned")])
def test_adamw_multi_checks_before_launching(bad, rc, says):
    assert _adamw(**bad) == rc
    assert says in lib.last_error()


def test_adamw_multi_without_tensors_is_nothing():
    assert _adamw(count=0) == 0
    assert _adamw(n=0, p=None, g=None) == 0


def test_adamw_multi_wrapper_refuses():
    p, m = torch.zeros(5), torch.zeros(1, 256)
    with pytest.raises(RuntimeError, match="GPU"):
        ops.adamw_multi([p], [p], [0], [1], m, m.clone())
    with pytest.raises(RuntimeError, match="one gradient"):
        ops.adamw_multi([p], [], [0], [1], m, m.clone())
    with pytest.raises(RuntimeError, match="float32 or bfloat16"):
        ops.adamw_multi([p.double()], [p.double()], [0], [1], m, m.clone())
    with pytest.raises(RuntimeError, match="all be"):
        ops.adamw_multi([p], [p.bfloat16()], [0], [1], m, m.clone())
    with pytest.raises(RuntimeError, match="contiguous"):
        ops.adamw_multi([torch.zeros(4, 3).t()], [torch.zeros(3, 4)], [0], [1], m, m.clone())
    with pytest.raises(RuntimeError, match="size"):
        ops.adamw_multi([p], [torch.zeros(6)], [0], [1], m, m.clone())
    with pytest.raises(RuntimeError, match="outside"):
        ops.adamw_multi([p], [p], [1], [1], m, m.clone())
    with pytest.raises(RuntimeError, match="m and v"):
        ops.adamw_multi([p], [p], [0], [1], m, torch.zeros(1, 128))
    with pytest.raises(RuntimeError, match="m_scale"):
        ops.adamw_multi([p], [p], [0], [1], m.to(torch.uint8), m.to(torch.uint8))
    with pytest.raises(RuntimeError, match="GPU"):
        MultiTensorAdamW([torch.nn.Parameter(p)])
    with pytest.raises(ValueError):
        MultiTensorAdamW([torch.nn.Parameter(p)], betas=(0.9, 1.0))
    with pytest.raises(ValueError):
        MultiTensorAdamW([torch.nn.Parameter(p)], lr=-1.0)
