"""CPU: the helper that reads addresses, gradients and step counts of a list of tensors (neat_host_step_list) -- what it takes, and
that it says no, without raising, to every list that is not as it was laid out."""
import array

import pytest
import torch

from neat_amd import lib


def call(params, sizes=None, bf16=False, device=-1, steps=None):
    sizes = array.array("q", [p.numel() for p in params] if sizes is None else sizes)
    n = len(sizes)
    steps = array.array("i", steps or [0] * n)
    p, g, now = array.array("Q", bytes(8 * n)), array.array("Q", bytes(8 * n)), array.array("i", bytes(4 * n))
    rc = lib.step_list()(params, n, sizes.buffer_info()[0], bf16, device, steps.buffer_info()[0], p.buffer_info()[0], g.buffer_info()[0],
                         now.buffer_info()[0])
    return rc, list(p), list(g), list(now)


def make(dtype=torch.float32):
    ps = [torch.nn.Parameter(torch.zeros(s, dtype=dtype)) for s in ((3,), (4, 5), (), (0,), (7, 1, 2))]
    for p in ps:
        p.grad = torch.ones_like(p)
    return ps


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_addresses_and_counts(dtype):
    ps = make(dtype)
    assert call(ps, bf16=dtype == torch.bfloat16, steps=[0, 5, 2, 9, 1]) == (
        1, [p.data_ptr() for p in ps], [p.grad.data_ptr() for p in ps], [1, 6, 3, 10, 2])
    assert call(ps, bf16=dtype != torch.bfloat16)[0] == 0


def test_an_empty_list():
    assert call([]) == (1, [], [], [])


def test_gradients_that_are_views_of_one_buffer():
    ps, flat = make(), torch.zeros(64)
    at = 1
    for p in ps:
        p.grad = flat[at:at + p.numel()].view_as(p)
        at += p.numel()
    rc, _, g, _ = call(ps)
    assert rc == 1 and g[0] == flat.data_ptr() + 4 and g[1] == flat.data_ptr() + 16


def test_what_is_not_as_laid_out():
    ps = make()
    assert call(tuple(ps), [p.numel() for p in ps])[0] == 0           # no list
    assert call(ps[:4], [p.numel() for p in ps])[0] == 0              # another length
    assert call(ps, [3, 20, 1, 0, 15])[0] == 0                        # another size
    assert call(ps, device=0)[0] == 0                                 # another device
    assert call(ps[:1] + [None] + ps[2:], [p.numel() for p in ps])[0] == 0
    assert call([3.0], [1])[0] == 0
    ps[2].grad = None
    assert call(ps)[0] == 0
    ps = make()
    ps[1].grad = torch.ones(5, 4).t()                                 # not contiguous
    assert call(ps)[0] == 0
    ps[1].grad = torch.ones(4, 5).to_sparse()
    assert call(ps)[0] == 0
    ps = make()
    ps[1].data = torch.zeros(4, 10)[:, ::2]                           # the parameter re-pointed to a strided view
    assert call(ps)[0] == 0
    ps = make()
    ps[1].data = torch.zeros(4, 5, dtype=torch.bfloat16)              # ... to another type
    assert call(ps)[0] == 0
    ps = make()
    ps[1].data = torch.zeros(2, 5)                                    # ... to fewer elements, the gradient left as it was
    assert call(ps, [3, 20, 1, 0, 14])[0] == 0 and call(ps, [3, 10, 1, 0, 14])[0] == 0
