"""GPU: an AdamW step over many tensors counts as a write for autograd, as torch.optim.AdamW's does -- a backward pass that saved a
parameter before the step raises an error instead of multiplying with what the parameter has become."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from neat_amd import ops  # noqa: E402
from neat_amd.optim import MultiTensorAdamW  # noqa: E402

DEV = "cuda"


@pytest.mark.parametrize("missing", [False, True])           # both ways through step()
@pytest.mark.parametrize("make", [torch.optim.AdamW, MultiTensorAdamW])
def test_a_backward_pass_behind_the_step_is_refused(make, missing):
    w, q, idle = (torch.nn.Parameter(torch.full((8,), 2.0, device=DEV)) for _ in range(3))
    opt = make([w, q, idle])
    loss = (w * w * q).sum()
    loss.backward(retain_graph=True)
    if not missing:
        idle.grad = torch.ones_like(idle)
    was = idle._version
    opt.step()
    assert (idle._version > was) == (not missing)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_the_operator_itself_counts_as_a_write():
    w = torch.nn.Parameter(torch.full((8,), 2.0, device=DEV))
    m, v = torch.zeros(1, 256, device=DEV), torch.zeros(1, 256, device=DEV)
    loss = (w * w).sum()
    ops.adamw_multi([w], [torch.ones(8, device=DEV)], [0], [1], m, v)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    assert m._version > 0 and v._version > 0


def test_inference_tensors_still_step():
    with torch.inference_mode():
        p = torch.full((8,), 2.0, device=DEV)
    opt = MultiTensorAdamW([p])
    with torch.inference_mode():
        p.grad = torch.ones(8, device=DEV)
    opt.step()
    assert (p < 2.0).all()
