"""GPU: parameters that share memory are refused when the optimizer is built -- one launch would update both at once, in any order."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from neat_amd.optim import MultiTensorAdamW  # noqa: E402

DEV = "cuda"


def test_parameters_that_share_memory_are_refused():
    flat = torch.zeros(1000, device=DEV)
    one, two, three = (torch.nn.Parameter(flat[a:b]) for a, b in ((0, 300), (299, 600), (600, 1000)))
    tied = torch.nn.Parameter(flat[600:1000].view(20, 20))
    for ps in ([one, two], [two, one, three], [three, tied], [dict(params=[one, tied]), dict(params=[three])]):
        with pytest.raises(ValueError, match="share memory"):
            MultiTensorAdamW(ps)


def test_neighbours_and_empty_parameters_are_not():
    flat = torch.zeros(1000, device=DEV)
    ps = [torch.nn.Parameter(flat[a:b]) for a, b in ((0, 300), (300, 600), (450, 450), (600, 1000))]
    opt = MultiTensorAdamW(ps, lr=1e-3, weight_decay=0.0)
    for p in ps:
        p.grad = torch.ones_like(p)
    opt.step()
    assert ((flat + 1e-3).abs() < 1e-6).all()
