"""GPU: a step of MultiTensorAdamW that is refused has changed nothing, whichever list of tensors it is refused for."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from neat_amd.optim import MultiTensorAdamW  # noqa: E402

DEV = "cuda"


def state(opt, params):
    return [t.detach().clone() for t in params] + [t.clone() for t in opt._buffers()], opt._step_counts()


def not_contiguous(p):
    p.data = torch.randn(p.numel() * 2, device=DEV)[::2]


def another_type(p):
    p.data = p.data.bfloat16()


def on_the_host(p):
    p.data = p.data.cpu()


def sparse_gradient(p):
    p.grad = p.grad.to_sparse()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("spoil", [not_contiguous, another_type, on_the_host, sparse_gradient])
def test_a_refused_step_has_changed_nothing(bits, spoil):
    gen = torch.Generator(device=DEV).manual_seed(1)
    ps = [torch.nn.Parameter(torch.randn(n, generator=gen, device=DEV)) for n in (300, 5, 700)]
    opt = MultiTensorAdamW([dict(params=ps[:2]), dict(params=ps[2:], lr=1e-2)], state_bits=bits)
    for p in ps:
        p.grad = torch.randn(p.shape, generator=gen, device=DEV)
    opt.step()
    (before, counts), kept = state(opt, ps), (ps[2].data, ps[2].grad)
    spoil(ps[2])
    with pytest.raises(RuntimeError):
        opt.step()
    ps[2].grad = None
    ps[2].data, ps[2].grad = kept
    torch.cuda.synchronize()
    after, counts_after = state(opt, ps)
    assert counts == counts_after == [1, 1, 1]
    assert all(torch.equal(a, b) for a, b in zip(before, after))
    opt.step()
    assert opt._step_counts() == [2, 2, 2]
