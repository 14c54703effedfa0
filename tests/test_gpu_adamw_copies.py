"""GPU: copies and pickles of MultiTensorAdamW carry its moments and step counts, and a state that does not fit is refused whole."""
import copy
import io
import pickle

import pytest
import torch

pytestmark = pytest.mark.gpu

from neat_amd.optim import MultiTensorAdamW  # noqa: E402

DEV = "cuda"


class Net(torch.nn.Module):
    def __init__(self, bits):
        super().__init__()
        gen = torch.Generator(device=DEV).manual_seed(3)
        make = lambda n, t: torch.nn.Parameter(torch.randn(n, generator=gen, device=DEV).to(t))  # noqa: E731
        self.a, self.b, self.c = make(300, torch.float32), make(1000, torch.bfloat16), make(7, torch.float32)
        self.opt = MultiTensorAdamW([dict(params=[self.a, self.b], lr=1e-2), dict(params=[self.c])], state_bits=bits)


def steps(net, seed, count=2):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    for k in range(count):
        for p in net.parameters():
            p.grad = torch.randn(p.shape, generator=gen, device=DEV).to(p.dtype)
        if k == 0:
            net.c.grad = None
        net.opt.step()


def pickled(net):
    return pickle.loads(pickle.dumps(net))


def saved(net):
    f = io.BytesIO()
    torch.save(net, f)
    f.seek(0)
    return torch.load(f, weights_only=False)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("how", [copy.deepcopy, pickled, saved])
def test_copies_go_on_where_the_original_was(how, bits):
    net = Net(bits)
    steps(net, 1)
    twin = how(net)
    assert twin.opt._step_counts() == net.opt._step_counts() == [2, 2, 1] and twin.opt.param_groups[0]["lr"] == 1e-2
    assert twin.opt.param_groups[0]["params"][0] is twin.a and twin.a is not net.a
    steps(net, 2), steps(twin, 2)
    for p, q in zip(net.parameters(), twin.parameters()):
        assert torch.equal(p, q) and p.data_ptr() != q.data_ptr()
        assert all(torch.equal(s, t) for s, t in zip(net.opt.moments(p)[:2], twin.opt.moments(q)[:2]))
    assert twin.opt.exp_avg.data_ptr() == twin.opt._m.data_ptr() != net.opt._m.data_ptr()
    with pytest.raises(RuntimeError):
        twin.opt.add_param_group(dict(params=[torch.nn.Parameter(torch.zeros(3, device=DEV))]))


@pytest.mark.parametrize("bits", [32, 8])
def test_a_state_that_does_not_fit_is_refused_whole(bits):
    net, other = Net(bits), Net(bits)
    steps(net, 1)
    good = copy.deepcopy(net.opt.state_dict())
    for g in other.opt.param_groups:
        g["lr"] = 0.5
    for spoil in (lambda s: s["buffers"].pop(), lambda s: s["steps"].pop(), lambda s: s["buffers"].__setitem__(1, s["buffers"][1][:1])):
        bad = copy.deepcopy(good)
        spoil(bad["state"])
        with pytest.raises(ValueError, match="laid out"):
            other.opt.load_state_dict(bad)
        assert [g["lr"] for g in other.opt.param_groups] == [0.5, 0.5] and other.opt._step_counts() == [0, 0, 0]
        assert not other.opt._m.any()
    other.opt.load_state_dict(good)
    assert other.opt._step_counts() == [2, 2, 1] and all(torch.equal(s, t) for s, t in zip(other.opt._buffers(), net.opt._buffers()))
