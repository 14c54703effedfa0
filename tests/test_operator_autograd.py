"""CPU: operators that record nothing for autograd refuse activations that autograd follows (what they refuse next on a host
tensor is that it is one), and take them under no_grad or detached."""
import pytest
import torch

from neat_amd import ops


def z(grad):
    return torch.zeros(4, 8, requires_grad=grad)


def v(grad):
    return torch.zeros(4, requires_grad=grad)


W = torch.nn.Parameter(torch.ones(8))
T = torch.zeros(4, dtype=torch.int64)
CALLS = [
    lambda g: ops.token_logprobs(z(g), T),
    lambda g: ops.token_logprobs_bwd(z(g), T, torch.zeros(3, 4), v(False)),
    lambda g: ops.token_logprobs_bwd(z(False), T, torch.zeros(3, 4), v(g)),
    lambda g: ops.token_logprobs_bwd(z(False), T, torch.zeros(3, 4), v(False), v(g)),
    lambda g: ops.token_logprobs_bwd(z(False), T, torch.zeros(3, 4), v(False), out=z(g)),
    lambda g: ops.token_logprobs_fwd_bwd(z(g), T, v(False)),
    lambda g: ops.token_logprobs_fwd_bwd(z(False), T, v(g)),
    lambda g: ops.token_logprobs_fwd_bwd(z(False), T, v(False), out=z(g)),
    lambda g: ops.res_norm_fwd(z(g), z(False), W),
    lambda g: ops.res_norm_fwd(z(False), z(g), W),
    lambda g: ops.res_norm_fwd(z(False), z(False), W, x_out=z(g)),
    lambda g: ops.res_norm_bwd(z(g), None, z(False), z(False), torch.zeros(4, 4), W),
    lambda g: ops.res_norm_bwd(z(False), z(g), z(False), z(False), torch.zeros(4, 4), W),
    lambda g: ops.res_norm_bwd(z(False), None, z(g), z(False), torch.zeros(4, 4), W),
    lambda g: ops.res_norm_bwd(z(False), None, z(False), z(g), torch.zeros(4, 4), W),
]


@pytest.mark.parametrize("k", range(len(CALLS)))
def test_what_autograd_follows_is_refused(k):
    with pytest.raises(RuntimeError, match="records nothing for autograd"):
        CALLS[k](True)
    with pytest.raises(RuntimeError, match="no CPU path"):
        CALLS[k](False)                              # weights may be Parameters
    with torch.no_grad(), pytest.raises(RuntimeError, match="no CPU path"):
        CALLS[k](True)


def made(shape, grad):
    t = torch.nn.Parameter(torch.ones(shape))
    return torch.tanh(t) if grad else t                  # what a network has computed / a leaf


FWD = [lambda g: dict(pre_w=made(8, g)), lambda g: dict(pre_w=W, pre_b=made(8, g)), lambda g: dict(pre_w=W, post_w=made(8, g)),
       lambda g: dict(pre_w=W, post_w=W, post_b=made(8, g)), lambda g: dict(pre_w=W, scale=made(8, g)),
       lambda g: dict(pre_w=W, gate=made((2, 8), g))]


@pytest.mark.parametrize("k", range(len(FWD)))
def test_weights_and_gates_that_a_graph_has_computed_are_refused(k):
    def call(g):
        if "pre_b" in FWD[k](g):
            return ops.res_norm_fwd(z(False), z(False), **FWD[k](g))
        ops.res_norm_bwd(z(False), None, z(False), z(False), torch.zeros(4, 4), **FWD[k](g))

    def forward(g):
        return ops.res_norm_fwd(z(False), z(False), **FWD[k](g))
    for f in (call, forward):
        with pytest.raises(RuntimeError, match="records nothing for autograd"):
            f(True)
        with pytest.raises(RuntimeError, match="no CPU path"):
            f(False)
        with torch.no_grad(), pytest.raises(RuntimeError, match="no CPU path"):
            f(True)
