"""GPU: the largest and smallest scales that are taken."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from neat_amd import ops  # noqa: E402

DEV = "cuda"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [5, 3000, 70000])
def test_the_ends_of_the_range(V, dtype):
    z = torch.full((3, V), -1.0, dtype=dtype, device=DEV)
    z[0, 2], z[1, 1], z[2, 3] = 1.0, 0.5, 0.0
    t, a = torch.tensor([2, 1, 3], device=DEV), torch.ones(3, device=DEV)
    # every other exponential is exactly zero: the row's own largest has probability 1
    logp, ent, dz = ops.token_logprobs_fwd_bwd(z, t, a, a, scale=2.0 ** 100)
    assert (logp == 0).all() and (ent == 0).all() and (dz == 0).all()
    # and all are alike: log V to within the roundings of a sum of V ones (exact below 2^24) and a logarithm
    logp, ent, dz = ops.token_logprobs_fwd_bwd(z, t, a, None, scale=1e-37)
    lim = 8 * 2.0 ** -24 * math.log(V)
    assert (logp + math.log(V)).abs().max() <= lim and (ent - math.log(V)).abs().max() <= lim and torch.isfinite(dz).all()
