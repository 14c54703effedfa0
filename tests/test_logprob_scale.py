"""CPU: scales above 2^100 are refused before anything is launched: products of the scale overflow there, and 0 times infinity is NaN (in
gradients from 2^120, in every result from 2^127).  Addresses are made up."""
import pytest

from neat_amd import lib


@pytest.mark.parametrize("scale", [1.3e30, 1e36, 2.4e38, 3.4e38])
def test_scales_that_overflow_are_refused(scale):
    L = lib.load()
    for rc in (L.neat_token_logprobs(64, 100, 0, 64, scale, 0, 64, 64, 64, None, None, 4, 100, None, None),
               L.neat_token_logprobs_bwd(64, 100, 0, 64, 64, 64, 64, scale, 64, 100, 4, 100, None),
               L.neat_token_logprobs_fwd_bwd(64, 100, 0, 64, 64, 64, scale, 64, 64, 64, 64, 100, 4, 100, None, None)):
        assert rc == -2 and "scale" in lib.last_error()
