"""GPU: outputs that a caller passes to an operator count as written in place for autograd."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from neat_amd import ops  # noqa: E402

DEV = "cuda"


def test_outputs_that_are_passed_in_count_as_written():
    z, t, a = torch.randn(4, 8, device=DEV), torch.zeros(4, dtype=torch.int64, device=DEV), torch.ones(4, device=DEV)
    out, w = torch.zeros_like(z), torch.ones(8, device=DEV)
    _, _, stats, _, _ = ops.token_logprobs(z, t)
    for call, written in ((lambda: ops.token_logprobs_bwd(z, t, stats, a, out=out), (out,)),
                          (lambda: ops.token_logprobs_fwd_bwd(z, t, a, out=out), (out,)),
                          (lambda: ops.res_norm_fwd(z, z, w, x_out=out), (out,)),
                          (lambda: ops.token_logprobs_fwd_bwd(z, t, a, out=z), (z,))):
        before = [q._version for q in written]
        call()
        assert all(q._version > b for q, b in zip(written, before))
    x_out, _, stats = ops.res_norm_fwd(z, z, w)
    before, kept = out._version, z._version
    ops.res_norm_bwd(z, None, z, x_out, stats, w, dx=out)
    assert out._version > before and z._version == kept


def test_a_graph_that_saved_the_logits_sees_that_they_are_overwritten():
    leaf = torch.randn(4, 8, device=DEV, requires_grad=True)
    z = leaf * 2.0
    loss = (z * z).sum()
    with torch.no_grad():
        ops.token_logprobs_fwd_bwd(z, torch.zeros(4, dtype=torch.int64, device=DEV), torch.ones(4, device=DEV), out=z)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
