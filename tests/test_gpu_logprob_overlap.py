"""GPU: gradients written between the rows of the logits, beside them or over them give what a buffer of their own gives; those that
overlap them otherwise are refused and leave the logits alone."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from neat_amd import ops  # noqa: E402

DEV = "cuda"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [5, 300, 5000, 70000])
def test_beside_between_and_over_the_logits(V, dtype):
    gen = torch.Generator(device=DEV).manual_seed(V)
    R, a = 4, torch.randn(4, generator=gen, device=DEV)
    t = torch.randint(0, V, (R,), generator=gen, device=DEV)
    z0 = torch.randn(R, V, generator=gen, device=DEV).to(dtype)
    want = ops.token_logprobs_fwd_bwd(z0, t, a, a)[2]

    def layouts():
        buf = torch.zeros(R, 2 * V + 3, dtype=dtype, device=DEV)
        yield buf[:, :V], buf[:, V:2 * V]                     # columns of one buffer
        yield buf[:, V + 1:2 * V + 1], buf[:, 1:V + 1]
        buf = torch.zeros(2 * R, V, dtype=dtype, device=DEV)
        yield buf[::2], buf[1::2]                             # rows in turn
        yield buf[:R], buf[R:]
        flat = torch.zeros(R * (V + 2) + 2 * R * V + 2 * V, dtype=dtype, device=DEV)
        yield flat.as_strided((R, V), (V + 2, 1)), flat.as_strided((R, V), (2 * V, 1), R * (V + 2))
        yield buf[:R], buf[:R]
    for z, out in layouts():
        z.copy_(z0)
        _, _, stats, _, _ = ops.token_logprobs(z, t)
        ops.token_logprobs_bwd(z, t, stats, a, a, out=out)
        two = out.clone()
        z.copy_(z0)
        assert torch.equal(ops.token_logprobs_fwd_bwd(z, t, a, a, out=out)[2], want)
        close = (two.float() - want.float()).abs() <= 2.0 ** -7 * want.float().abs() + 1e-6
        assert close.all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("off", [1, 40, 299, 300])
def test_other_overlaps_are_refused(off, dtype):
    R, V = 3, 300
    flat = torch.randn(R * V + off, device=DEV).to(dtype)
    z, out, was = flat[:R * V].view(R, V), flat[off:].view(R, V), flat.clone()
    t, a = torch.zeros(R, dtype=torch.int64, device=DEV), torch.ones(R, device=DEV)
    _, _, stats, _, _ = ops.token_logprobs(z, t)
    for call in (lambda p, q: ops.token_logprobs_bwd(p, t, stats, a, out=q), lambda p, q: ops.token_logprobs_fwd_bwd(p, t, a, out=q)):
        for p, q in ((z, out), (out, z)):
            with pytest.raises(RuntimeError, match="overlaps"):
                call(p, q)
    assert torch.equal(flat, was)
