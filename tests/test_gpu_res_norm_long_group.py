"""GPU: the gates' gradients of res_norm_bwd where one sequence holds most rows among a thousand short or empty ones.

Every term of a gate's gradient is the same number here, e n = (1.1f * 0.7f), so that roundings of a sum go the same way and add up:
a long chain of additions is off by hundreds of u (u = 2^-24), which random terms hide.  A sum is formed of a run's rows (at most 8 a
team at these sizes), the runs' sums in 16 slices (the longest group has 1 907 of them: 120 a slice) and the slices: 8 + 120 + 16
additions, each off by u of a partial sum no larger than the whole; the product and the scale are two roundings more."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from neat_amd import ops  # noqa: E402

DEV = "cuda"
U = 2.0 ** -24
ROWS, COLS = 14851, 768


def lengths(kind):
    if kind == "among short ones":
        return [1] * 500 + [ROWS - 1020] + [1] * 520
    if kind == "among empty ones":
        return [0] * 700 + [ROWS - 3] + [0] * 317 + [3, 0, 0]
    if kind == "two neighbours":
        return [1] * 10 + [7000, 0, 6841] + [1] * 1000 + [0] * 8
    return [900] * 16 + [451] + [0] * 1004                    # a workgroup of long ones


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["among short ones", "among empty ones", "two neighbours", "sixteen together"])
def test_equal_terms(kind, dtype):
    n = torch.tensor(lengths(kind))
    assert int(n.sum()) == ROWS and len(n) == 1021
    cu = torch.cat([torch.zeros(1, dtype=torch.int64), n.cumsum(0)]).to(torch.int32).to(DEV)
    h = torch.full((ROWS, COLS), 0.7, device=DEV).to(dtype)
    zero, one = torch.zeros(ROWS, COLS, device=DEV), torch.ones(COLS, device=DEV)
    gate = torch.ones(1021, COLS, device=DEV)
    dres = torch.full_like(zero, 1.1)
    x_out, _, stats = ops.res_norm_fwd(zero, h, one, gate=gate, cu=cu, kind="rms")
    _, _, g = ops.res_norm_bwd(zero.to(dtype), dres, h, x_out, stats, one, gate=gate, cu=cu, kind="rms")
    want = (n.double() * float(dres[0, 0]) * float(h[0, 0]))[:, None].to(DEV)
    off = ((g["gate"].double() - want).abs() / want.clamp_min(1e-300)).amax(1)
    assert (off <= (8 + 120 + 16 + 2) * U).all(), float(off.max() / U)
    assert (g["gate"][n == 0] == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["among short ones", "among empty ones", "two neighbours", "sixteen together"])
def test_random_terms_and_repeats(kind, dtype):
    n = torch.tensor(lengths(kind))
    cu = torch.cat([torch.zeros(1, dtype=torch.int64), n.cumsum(0)]).to(torch.int32).to(DEV)
    gen = torch.Generator(device=DEV).manual_seed(5)
    h = torch.randn(ROWS, COLS, generator=gen, device=DEV).to(dtype)
    dres, scale = torch.randn(ROWS, COLS, generator=gen, device=DEV), torch.randn(COLS, generator=gen, device=DEV)
    gate = torch.randn(1021, COLS, generator=gen, device=DEV)
    zero, one = torch.zeros(ROWS, COLS, device=DEV), torch.ones(COLS, device=DEV)
    x_out, _, stats = ops.res_norm_fwd(zero, h, one, scale=scale, gate=gate, cu=cu)
    runs = [ops.res_norm_bwd(zero.to(dtype), dres, h, x_out, stats, one, scale=scale, gate=gate, cu=cu)[2] for _ in range(2)]
    assert all(torch.equal(runs[0][k], runs[1][k]) for k in runs[0])
    of = torch.repeat_interleave(torch.arange(1021, device=DEV), n.to(DEV))
    terms, sums = dres.double() * h.double(), torch.zeros(1021, COLS, dtype=torch.float64, device=DEV)
    want, size = sums.index_add(0, of, terms) * scale.double(), sums.index_add(0, of, terms.abs()) * scale.double().abs()
    assert ((runs[0]["gate"].double() - want).abs() <= (8 + 120 + 16 + 3) * U * size).all()
