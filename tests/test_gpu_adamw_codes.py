"""GPU: the codes that 8-bit first moments get (optim.MultiTensorAdamW), on every step, against the rule in exact arithmetic.

A first moment is M = m0 + (g - m0) w, with m0 = code x power of two held, g the gradient and w = 1 - beta1 as a float64.  Its code
is the e4m3 number nearest to M, even for ties.  Where M lies next to the middle c of two codes, the sign of M - c decides, which
float64 gives exactly: m0 - c and a = g - m0 are short numbers, w is cut into w1 (24 bits) and w2 (29), a w1 and a w2 have at most 53
bits each, and (m0 - c) + a w1 loses nothing to rounding next to the middle, where the two nearly cancel."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from neat_amd.optim import MultiTensorAdamW  # noqa: E402

DEV = "cuda"


def codes(m0, g, w, scale):
    """(e4m3 numbers of the exact moments, how many of them rounding in 32 bits gets wrong) -- float64 [blocks, 256], scale
    [blocks, 1]."""
    w1 = float(torch.tensor(w, dtype=torch.float32))
    a = g - m0
    q = (m0 + a * w) / scale
    step = torch.exp2(torch.floor(torch.log2(q.abs().clamp(min=2.0 ** -6))) - 3)
    low = torch.floor(q / step)
    side = (m0 - (low + 0.5) * step * scale + a * w1) + a * (w - w1)
    up = torch.where(side == 0, low % 2 != 0, side > 0)
    want = (low + up.double()) * step
    m32 = m0.float() + (g.float() - m0.float()) * torch.tensor(w, dtype=torch.float32, device=DEV)
    return want, int(((m32 / scale.float()).to(torch.float8_e4m3fn).double() != want).sum())


@pytest.mark.parametrize("beta1", [0.9, 0.95, 0.5])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_codes_of_first_moments_are_those_of_the_exact_moments(dtype, beta1):
    n = 1 << 20
    gen = torch.Generator(device=DEV).manual_seed(9)
    p = torch.nn.Parameter(torch.zeros(n, device=DEV, dtype=dtype))
    opt = MultiTensorAdamW([p], lr=0.0, betas=(beta1, 0.999), weight_decay=0.0, state_bits=8)
    held, ties = torch.zeros(n // 256, 256, dtype=torch.float64, device=DEV), 0
    # gradients of the same size as the moment, or larger and smaller, the same one twice among them: what is short lands in the
    # middle between two codes (bfloat16: a few per cent of all moments)
    g = torch.zeros(n, device=DEV, dtype=dtype)
    for k in range(6):
        if k != 1:
            g = (torch.randn(n, generator=gen, device=DEV) * torch.exp(torch.randn(n, generator=gen, device=DEV)) * 1e-3).to(dtype)
        p.grad = g
        opt.step()
        scale = opt.exp_avg_scale.double().view(-1, 1)
        want, wrong = codes(held, g.double().view(-1, 256), 1.0 - beta1, scale)
        got = opt.exp_avg.double().view(-1, 256)
        assert torch.equal(got, want), (k, int((got != want).sum()))
        held, ties = got * scale, ties + wrong
    if dtype == torch.bfloat16 and beta1 != 0.5:
        assert ties > 1000                               # the inputs do reach what is tested
