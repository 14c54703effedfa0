"""GPU: AdamW over many tensors (neat_adamw_multi, optim.MultiTensorAdamW) against the rule in 64 bits.

Tolerances (u = 2^-24, half a step of float32): a moment takes at most three roundings a step, each relative to a value no larger
than the largest of |m|, |g| (or |v|, g^2) seen, so |err m| <= 3 u k max(|m|, |g|) after k steps; the step divides it by the
denominator and adds eight roundings of its own (sqrt, two divisions, the rates, the products), the parameter two more.  bfloat16
parameters round once more: seven bits behind the leading one, numbers of [1, 2) lie 2^-7 apart, so by up to 2^-8 of the value.  8-bit moments: half a step of e4m3, 2^-4 of the value, or half of
its smallest number, 2^-10 of the block's power of two."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from neat_amd import ops  # noqa: E402
from neat_amd.optim import MultiTensorAdamW  # noqa: E402

DEV = "cuda"
U = 2.0 ** -24
LR, B1, B2, EPS, WD = 2e-3, 0.9, 0.999, 1e-8, 1e-2


def _params(sizes, dtype, seed, bucket=False):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    if bucket:                                       # views of one buffer that start at any element
        flat = (torch.randn(1 + sum(sizes), generator=gen, device=DEV) * 0.1).to(dtype)
        out, at = [], 1
        for n in sizes:
            out.append(torch.nn.Parameter(flat[at:at + n]))
            at += n
        return out
    return [torch.nn.Parameter((torch.randn(n, generator=gen, device=DEV) * 0.1).to(dtype)) for n in sizes]


def _grads(params, seed, bucket=False):
    for p, g in zip(params, _params([p.numel() for p in params], params[0].dtype, seed, bucket)):
        p.grad = (g.detach() if bucket else g.detach().clone()).view_as(p)


def _step64(p, g, m, v, k):
    """One step in 64 bits -> (p, m, v, the denominator)."""
    p, g = p.double(), g.double()
    m = m + (g - m) * (1 - B1)
    v = v * B2 + g * g * (1 - B2)
    d = torch.sqrt(v) / math.sqrt(1 - B2 ** k) + EPS
    return p * (1 - LR * WD) - LR / (1 - B1 ** k) * m / d, m, v, d


def _p_bound(p, m, g, d, k, dtype):
    step = LR / (1 - B1 ** k) / d
    b = 3 * U * p.abs() + step * (3 * U * torch.maximum(m.abs(), g.double().abs()) + 8 * U * m.abs()) + 1e-37
    return b + (2.0 ** -8 * (1 + 8 * U) * p.abs() if dtype == torch.bfloat16 else 0)


SIZES = [1, 2, 3, 4, 5, 255, 256, 257, 512, 1023, 4096, 70001]


@pytest.mark.parametrize("bucket", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_moments_in_32_bits(dtype, bucket):
    ps = _params(SIZES, dtype, 1, bucket)
    opt = MultiTensorAdamW(ps, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD)
    ms = [torch.zeros(p.shape, dtype=torch.float64, device=DEV) for p in ps]
    vs = [torch.zeros_like(m) for m in ms]
    top = [torch.zeros_like(m) for m in ms]
    for k in range(1, 5):
        _grads(ps, 10 + k, bucket)
        before = [p.detach().clone() for p in ps]
        opt.step()
        for i, p in enumerate(ps):
            g = p.grad
            want, ms[i], vs[i], d = _step64(before[i], g, ms[i], vs[i], k)
            top[i] = torch.maximum(top[i], g.double().abs())
            m, v, steps = opt.moments(p)
            assert steps == k
            assert ((m.double() - ms[i]).abs() <= 3 * U * k * top[i]).all()
            assert ((v.double() - vs[i]).abs() <= 3 * U * k * top[i] ** 2 + 1e-44).all()
            # the moments' own error enters the step: top instead of this step's gradient, k steps of it
            bound = _p_bound(want, ms[i], top[i] * k, d, k, dtype) + LR / (1 - B1 ** k) * ms[i].abs() / d * 3 * U * k * top[i] ** 2 / vs[i].clamp_min(1e-300)
            assert ((p.double() - want).abs() <= bound).all(), (i, k)
    assert all((opt._m.view(-1)[lo * 256 + n:(lo + -(-n // 256)) * 256] == 0).all() for lo, n in zip(opt._first, opt._numel))


@pytest.mark.parametrize("bucket", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_moments_in_8_bits(dtype, bucket):
    """Every step is compared with the 64-bit step from the state that the codes stand for."""
    ps = _params(SIZES, dtype, 2, bucket)
    opt = MultiTensorAdamW(ps, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD, state_bits=8)
    for k in range(1, 5):
        _grads(ps, 20 + k, bucket)
        for p in ps[:3]:
            p.grad.mul_(1e-6)                        # and a gradient far below its block's largest
        ps[-1].grad[::300] *= 1e-7
        before = [p.detach().clone() for p in ps]
        held = []
        for p, lo, n in zip(ps, opt._first, opt._numel):
            rows = slice(lo, lo + -(-n // 256))
            m = opt.exp_avg[rows].double() * opt.exp_avg_scale[rows, None].double()
            r = opt.exp_avg_root[rows].double() * opt.exp_avg_root_scale[rows, None].double()
            held.append((m.view(-1)[:n].view(p.shape), (r * r).view(-1)[:n].view(p.shape)))
        opt.step()
        for i, p in enumerate(ps):
            want, m, v, d = _step64(before[i], p.grad, *held[i], k)
            # the decoded root squared is rounded once more before it is used
            bound = _p_bound(want, m, p.grad, d, k, dtype) + LR / (1 - B1 ** k) * m.abs() / d * 4 * U
            bound += LR / (1 - B1 ** k) / d * 2 * U * held[i][0].abs()
            assert ((p.double() - want).abs() <= bound).all(), (i, k)
            lo, n = opt._first[i], p.numel()
            nb = -(-n // 256)
            for code, scale, x in ((opt.exp_avg, opt.exp_avg_scale, m), (opt.exp_avg_root, opt.exp_avg_root_scale, torch.sqrt(v))):
                s = scale[lo:lo + nb].double()
                full = torch.zeros(nb * 256, dtype=torch.float64, device=DEV)
                full[:n] = x.reshape(-1)
                full = full.view(nb, 256)
                big = full.abs().amax(1)
                assert torch.equal(torch.exp2(torch.round(torch.log2(s))), s)
                assert ((big <= 448 * s * (1 + 8 * U)) & ((big > 224 * s * (1 - 8 * U)) | (s == 2.0 ** -126))).all()
                got = code[lo:lo + nb].double() * s[:, None]
                slack = 2.0 ** -4 * full.abs() + 2.0 ** -10 * s[:, None]
                if x is not m:
                    assert ((got > 0) | (full == 0)).all()                 # a root above zero stays above zero
                    slack = torch.where((full > 0) & (full < 2.0 ** -9 * s[:, None]), 2.0 ** -9 * s[:, None], slack)
                assert ((got - full).abs() <= slack * (1 + 16 * U)).all()


def test_codes_follow_nearest_even_like_torch():
    """All codes of a block: the kernel's rounding is torch's own float8_e4m3fn conversion."""
    g = torch.linspace(-448, 448, 4096, device=DEV)
    g[::256] = 448.0                                 # every block's power of two is 2^0 for m = g (beta1 = 0)
    p = torch.nn.Parameter(torch.zeros(4096, device=DEV))
    p.grad = g.clone()
    opt = MultiTensorAdamW([p], lr=0.0, betas=(0.0, 0.5), weight_decay=0.0, state_bits=8)
    opt.step()
    assert (opt.exp_avg_scale == 1).all()
    assert torch.equal(opt.exp_avg.view(-1).float(), g.to(torch.float8_e4m3fn).float())
    assert torch.equal(p.detach(), torch.zeros_like(p))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_codes_of_roots_are_those_of_the_exact_roots(dtype):
    """16 million roots: next to no border between two codes is one rounded to the other side (32 bits alone round a few there).
    Second moments are normal here, and no block's largest is at a border of the scales."""
    n = 1 << 22
    p = torch.nn.Parameter(torch.zeros(n, device=DEV, dtype=dtype))
    opt = MultiTensorAdamW([p], lr=0.0, betas=(B1, B2), weight_decay=0.0, state_bits=8)
    gen = torch.Generator(device=DEV).manual_seed(8)
    was = torch.zeros(n // 256, 256, dtype=torch.float64, device=DEV)
    for _ in range(4):
        p.grad = (torch.randn(n, generator=gen, device=DEV) * torch.exp(torch.randn(n, generator=gen, device=DEV)) * 1e-3).to(dtype)
        opt.step()
        scale = opt.exp_avg_root_scale.view(-1, 1).double()
        q = torch.sqrt(was ** 2 * B2 + p.grad.double().view(-1, 256) ** 2 * (1 - B2)) / scale
        step = torch.exp2(torch.floor(torch.log2(q.clamp(min=2.0 ** -6))) - 3)
        want = torch.where(q > 0, (torch.round(q / step) * step).clamp(min=2.0 ** -9), q)
        got = opt.exp_avg_root.view(-1, 256).double()
        assert torch.equal(got, want), int((got != want).sum())
        was = got * scale


@pytest.mark.parametrize("bits", [32, 8])
def test_what_is_not_finite_stays_where_it_is(bits):
    p, q = _params([700, 700], torch.float32, 3)
    p.grad, q.grad = torch.full_like(p, 0.5), torch.full_like(q, 0.5)
    p.grad[5], p.grad[300], p.grad[301] = math.nan, math.inf, -math.inf
    opt = MultiTensorAdamW([p, q], lr=LR, state_bits=bits)
    start = p.detach().clone()
    opt.step()
    bad = torch.zeros(700, dtype=torch.bool, device=DEV)
    bad[[5, 300, 301]] = True
    assert torch.equal(~torch.isfinite(p), bad) and torch.isfinite(q).all()
    m, v, _ = opt.moments(p)
    assert torch.equal(~torch.isfinite(m), bad) and torch.equal(~torch.isfinite(v), bad)
    # |step| = lr for a first step without decay beside the default decay's 1 - lr wd
    assert ((p - start * (1 - LR * 1e-2)).abs()[~bad] - LR).abs().max() < 1e-6


@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors_groups_missing_gradients_and_mixed_types(bits):
    a = _params([17 + 3 * i for i in range(100)], torch.float32, 4)
    b = _params([300] * 130, torch.bfloat16, 5)
    one = [torch.nn.Parameter(p.detach().clone()) for p in a + b]
    every = a + b
    opt = MultiTensorAdamW([dict(params=every[:150], lr=1e-2, weight_decay=0.0), dict(params=every[150:], lr=1e-3)], state_bits=bits)
    for k in range(3):
        _grads(a, 40 + k)
        _grads(b, 50 + k)
        if k == 1:
            for p in every[::7]:
                p.grad = None
        for p, q in zip(every, one):
            q.grad = None if p.grad is None else p.grad.clone()
        opt.step()
        if k == 0:
            alone = [MultiTensorAdamW([q], lr=1e-2 if i < 150 else 1e-3, weight_decay=0.0 if i < 150 else 1e-2, state_bits=bits)
                     for i, q in enumerate(one)]
        for o in alone:
            o.step()
    for i, (p, q) in enumerate(zip(every, one)):
        assert torch.equal(p, q), i                  # together and one at a time give the same bits
        assert opt.moments(p)[2] == (2 if i % 7 == 0 else 3) == alone[i].moments(q)[2]


def test_against_the_flat_optimizer_and_torch():
    from neat_amd.optim import AdamW
    a = _params([512] * 12, torch.float32, 6)
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    c = [torch.nn.Parameter(p.detach().clone()) for p in a]
    oa, ob, oc = MultiTensorAdamW(a, lr=LR), AdamW(b, lr=LR), torch.optim.AdamW(c, lr=LR)
    for k in range(3):
        _grads(a, 60 + k)
        for p, q, r in zip(a, b, c):
            q.grad.copy_(p.grad)
            r.grad = p.grad.clone()
        oa.step(), ob.step(), oc.step()
    for p, q, r in zip(a, b, c):
        # three steps, each with at most 3 roundings of the parameter and 16 of the step (|step| <= 4 lr here)
        tol = 3 * (3 * U * p.abs() + 16 * U * 4 * LR)
        assert ((p - q).abs() <= tol).all() and ((p - r).abs() <= tol).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_state_dict_carries_on(bits):
    a = _params([5, 300, 1000], torch.float32, 7)
    oa = MultiTensorAdamW(a, lr=LR, state_bits=bits)
    for k in range(2):
        _grads(a, 70 + k)
        oa.step()
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    ob = MultiTensorAdamW(b, lr=1.0, state_bits=bits)
    import copy
    ob.load_state_dict(copy.deepcopy(oa.state_dict()))
    assert ob.param_groups[0]["lr"] == LR
    _grads(a, 79)
    for p, q in zip(a, b):
        q.grad = p.grad.clone()
    oa.step(), ob.step()
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    with pytest.raises(ValueError):
        MultiTensorAdamW(b, state_bits=40 - bits).load_state_dict(oa.state_dict())


def test_on_another_stream_and_refused_in_a_capture():
    a = _params([300, 5000], torch.float32, 8)
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    _grads(a, 80)
    for p, q in zip(a, b):
        q.grad = p.grad.clone()
    oa, ob = MultiTensorAdamW(a), MultiTensorAdamW(b)
    oa.step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ob.step()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="graph would replay"):
        with torch.cuda.graph(graph):
            oa.step()
    torch.cuda.synchronize()
    assert oa.moments(a[0])[2] == 1                  # a refused step is not counted


def test_transposed_gradient_empty_tensor_and_refusals():
    w, e = torch.nn.Parameter(torch.randn(7, 9, device=DEV)), torch.nn.Parameter(torch.empty(0, device=DEV))
    w2 = torch.nn.Parameter(w.detach().clone())
    g = torch.randn(9, 7, device=DEV)
    w.grad, e.grad, w2.grad = g.t(), torch.empty(0, device=DEV), g.t().contiguous()
    MultiTensorAdamW([w, e]).step()
    MultiTensorAdamW([w2]).step()
    assert torch.equal(w, w2)
    with pytest.raises(ValueError):
        MultiTensorAdamW([w], state_bits=16)
    with pytest.raises(ValueError):
        MultiTensorAdamW([w, w])
    with pytest.raises(RuntimeError):
        MultiTensorAdamW([torch.nn.Parameter(torch.zeros(3, dtype=torch.float16, device=DEV))])
    with pytest.raises(RuntimeError):
        MultiTensorAdamW([torch.nn.Parameter(torch.zeros(4, 3, device=DEV).t())])
    opt = MultiTensorAdamW([w])
    with pytest.raises(RuntimeError):
        opt.add_param_group(dict(params=[w2]))
    m = torch.zeros(1, 256, device=DEV)
    with pytest.raises(RuntimeError, match="outside"):
        ops.adamw_multi([w], [w.grad.contiguous()], [1], [1], m, torch.zeros_like(m))
    with pytest.raises(RuntimeError, match="step=0"):
        ops.adamw_multi([w], [w.grad.contiguous()], [0], [0], m, torch.zeros_like(m))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("g", [1e-10, 1e-18, 1e-19, 1e-20])
def test_gradients_whose_square_is_subnormal(bits, g):
    """The second moment (1e-3 g^2) is a subnormal float32 here, which holds it to 2^-149: off by at most 2^-150 / (1e-3 g^2) of
    itself, the step by half of that.  It stays above zero, and the step is no larger than with any other gradient."""
    p = torch.nn.Parameter(torch.zeros(300, device=DEV))
    p.grad = torch.full_like(p, g)
    p.grad[::7] = 0.0
    opt = MultiTensorAdamW([p], lr=LR, betas=(B1, B2), eps=1e-30, weight_decay=0.0, state_bits=bits)
    opt.step()
    m, v, _ = opt.moments(p)
    some = p.grad > 0
    rel = 16 * U + 0.5 * 2.0 ** -150 / (1e-3 * g * g) * 1.01
    assert ((p.detach().double() / -LR - 1).abs()[some] <= rel + g * 0).all() and (p[~some] == 0).all()
    if bits == 32:
        assert ((v > 0) == some).all()
    else:
        assert ((opt.exp_avg_root.float().view(-1)[:300] > 0) == some).all()


def test_a_scalar_parameter_and_a_closure():
    p = torch.nn.Parameter(torch.tensor(2.0, device=DEV))
    opt = MultiTensorAdamW([p], lr=LR, weight_decay=0.0)

    def closure():
        opt.zero_grad()
        loss = 3.0 * p
        loss.backward()
        return loss
    assert float(opt.step(closure)) == 6.0
    assert abs(float(p) - (2.0 - LR)) <= 4 * U and opt.moments(p)[0].shape == ()
