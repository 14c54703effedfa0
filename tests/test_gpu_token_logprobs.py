"""GPU: log probabilities of given tokens, entropy, alternatives and gradient against the definitions in 64 bits.

Tolerances (u = 2^-24, half a step of float32).  d_j = f (x_j - m) takes two roundings and exp2 three more (its argument's
conversion and its own unit in the last place, 2u), so each term of s is off by (5 + 2|d_j|) u of itself; a lane adds at most 64
terms and the joining at most 30: s is off by (100 + 2 E|d|) u of itself, E the mean under p.  log s then by that much, its own
rounding is 2u |log s|, logp_t adds 3u |d_t|.  The entropy's second part sum(p d) is a sum of terms of one sign and is off by
(200 + ...) u of itself in the same way.  The gradient multiplies p, off by (110 + 2|d_j| + 2 E|d|) u, with a + b (logp_j + H),
whose own error is that of logp and H.  bfloat16 results round once more: half a step, 2^-8 of the value."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from neat_amd import lib, ops  # noqa: E402

DEV = "cuda"
U = 2.0 ** -24
NEG = -math.inf


def ref64(x, t, f, k=0, a=None, b=None):
    """(values, tolerances) from the definitions in 64 bits, on the CPU; rows may be masked."""
    x = x.detach().cpu().double()
    m = x.amax(1, keepdim=True)
    m = torch.where(m == NEG, torch.zeros_like(m), m)
    d = f * (x - m)
    e = torch.exp(d)
    s = e.sum(1, keepdim=True)
    none = s == 0
    p = torch.where(e > 0, e / s, torch.zeros_like(e))
    dd = torch.where(e > 0, d, torch.zeros_like(d))
    logs = torch.log(torch.where(none, torch.ones_like(s), s))
    mean = (p * dd.abs()).sum(1, keepdim=True)
    ent = torch.where(none, torch.zeros_like(s), logs + mean)
    off = (100 + 2 * mean + 2 * logs.abs()) * U                     # of log s
    tol_ent = off + (300 * mean + 4 * (p * dd * dd).sum(1, keepdim=True)) * U
    lp = torch.where(none, torch.full_like(d, NEG), d - logs)
    tol_lp = off + 3 * U * torch.where(torch.isfinite(d), d.abs(), torch.zeros_like(d))
    out = dict(ent=(ent[:, 0], tol_ent[:, 0]), lp=(lp, tol_lp))
    if t is not None:
        tc = t.cpu()
        at = tc.clamp(0, x.shape[1] - 1)[:, None]
        v = torch.where(tc < 0, torch.zeros(len(tc)).double(), lp.gather(1, at)[:, 0])
        out["logp"] = (v, tol_lp.gather(1, at)[:, 0])
    if k:
        key = torch.where(torch.isnan(x), torch.full_like(x, NEG), x)
        idx = torch.argsort(key, dim=1, descending=True, stable=True)[:, :k]
        out["idx"], out["top"] = idx, (lp.gather(1, idx), tol_lp.gather(1, idx))
    if a is not None or b is not None:
        z = torch.zeros(x.shape[0], dtype=torch.float64)
        a64 = z if a is None else torch.where(t.cpu() < 0, z, a.cpu().double())
        b64 = z if b is None else b.cpu().double()
        a64 = torch.where(none[:, 0], z, a64)
        w = torch.where(e > 0, dd - logs + ent, torch.zeros_like(d))
        g = -p * (a64[:, None] + b64[:, None] * w)
        tol = p * ((a64.abs()[:, None] + b64.abs()[:, None] * w.abs()) * (120 + 2 * dd.abs() + 2 * mean) * U
                   + b64.abs()[:, None] * (tol_ent + tol_lp + 4 * U * (logs.abs() + ent)))
        if a is not None:
            at = t.cpu().clamp(min=0)[:, None]
            g = g.scatter_add(1, at, a64[:, None])
            tol = tol.scatter_add(1, at, 4 * U * a64.abs()[:, None])
        out["dz"] = (f * g, f * tol + 2 * U * (f * g).abs() + 1e-37)
    return out


def close(got, want, what="", dtype=torch.float32):
    v, tol = want
    g = got.detach().cpu().double()
    assert torch.equal(torch.isnan(g), torch.isnan(v)), what
    assert torch.equal(g == NEG, v == NEG), what
    ok = torch.isfinite(v)
    assert torch.isfinite(g[ok]).all(), what
    bound = tol[ok] + (2.0 ** -8 * v[ok].abs() if dtype == torch.bfloat16 else 0)
    over = (g[ok] - v[ok]).abs() > bound
    assert not over.any(), (what, g[ok][over][:4], v[ok][over][:4], bound[over][:4])


def logits(R, V, dtype, seed, scale=1.0, pad=0, off=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    wide = torch.full((R, V + pad + off), 7.0, dtype=dtype, device=DEV)
    z = wide[:, off:off + V]
    z.copy_(torch.randn(R, V, generator=gen, device=DEV) * (2.5 if scale == 1.0 else 0.04))
    return z, torch.randint(0, V, (R,), generator=gen, device=DEV), wide


def weights(R, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(R, generator=gen, device=DEV), torch.randn(R, generator=gen, device=DEV)


SHAPES = [(1, 1), (3, 2), (5, 7), (5, 33), (4, 511), (2, 2048), (3, 2049), (2, 4097), (2, 8192), (3, 8193), (2, 16384), (3, 16385),
          (2, 32768), (2, 32769), (1, 49408), (2, 57345), (2, 65536), (2, 65537), (1, 140001)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("R,V", SHAPES)
def test_forward_and_alternatives(R, V, dtype):
    for k, scale, pad, off in ((0, 1.0, 0, 0), (1, 1.0, 1, 0), (min(5, V), 100.0, 0, 0), (min(32, V), 1.0, 5, 3)):
        z, t, _ = logits(R, V, dtype, V + k, scale, pad, off)
        want = ref64(z, t, scale, k)
        logp, ent, stats, top, idx = ops.token_logprobs(z, t, scale=scale, k=k)
        close(logp, want["logp"], ("logp", k))
        close(ent, want["ent"], ("ent", k))
        if k:
            assert torch.equal(idx.cpu().long(), want["idx"]), k
            close(top, want["top"], ("top", k))
        else:
            assert top is None and idx is None


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("R,V", SHAPES)
def test_gradient(R, V, dtype):
    for scale, pad, off in ((1.0, 0, 0), (100.0, 5, 3)):
        z, t, wide = logits(R, V, dtype, 3 * V, scale, pad, off)
        a, b = weights(R, V)
        if R > 2:
            t[1] = -1
        want = ref64(z, t, scale, 0, a, b)
        logp, ent, stats, _, _ = ops.token_logprobs(z, t, scale=scale)
        close(ops.token_logprobs_bwd(z, t, stats, a, b, scale=scale), want["dz"], "bwd", dtype)
        logp2, ent2, dz = ops.token_logprobs_fwd_bwd(z, t, a, b, scale=scale)
        close(dz, want["dz"], "fwd_bwd", dtype)
        close(logp2, want["logp"]), close(ent2, want["ent"])
        # one weight alone
        close(ops.token_logprobs_bwd(z, None, stats, None, b, scale=scale), ref64(z, t, scale, 0, None, b)["dz"], "b", dtype)
        close(ops.token_logprobs_fwd_bwd(z, t, a, None, scale=scale)[2], ref64(z, t, scale, 0, a, None)["dz"], "a", dtype)
        # into a wider buffer, whose other columns stay, and over the logits themselves
        out = torch.full_like(wide, 3.0)
        view = out[:, off:off + V]
        ops.token_logprobs_bwd(z, t, stats, a, b, scale=scale, out=view)
        close(view, want["dz"], "strided", dtype)
        assert (out[:, :off] == 3.0).all() and (out[:, off + V:] == 3.0).all()
        copy = wide.clone()
        cz = copy[:, off:off + V]
        assert ops.token_logprobs_fwd_bwd(cz, t, a, b, scale=scale, out=cz)[2] is cz
        close(cz, want["dz"], "in place", dtype)
        assert (copy[:, :off] == 7.0).all() and (copy[:, off + V:] == 7.0).all()
        ops.token_logprobs_bwd(z, t, stats, a, b, scale=scale, out=z)
        close(z, want["dz"], "in place, alone", dtype)


def test_gradient_against_differences():
    """Central differences of the 64-bit value: off by h^2/6 of the third derivative (|.| <= 8 f^3 (|a| + 12 |b|) here) and by
    1e-15 / h of the value's rounding."""
    z, t, _ = logits(4, 21, torch.float32, 5)
    a, b = weights(4, 6)
    _, _, dz = ops.token_logprobs_fwd_bwd(z, t, a, b, scale=1.25)
    h, want = 1e-4, ref64(z, t, 1.25, 0, a, b)["dz"]

    def value(x):
        r = ref64(x, t, 1.25)
        return (a.cpu().double() * r["logp"][0] + b.cpu().double() * r["ent"][0])
    for j in range(21):
        up, dn = z.cpu().double().clone(), z.cpu().double().clone()
        up[:, j] += h
        dn[:, j] -= h
        num = (value(up) - value(dn)) / (2 * h)
        lim = h * h / 6 * 8 * 1.25 ** 3 * (a.abs() + 12 * b.abs()).cpu().double() + 2e-11 + want[1][:, j]
        assert ((dz[:, j].cpu().double() - num).abs() <= lim).all(), j


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [40, 3000, 9000, 40000, 70000])
def test_ties_go_to_the_lowest_index(V, dtype):
    gen = torch.Generator(device=DEV).manual_seed(V)
    z = torch.randint(-3, 4, (4, V), generator=gen, device=DEV).to(dtype)
    z[1] = 1.5                                              # a row of equal values
    z[2] = torch.where(torch.arange(V, device=DEV) % 2 == 0, 0.0, -0.0).to(dtype)     # both zeros are one value
    z[3] = torch.arange(V, device=DEV).to(dtype)            # ascending (bfloat16: long runs of one value)
    for k in (1, 4, 32):
        _, _, _, top, idx = ops.token_logprobs(z, None, k=k)
        want = ref64(z, None, 1.0, k)
        assert torch.equal(idx.cpu().long(), want["idx"])
        close(top, want["top"])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [40, 1000, 9000, 49408])
def test_alternatives_on_both_sides_of_zero(V, dtype):
    """Rows below zero, rows whose k-th alternative is next to zero, and rows with fewer unmasked entries than alternatives."""
    gen = torch.Generator(device=DEV).manual_seed(V)
    z = torch.randn(6, V, generator=gen, device=DEV)
    z[0] = -z[0].abs() - 1
    z[1] = -z[1].abs() * 1e30
    z[2] = torch.where(torch.arange(V, device=DEV) < 7, z[2].abs(), -z[2].abs())
    z[3] = torch.where(torch.arange(V, device=DEV) % 9 == 0, z[3].abs() * 1e-30, -z[3].abs() * 1e-30)
    z[4] = torch.where(torch.arange(V, device=DEV) < 3, z[4], NEG)
    z[5] = -(torch.arange(V, device=DEV).float() + 1)
    z = z.to(dtype)
    for k in (1, 7, 8, 32):
        _, _, _, top, idx = ops.token_logprobs(z, None, k=k)
        want = ref64(z, None, 1.0, k)
        assert torch.equal(idx.cpu().long(), want["idx"]), k
        close(top, want["top"])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [2048, 8192, 16384, 32768, 65536])
def test_alternatives_that_one_lane_holds(V, dtype):
    """The largest values sit where single lanes, or single groups of lanes, read: the most candidates a row can have."""
    gen = torch.Generator(device=DEV).manual_seed(V)
    rows = []
    for period, run in ((256, 4), (1024, 8), (2048, 16), (4096, 16), (8192, 32), (8192, 8)):
        z = torch.randn(V, generator=gen, device=DEV)
        at = torch.arange(V, device=DEV)
        z[at % period < run] += 50 + torch.rand(int((at % period < run).sum()), generator=gen, device=DEV)
        rows.append(z)
    z = torch.stack(rows).to(dtype)
    for k in (3, 32):
        _, _, _, top, idx = ops.token_logprobs(z, None, k=k)
        want = ref64(z, None, 1.0, k)
        assert torch.equal(idx.cpu().long(), want["idx"])
        close(top, want["top"])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [5, 40, 3000, 20000, 70001])
def test_masks(V, dtype):
    R = 9
    z, t, _ = logits(R, V, dtype, V)
    gen = torch.Generator(device=DEV).manual_seed(1)
    lowest = torch.finfo(dtype).min
    z.masked_fill_(torch.rand(z.shape, generator=gen, device=DEV) < 0.5, NEG)
    z[0] = NEG                                              # nothing left
    z[1] = NEG
    z[1, V - 1] = -3.0                                      # one left, the last
    z[2] = lowest                                           # masked by the type's lowest value: uniform
    z[3] = lowest
    z[3, V // 2] = 2.0
    z[4, 0], z[4, 1] = math.nan, 0.5
    z[5] = math.nan
    z[6, V - 1] = math.inf
    z[7, :] = z[7].nan_to_num(neginf=lowest)
    z[8, 0] = 1.0
    t[7] = -1
    a, b = weights(R, 3)
    k = min(5, V)
    logp, ent, stats, top, idx = ops.token_logprobs(z, t, k=k)
    want = ref64(z, t, 1.0, k, a, b)
    fine = [0, 1, 2, 3, 7, 8]
    bad = [4, 5, 6]
    assert torch.equal(idx.cpu().long(), want["idx"])       # NaN is last, with the masked places
    cut = lambda w: (w[0][fine], w[1][fine])  # noqa: E731
    close(logp[fine], cut(want["logp"])), close(ent[fine], cut(want["ent"])), close(top[fine], cut(want["top"]))
    assert torch.isnan(logp[bad]).all() and torch.isnan(ent[bad]).all() and torch.isnan(top[bad]).all()
    for dz in (ops.token_logprobs_bwd(z, t, stats, a, b), ops.token_logprobs_fwd_bwd(z, t, a, b)[2]):
        close(dz[fine], cut(want["dz"]), "dz", dtype)
        assert (dz[0] == 0).all() and torch.isnan(dz[bad]).all()
    assert float(ent[0]) == 0 and float(logp[0]) == NEG and float(ent[1]) == 0


def test_a_target_that_no_row_has_shows():
    z, t, _ = logits(3, 50, torch.float32, 1)
    t[1] = 50
    a, b = weights(3, 1)
    logp, ent, stats, _, _ = ops.token_logprobs(z, t)
    dz = ops.token_logprobs_bwd(z, t, stats, a, b)
    assert torch.isnan(logp[1]) and torch.isfinite(logp[[0, 2]]).all() and torch.isfinite(ent).all()
    assert torch.isnan(dz[1]).all() and torch.isfinite(dz[[0, 2]]).all()


def test_rows_that_overlap_the_same_storage_and_empty_batches():
    z, t, _ = logits(1, 300, torch.float32, 2)
    with pytest.raises(RuntimeError, match="overlap"):
        ops.token_logprobs(z.expand(4, 300), t.expand(4).contiguous())
    with pytest.raises(RuntimeError, match="adjacent"):
        ops.token_logprobs(torch.zeros(8, 5, device=DEV).t())
    e = torch.empty(0, 300, device=DEV)
    logp, ent, stats, top, idx = ops.token_logprobs(e, torch.empty(0, dtype=torch.int64, device=DEV), k=3)
    assert logp.shape == (0,) and top.shape == (0, 3)
    assert ops.token_logprobs_bwd(e, None, stats, None, ent).shape == (0, 300)


def test_repeats_are_equal_bit_for_bit():
    z, t, _ = logits(64, 70001, torch.bfloat16, 9)
    a, b = weights(64, 9)
    one = (*ops.token_logprobs(z, t, k=32), ops.token_logprobs_fwd_bwd(z, t, a, b)[2])
    for _ in range(3):
        two = (*ops.token_logprobs(z, t, k=32), ops.token_logprobs_fwd_bwd(z, t, a, b)[2])
        assert all(torch.equal(x, y) for x, y in zip(one, two))


@pytest.mark.parametrize("V", [5000, 70001])
def test_on_another_stream_and_in_a_graph(V):
    z, t, _ = logits(6, V, torch.float32, 11)
    a, b = weights(6, 11)

    def both():
        logp, ent, stats, top, idx = ops.token_logprobs(z, t, k=7)
        return logp, ent, top, idx, ops.token_logprobs_bwd(z, t, stats, a, b), *ops.token_logprobs_fwd_bwd(z, t, a, b)
    want = both()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = both()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(x, y) for x, y in zip(want, got))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = both()
    for seed in (12, 13, 14):
        z.copy_(logits(6, V, torch.float32, seed)[0])
        want = both()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(want, held))


def test_limits_of_length():
    L = lib.load()
    assert L.neat_token_logprobs(64, 1 << 30, 0, None, 1.0, 0, None, 64, None, None, None, 2, (1 << 21) + 1, 64, None) == -1
    V = 2097152                                             # the longest float32 row: 64 pieces
    z, t, _ = logits(2, V, torch.float32, 21)
    want = ref64(z, t, 1.0, 32)
    logp, ent, stats, top, idx = ops.token_logprobs(z, t, k=32)
    assert torch.equal(idx.cpu().long(), want["idx"])
    close(logp, want["logp"]), close(ent, want["ent"]), close(top, want["top"])


def test_offsets_beyond_32_bits():
    """A row pitch that puts the last row 4.4 GB behind the first: only the rows' own bytes are touched."""
    pitch = 1_100_000_000
    buf = torch.empty(pitch * 4 + 1000, dtype=torch.bfloat16, device=DEV)
    z = buf.as_strided((5, 1000), (pitch, 1))
    z.copy_(torch.randn(5, 1000, device=DEV))
    t = torch.randint(0, 1000, (5,), device=DEV)
    a, b = weights(5, 1)
    want = ref64(z, t, 1.0, 3, a, b)
    logp, ent, stats, top, idx = ops.token_logprobs(z, t, k=3)
    assert torch.equal(idx.cpu().long(), want["idx"])
    close(logp, want["logp"]), close(top, want["top"])
    ops.token_logprobs_bwd(z, t, stats, a, b, out=z)
    close(z, want["dz"], "far", torch.bfloat16)
