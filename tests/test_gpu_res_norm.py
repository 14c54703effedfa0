"""GPU: the norms around a block with its gate and residual scale (ops.res_norm_fwd / _bwd) against the formulas in 64 bits.

Tolerances (u = 2^-24, half a step of float32).  A sum over a row's columns takes at most 16 additions in a lane (times four
values added first) and 10 across lanes and waves: off by 28 u of the sum of magnitudes.  So the mean is off by 28 u mean|v|, a
centred value by that and its own rounding, the deviation's reciprocal by 24 u of itself (half of the sum's 28 u, the division,
eps, the root's own unit), and uh by  r (28 u mean|v|) + 30 u |uh|.  The backward formulas are followed term by term in the same
way (``unit_bwd``).  Sums over rows add up to ten rows a team for the sizes here, 4 teams, up to 96 workgroups a slice and 16
slices: 126 u of the sum of magnitudes, and each term's own error.  A group's slots are at most 126 here in the same way.  Each test compares with the 64-bit result of what the kernel itself read (x_out,
h), so that errors do not compound.  bfloat16 results round once more: 2^-8 of the value."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from neat_amd import ops  # noqa: E402

DEV = "cuda"
U = 2.0 ** -24
HALF = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8}
EPS = 1e-5


def unit(v, kind):
    """(uh, 1/deviation, tolerance of uh) in 64 bits."""
    mu = v.mean(1, keepdim=True) if kind == "ln" else torch.zeros(len(v), 1, dtype=v.dtype, device=v.device)
    r = 1 / torch.sqrt(((v - mu) ** 2).mean(1, keepdim=True) + EPS)
    uh = (v - mu) * r
    shift = 28 * U * v.abs().mean(1, keepdim=True) if kind == "ln" else 0.0
    return uh, r, r * shift + 30 * U * uh.abs()


def unit_bwd(z, tz, uh, tuh, r, kind):
    """N'(d) for z = d w (off by tz) and its tolerance."""
    m1 = z.mean(1, keepdim=True) if kind == "ln" else torch.zeros_like(r)
    t1 = (28 * U * z.abs().mean(1, keepdim=True) + tz.mean(1, keepdim=True)) if kind == "ln" else torch.zeros_like(r)
    q = z * uh
    m2 = q.mean(1, keepdim=True)
    t2 = 30 * U * q.abs().mean(1, keepdim=True) + (tz * uh.abs() + z.abs() * tuh).mean(1, keepdim=True)
    out = r * (z - m1 - uh * m2)
    tol = r * (tz + t1 + uh.abs() * t2 + tuh * m2.abs() + 4 * U * (z.abs() + m1.abs() + (uh * m2).abs())) + 30 * U * out.abs()
    return out, tol


def make(rows, cols, dtype, kind, post, scale, gate, seed, shift=0.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    p = dict(pre_w=1 + 0.3 * r(cols), post_w=1 + 0.3 * r(cols) if post else None, post_b=0.2 * r(cols) if post else None,
             scale=0.5 + 0.2 * r(cols) if scale else None, gate=None, cu=None, kind=kind)
    pre_b = 0.2 * r(cols)
    if gate == "even":
        n = next(k for k in (7, 5, 3, 2, 1) if rows % k == 0)
        p["gate"] = r(n, cols)
    elif gate == "each":
        p["gate"] = r(rows, cols)
    elif gate == "one":
        p["gate"] = r(1, cols)
    elif gate == "ragged":                               # lengths of zero and one among them, an empty one first and last
        cut = sorted(torch.randint(0, rows + 1, (9,), generator=torch.Generator().manual_seed(seed)).tolist() + [0, min(1, rows)])
        cu = [0] + cut + [rows, rows]
        p["gate"], p["cu"] = r(len(cu) - 1, cols), torch.tensor(cu, dtype=torch.int32, device=DEV)
    x, h = r(rows, cols) * 1.5 + shift, (r(rows, cols) + shift).to(dtype)
    return x, h, pre_b, p, (r(rows, cols)).to(dtype), r(rows, cols)


def group_rows(p, rows):
    """Group of every row, or None."""
    if p["gate"] is None:
        return None
    n = p["gate"].shape[0]
    if p["cu"] is None:
        return torch.arange(rows, device=DEV) // (rows // n)
    return torch.repeat_interleave(torch.arange(n, device=DEV), (p["cu"][1:] - p["cu"][:-1]).long())


def within(got, want, tol, what, dtype=torch.float32):
    d, lim = (got.double() - want).abs(), tol + HALF[dtype] * want.abs() + 2 * U * want.abs() + 1e-38
    assert (d <= lim).all(), (what, float(d.max()), float((d / lim).max()))


def check(rows, cols, dtype, kind, post, scale, gate, seed=0, shift=0.0):
    x, h, pre_b, p, dy, dres = make(rows, cols, dtype, kind, post, scale, gate, seed, shift)
    x_out, y, stats = ops.res_norm_fwd(x, h, p["pre_w"], pre_b, eps=EPS, **{k: v for k, v in p.items() if k != "pre_w"})
    D = lambda t: t.double()  # noqa: E731
    of = group_rows(p, rows)
    f = torch.ones(1, cols, dtype=torch.float64, device=DEV)
    if of is not None:
        f = f * D(p["gate"])[of]
    if scale:
        f = f * D(p["scale"])
    if post:
        hh, r1, th = unit(D(h), kind)
        n = hh * D(p["post_w"]) + D(p["post_b"])
        tn = D(p["post_w"]).abs() * th + 3 * U * ((hh * D(p["post_w"])).abs() + D(p["post_b"]).abs())
    else:
        hh, r1, th, n = None, None, None, D(h)
        tn = torch.zeros_like(n)
    within(x_out, D(x) + n * f, tn * f.abs() + 4 * U * (n * f).abs(), "x_out")
    xh, r2, tx = unit(D(x_out), kind)
    within(y, xh * D(p["pre_w"]) + D(pre_b), D(p["pre_w"]).abs() * tx + 3 * U * ((xh * D(p["pre_w"])).abs() + D(pre_b).abs()), "y", dtype)

    args = {k: v for k, v in p.items() if k != "pre_w"}
    dx, dh, gr = ops.res_norm_bwd(dy, dres, h, x_out, stats, p["pre_w"], **args)
    z = D(dy) * D(p["pre_w"])
    b, tb = unit_bwd(z, U * z.abs(), xh, tx, r2, kind)
    e, te = D(dres) + b, tb + 2 * U * D(dres).abs()
    within(dx, e, te, "dx")
    dn, tdn = e * f, te * f.abs() + 3 * U * (e * f).abs()
    a, ta = e * n, te * n.abs() + e.abs() * tn + 2 * U * (e * n).abs()

    def col(name, term, tol):
        within(gr[name], term.sum(0), tol.sum(0) + 126 * U * term.abs().sum(0), name)
    col("pre_w", D(dy) * xh, D(dy).abs() * tx + U * (D(dy) * xh).abs())
    col("pre_b", D(dy), torch.zeros_like(b))
    if post:
        z1 = dn * D(p["post_w"])
        v, tv = unit_bwd(z1, tdn * D(p["post_w"]).abs() + 2 * U * z1.abs(), hh, th, r1, kind)
        within(dh, v, tv, "dh", dtype)
        col("post_w", dn * hh, tdn * hh.abs() + dn.abs() * th + U * (dn * hh).abs())
        col("post_b", dn, tdn)
    else:
        within(dh, dn, tdn, "dh", dtype)
    if scale:
        w = D(p["gate"])[of] if of is not None else torch.ones(1, cols, dtype=torch.float64, device=DEV)
        col("scale", a * w, ta * w.abs() + 4 * U * (a * w).abs())
    if of is not None:
        s = D(p["scale"]) if scale else torch.ones(cols, dtype=torch.float64, device=DEV)
        zero = torch.zeros_like(D(p["gate"]))
        want = zero.index_add(0, of, a) * s
        tol = (zero.index_add(0, of, ta) + 126 * U * zero.index_add(0, of, a.abs())) * s.abs() + 2 * U * want.abs()
        within(gr["gate"], want, tol, "gate")
    assert set(gr) == {"pre_w", "pre_b"} | ({"post_w", "post_b"} if post else set()) | ({"scale"} if scale else set()) | (
        {"gate"} if of is not None else set())


GATES = [None, "one", "even", "each", "ragged"]


@pytest.mark.parametrize("rows,cols", [(1, 4), (3, 64), (2, 68), (77, 256), (5, 260), (130, 512), (7, 516), (64, 768), (33, 1024),
                                       (9, 1028), (40, 1280), (17, 1664), (12, 2048), (5, 2052), (21, 3000), (11, 4096), (1, 4096)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_sizes(rows, cols, dtype):
    for i, gate in enumerate(GATES):
        check(rows, cols, dtype, ("ln", "rms")[i % 2], i % 3 != 2, i % 4 != 1, gate, seed=rows + i)
        check(rows, cols, dtype, ("rms", "ln")[i % 2], i % 3 == 2, i % 4 == 1, gate, seed=rows + i + 9)


@pytest.mark.parametrize("gate", GATES)
@pytest.mark.parametrize("scale", [False, True])
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("kind", ["ln", "rms"])
def test_every_combination(kind, post, scale, gate):
    check(301, 512, torch.bfloat16, kind, post, scale, gate, seed=5)
    check(60, 1536, torch.float32, kind, post, scale, gate, seed=6)


@pytest.mark.parametrize("gate", GATES)
@pytest.mark.parametrize("rows,cols,dtype", [(9001, 512, torch.bfloat16), (20011, 64, torch.float32), (9001, 768, torch.bfloat16),
                                             (5003, 1280, torch.bfloat16), (4001, 1024, torch.float32), (2503, 4096, torch.bfloat16)])
def test_more_rows_than_teams(rows, cols, dtype, gate):
    """Every team has several rows, and groups begin and end inside and between teams."""
    check(rows, cols, dtype, "ln", True, True, gate, seed=rows)


def test_more_rows_than_the_largest_grid_has_teams_for():
    """2.2 million short rows forward: several thousand more than two rows for each of the 2^20 teams."""
    rows, cols = (1 << 21) + 50_003, 8
    x, h, pre_b, p, _, _ = make(rows, cols, torch.bfloat16, "ln", True, True, None, 5)
    x_out, y, stats = ops.res_norm_fwd(x, h, p["pre_w"], pre_b, eps=EPS, **{k: v for k, v in p.items() if k != "pre_w"})
    for cut in (slice(0, 5000), slice(rows // 2, rows // 2 + 5000), slice(rows - 60_000, rows)):
        got = ops.res_norm_fwd(x[cut].contiguous(), h[cut].contiguous(), p["pre_w"], pre_b, eps=EPS,
                               **{k: v for k, v in p.items() if k != "pre_w"})
        assert torch.equal(x_out[cut], got[0]) and torch.equal(y[cut], got[1]) and torch.equal(stats[:, cut], got[2])


def test_far_from_zero_and_constant_rows():
    check(20, 512, torch.float32, "ln", True, True, None, seed=7, shift=300.0)
    x = torch.full((4, 256), 3.0, device=DEV)
    h = torch.zeros(4, 256, device=DEV)
    w, b = torch.ones(256, device=DEV), torch.full((256,), 0.25, device=DEV)
    x_out, y, st = ops.res_norm_fwd(x, h, w, b, post_w=w, post_b=b)
    assert torch.equal(x_out, x + 0.25) and torch.equal(y, torch.full_like(y, 0.25))
    dx, dh, g = ops.res_norm_bwd(torch.ones_like(h), None, h, x_out, st, w, post_w=w, post_b=b)
    assert torch.isfinite(dx).all() and torch.isfinite(dh).all() and all(torch.isfinite(t).all() for t in g.values())


def test_what_is_not_finite_stays_in_its_row():
    x, h, pre_b, p, dy, dres = make(50, 512, torch.float32, "ln", True, True, "ragged", 8)
    h[20, 3] = float("nan")
    h[21, 5] = float("inf")
    args = {k: v for k, v in p.items() if k != "pre_w"}
    x_out, y, st = ops.res_norm_fwd(x, h, p["pre_w"], pre_b, **args)
    dx, dh, _ = ops.res_norm_bwd(dy, dres, h, x_out, st, p["pre_w"], **args)
    keep = [i for i in range(50) if i not in (20, 21)]
    for t in (x_out, y, dx, dh):
        assert torch.isfinite(t[keep]).all() and not torch.isfinite(t[20]).any() and not torch.isfinite(t[21]).any()


@pytest.mark.parametrize("cols", [512, 1280])
def test_rows_behind_the_last_sequence(cols):
    rows, used = 90, 61
    x, h, pre_b, p, dy, dres = make(rows, cols, torch.bfloat16, "ln", True, True, None, 9)
    p["gate"] = torch.randn(4, cols, device=DEV)
    p["cu"] = torch.tensor([0, 10, 10, 33, used], dtype=torch.int32, device=DEV)
    args = {k: v for k, v in p.items() if k != "pre_w"}
    x_out, y, st = ops.res_norm_fwd(x, h, p["pre_w"], pre_b, **args)
    dx, dh, g = ops.res_norm_bwd(dy, dres, h, x_out, st, p["pre_w"], **args)
    for t in (x_out, y, dx, dh):
        assert (t[used:] == 0).all() and torch.isfinite(t[:used].float()).all()
    # the same as on the used rows alone: other rows take no part in any sum
    short = ops.res_norm_fwd(x[:used].contiguous(), h[:used].contiguous(), p["pre_w"], pre_b, **args)
    assert torch.equal(x_out[:used], short[0]) and torch.equal(y[:used], short[1])
    want = ops.res_norm_bwd(dy[:used].contiguous(), dres[:used].contiguous(), h[:used].contiguous(), short[0], short[2], p["pre_w"], **args)
    assert torch.equal(dx[:used], want[0]) and torch.equal(dh[:used], want[1])
    for k in g:
        assert torch.allclose(g[k], want[2][k], rtol=0, atol=float(120 * U * want[2][k].abs().max() * used)), k
    # buffers that are passed in keep what they held there; the stream may be updated in place, and so may its gradient
    xi, yi = x.clone(), torch.full_like(y, 5.0)
    a, b, st2 = ops.res_norm_fwd(xi, h, p["pre_w"], pre_b, x_out=xi, y=yi, **args)
    assert a is xi and torch.equal(xi[:used], x_out[:used]) and torch.equal(xi[used:], x[used:]) and (yi[used:] == 5.0).all()
    di, hi = dres.clone(), torch.full_like(dh, 5.0)
    ops.res_norm_bwd(dy, di, h, xi, st2, p["pre_w"], dx=di, dh=hi, **args)
    assert torch.equal(di[:used], dx[:used]) and torch.equal(di[used:], dres[used:]) and (hi[used:] == 5.0).all()
    assert torch.equal(hi[:used], dh[:used])


def test_offsets_that_name_more_rows_than_there_are_are_cut():
    x, h, pre_b, p, dy, dres = make(30, 512, torch.float32, "rms", False, False, None, 10)
    p["gate"] = torch.randn(3, 512, device=DEV)
    p["cu"] = torch.tensor([0, 10, 20, 30], dtype=torch.int32, device=DEV)
    args = {k: v for k, v in p.items() if k != "pre_w"}
    want = ops.res_norm_fwd(x, h, p["pre_w"], **args)
    grads = ops.res_norm_bwd(dy, dres, h, want[0], want[2], p["pre_w"], **args)
    args["cu"] = torch.tensor([0, 10, 20, 3000], dtype=torch.int32, device=DEV)
    got = ops.res_norm_fwd(x, h, p["pre_w"], **args)
    g2 = ops.res_norm_bwd(dy, dres, h, got[0], got[2], p["pre_w"], **args)
    assert all(torch.equal(a, b) for a, b in zip(want, got)) and torch.equal(grads[0], g2[0]) and torch.equal(grads[2]["gate"], g2[2]["gate"])


def test_no_rows():
    x, h, pre_b, p, dy, dres = make(0, 512, torch.float32, "ln", True, True, "one", 11)
    args = {k: v for k, v in p.items() if k != "pre_w"}
    x_out, y, st = ops.res_norm_fwd(x, h, p["pre_w"], pre_b, **args)
    dx, dh, g = ops.res_norm_bwd(dy, dres, h, x_out, st, p["pre_w"], **args)
    assert x_out.shape == dx.shape == (0, 512) and all((v == 0).all() for v in g.values())


def test_against_the_layer_norm_of_its_own():
    """Without post-norm, scale or gate: the residual add and neat_ln_fwd / neat_ln_bwd.  Same values up to both kernels' bounds."""
    x, h, pre_b, p, dy, dres = make(500, 768, torch.bfloat16, "ln", False, False, None, 12)
    x_out, y, st = ops.res_norm_fwd(x, h, p["pre_w"], pre_b, eps=EPS)
    assert torch.equal(x_out, x + h.float())
    y2, yf, mu, rs = ops.ln_fwd(x_out, p["pre_w"], pre_b, eps=EPS, out_f32=True)
    lim = 2 * (30 * U * (yf.abs() + pre_b.abs()) * 2 + 28 * U * x_out.abs().mean() * 3) + 2.0 ** -8 * yf.abs()
    assert ((y.float() - yf).abs() <= lim).all()
    dg, db = torch.zeros(768, device=DEV), torch.zeros(768, device=DEV)
    dxf, _ = ops.ln_bwd(dy, x_out, p["pre_w"], mu, rs, dres=dres, dgamma=dg, dbeta=db)
    dx, dh, g = ops.res_norm_bwd(dy, dres, h, x_out, st, p["pre_w"])
    assert (dx - dxf).abs().max() < 400 * U * float(dxf.abs().max())
    assert (g["pre_w"] - dg).abs().max() < 400 * U * 500 and (g["pre_b"] - db).abs().max() < 400 * U * 500
    assert torch.equal(dh, dx.to(torch.bfloat16))


@pytest.mark.parametrize("kind", ["ln", "rms"])
def test_gradients_against_differences(kind):
    """Central differences of the 64-bit function with step h: off by about h^2 of its third derivative (|.| < 50 here) and by
    1e-15 / h of its rounding; the kernel by 1e-5 of the largest gradient, far above its own bound."""
    rows, cols = 6, 12
    x, h, pre_b, p, dy, dres = make(rows, cols, torch.float32, kind, True, True, "even", 13)
    args = {k: v for k, v in p.items() if k != "pre_w"}
    x_out, y, st = ops.res_norm_fwd(x, h, p["pre_w"], pre_b, eps=EPS, **args)
    dx, dh, g = ops.res_norm_bwd(dy, dres, h, x_out, st, p["pre_w"], **args)
    of = group_rows(p, rows)
    base = dict(x=x.double(), h=h.double(), pre_w=p["pre_w"].double(), pre_b=pre_b.double(), post_w=p["post_w"].double(),
                post_b=p["post_b"].double(), scale=p["scale"].double(), gate=p["gate"].double())

    def value(v):
        n = unit(v["h"], kind)[0] * v["post_w"] + v["post_b"]
        xo = v["x"] + n * v["scale"] * v["gate"][of]
        return float((dres.double() * xo).sum() + (dy.double() * (unit(xo, kind)[0] * v["pre_w"] + v["pre_b"])).sum())
    got = dict(g, x=dx, h=dh)
    for name in got:
        for at in range(0, base[name].numel(), max(1, base[name].numel() // 5)):
            vals = []
            for step in (1e-5, -1e-5):
                v = dict(base)
                v[name] = base[name].clone()
                v[name].view(-1)[at] += step
                vals.append(value(v))
            num, mine = (vals[0] - vals[1]) / 2e-5, float(got[name].reshape(-1)[at])
            assert abs(num - mine) <= 1e-5 * max(1.0, float(got[name].abs().max())), (name, at, num, mine)


def test_repeats_streams_and_graphs():
    x, h, pre_b, p, dy, dres = make(333, 768, torch.bfloat16, "rms", True, True, "ragged", 14)
    args = {k: v for k, v in p.items() if k != "pre_w"}

    def both():
        x_out, y, st = ops.res_norm_fwd(x, h, p["pre_w"], pre_b, **args)
        dx, dh, g = ops.res_norm_bwd(dy, dres, h, x_out, st, p["pre_w"], **args)
        return [x_out, y, dx, dh] + [g[k] for k in sorted(g)]
    want = both()
    assert all(torch.equal(a, b) for a, b in zip(want, both()))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = both()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = both()
    for seed in (15, 16, 17):
        new = make(333, 768, torch.bfloat16, "rms", True, True, "ragged", seed)
        for dst, src in ((x, new[0]), (h, new[1]), (dy, new[4]), (dres, new[5]), (p["gate"], new[3]["gate"]), (p["cu"], new[3]["cu"])):
            dst.copy_(src)
        want = both()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, held))


def test_refusals():
    x, h, pre_b, p, dy, dres = make(8, 512, torch.float32, "ln", False, False, None, 18)
    w = p["pre_w"]
    for call, says in ((lambda: ops.res_norm_fwd(x, h[:, :256], w), "expected"), (lambda: ops.res_norm_fwd(x, h.half(), w), "expected"),
                       (lambda: ops.res_norm_fwd(x, h, w[:256]), "pre_w"), (lambda: ops.res_norm_fwd(x, h, w, kind="group"), "kind"),
                       (lambda: ops.res_norm_fwd(x, h, w, post_b=w), "post_b"),
                       (lambda: ops.res_norm_fwd(x, h, w, gate=torch.ones(3, 512, device=DEV)), "divide"),
                       (lambda: ops.res_norm_fwd(x, h, w, cu=torch.zeros(2, dtype=torch.int32, device=DEV)), "cu"),
                       (lambda: ops.res_norm_fwd(x.bfloat16(), h, w), "dtype"), (lambda: ops.res_norm_fwd(x, h.t().contiguous().t(), w), "contiguous"),
                       (lambda: ops.res_norm_fwd(x[:, :510].contiguous(), h[:, :510].contiguous(), w[:510].contiguous()), "cols=510"),
                       (lambda: ops.res_norm_fwd(x.view(-1)[1:3585].view(7, 512), h[:7], w), "aligned"),
                       (lambda: ops.res_norm_bwd(dy, dres[:4], h, x, torch.zeros(4, 8, device=DEV), w), "dres"),
                       (lambda: ops.res_norm_bwd(dy, dres, h, x, torch.zeros(2, 8, device=DEV), w), "stats")):
        with pytest.raises(RuntimeError, match=says):
            call()
