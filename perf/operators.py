"""Cases for the operators of an adaptation step in the form that language-model towers have them: the norms around a block
fused with its gate and residual scale, log probabilities of given tokens with their entropy, alternatives and gradient, and
an AdamW step over many tensors with states in 32 or 8 bits.

``run`` computes a case in elementary torch operations, or through ``neat_amd`` where ``own`` is true; ``exact`` computes it in
64 bits.  Sizes are those of the framework's own towers (512 and 768 columns, 77 positions, 49 408 tokens, 25 014 captions) or
generic."""
import math
import random

import torch

own = False

DEV = "cuda"
DT = {"f32": torch.float32, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "bf16": 2}
EPS = 1e-5
LR, B1, B2, AEPS, WD = 2e-4, 0.9, 0.999, 1e-8, 1e-3          # the adaptation step's own learning rate and decay
BLOCK = 256                                                   # elements that share an 8-bit state's scale


def _norm_case(name, rows, cols, kind="ln", post=True, scale=True, groups=0, ragged=False, dtype="bf16", train=True):
    c = dict(op="norm", rows=rows, cols=cols, kind=kind, post=post, scale=scale, groups=groups, ragged=ragged, dtype=dtype,
             train=train)
    return dict(c, name=name) if name else c


def _lp_case(name, rows, vocab, mode, k=0, scale=1.0, dtype="bf16", pad=0, masked=False):
    c = dict(op="logprob", rows=rows, vocab=vocab, mode=mode, k=k, scale=scale, dtype=dtype, pad=pad, masked=masked)
    return dict(c, name=name) if name else c


def _adam_case(name, kind, width, count, bits, dtype="f32"):
    c = dict(op="adamw", kind=kind, width=width, count=count, bits=bits, dtype=dtype)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one new token between two blocks of a text tower while serving: nothing but latency
        _norm_case("norm_one_token", 1, 512, train=False),
        # 1 024 captions at the full 77 positions through one junction of the text tower, with its backward pass; each
        # caption has a gate of its own (a conditioned, adaLN-like block)
        _norm_case("norm_captions", 78848, 512, groups=1024),
        # the same step on packed captions of ragged length, RMS norms, no post-norm scale: what packed text batches run
        _norm_case("norm_packed_rms", 14851, 768, kind="rms", groups=1021, ragged=True),
        # a gallery of images through a wide vision tower: forward only, LayerScale, no gate
        _norm_case("norm_gallery_wide", 50000, 1280, post=False, train=False),
        # the next token's log probability and five alternatives for one sequence over the CLIP vocabulary
        _lp_case("logprob_one_row", 1, 49408, "score", k=5),
        # 2 000 image queries scored against all captions of the retrieval set: odd row length, fp32 cosines times exp(logit_scale)
        _lp_case("logprob_captions", 2000, 25014, "score", k=10, scale=100.0, dtype="f32"),
        # loss and gradient of a captioning step: 64 captions of 77 tokens over the CLIP vocabulary, known weights
        _lp_case("logprob_step", 4928, 49408, "step"),
        # zero-shot classes with impossible ones masked, rows cut out of a wider buffer, weights that depend on the result
        _lp_case("logprob_masked_grad", 3001, 5000, "grad", scale=100.0, dtype="f32", pad=7, masked=True),
        # the 48 LayerNorm tensors of the adapted text tower: launch latency
        _adam_case("adamw_norms", "ln", 512, 48, 32),
        # every weight of a 12-layer text tower, states in 32 bits
        _adam_case("adamw_tower_32", "tower", 512, 12, 32),
        # the same with states in 8 bits and weights in bf16
        _adam_case("adamw_tower_8", "tower", 512, 12, 8, dtype="bf16"),
        # a list of tensors of any size, views of one bucket that start at odd places
        _adam_case("adamw_odd_8", "odd", 40000, 90, 8),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "logprob", "adamw"])
    if op == "norm":
        cols = 4 * _log_int(rng, 16, 1024)
        rows = _log_int(rng, 1, min(80000, 30_000_000 // cols))
        groups = rng.choice([0, 0, 1, 2])
        ragged = groups == 2
        if groups:
            groups = _log_int(rng, 1, min(rows, 2000))
            if not ragged:
                rows = max(1, rows // groups) * groups
        return _norm_case(None, rows, cols, rng.choice(["ln", "rms"]), rng.random() < 0.7, rng.random() < 0.7, groups, ragged,
                          rng.choice(["bf16", "f32"]), rng.random() < 0.6)
    if op == "logprob":
        vocab = _log_int(rng, 33, 150000)
        rows = _log_int(rng, 1, min(20000, 120_000_000 // vocab))
        mode = rng.choice(["score", "grad", "step"])
        dtype = rng.choice(["bf16", "f32"])
        return _lp_case(None, rows, vocab, mode, rng.randint(1, 32) if mode == "score" else 0,
                        100.0 if dtype == "f32" and rng.random() < 0.5 else rng.choice([1.0, 1.25]), dtype,
                        rng.choice([0, 0, 1, 5]), rng.random() < 0.3)
    kind = rng.choice(["ln", "tower", "odd"])
    bits, dtype = rng.choice([32, 8]), rng.choice(["f32", "bf16"])
    if kind == "ln":
        return _adam_case(None, kind, _log_int(rng, 64, 4096), rng.randint(1, 200), bits, dtype)
    if kind == "tower":
        return _adam_case(None, kind, 64 * rng.randint(1, 8), rng.randint(1, 12), bits, dtype)
    return _adam_case(None, kind, _log_int(rng, 10, 200000), rng.randint(1, 150), bits, dtype)


# ---- inputs ----
def _lengths(case):
    """Row counts of a packed batch's sequences: they add up to the rows, and a few may be empty."""
    r = random.Random(case["rows"] * 131 + case["groups"])
    cuts = sorted(r.randint(0, case["rows"]) for _ in range(case["groups"] - 1))
    return [b - a for a, b in zip([0] + cuts, cuts + [case["rows"]])]


def _sizes(case):
    w, n = case["width"], case["count"]
    if case["kind"] == "ln":
        return [w] * n
    if case["kind"] == "tower":
        return [3 * w * w, 3 * w, w * w, w, w, w, 4 * w * w, 4 * w, 4 * w * w, w, w, w] * n
    r = random.Random(w * 1009 + n)
    return [int(round(math.exp(r.uniform(0, math.log(w))))) for _ in range(n)]


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEV)


def _norm_inputs(case, gen):
    rows, cols, g, t = case["rows"], case["cols"], case["groups"], DT[case["dtype"]]
    s = {"x": _randn(gen, rows, cols) * 1.5 + 0.2, "h": (_randn(gen, rows, cols) * 0.7 + 0.1).to(t)}
    s["pre_w"], s["pre_b"] = 1 + 0.2 * _randn(gen, cols), 0.1 * _randn(gen, cols)
    s["post_w"] = 1 + 0.2 * _randn(gen, cols) if case["post"] else None
    s["post_b"] = 0.1 * _randn(gen, cols) if case["post"] else None
    s["scale"] = 0.3 + 0.1 * _randn(gen, cols) if case["scale"] else None
    s["gate"] = torch.tanh(_randn(gen, g, cols)) if g else None
    s["cu"] = None
    if case["ragged"]:
        cu = [0]
        for n in _lengths(case):
            cu.append(cu[-1] + n)
        s["cu"] = torch.tensor(cu, dtype=torch.int32, device=DEV)
    if case["train"]:
        s["dy"], s["dres"] = (_randn(gen, rows, cols) * 0.05).to(t), _randn(gen, rows, cols) * 0.1
    return s


def _lp_inputs(case, gen):
    rows, vocab, t = case["rows"], case["vocab"], DT[case["dtype"]]
    wide = torch.empty(rows, vocab + case["pad"], dtype=t, device=DEV)
    z = wide[:, :vocab]
    if case["scale"] > 50:                                    # cosines of related and unrelated pairs
        z.copy_(_randn(gen, rows, vocab) * 0.03 + 0.2)
    else:
        z.copy_(_randn(gen, rows, vocab) * 2.5)
    s = {"z": z, "t": torch.randint(0, vocab, (rows,), generator=gen, device=DEV)}
    if case["masked"]:
        for lo in range(0, rows, 2048):
            part = z[lo:lo + 2048]
            part.masked_fill_(torch.rand(part.shape, generator=gen, device=DEV) < 0.4, -math.inf)
        s["t"][rows // 3] = -1                                # a position without a target
        if rows > 2:
            z[rows // 2].fill_(-math.inf)                     # a row whose mask leaves nothing
    if case["mode"] != "score":
        s["a"] = -torch.rand(rows, generator=gen, device=DEV) / rows
        s["b"] = torch.rand(rows, generator=gen, device=DEV) * (0.3 / rows)
    return s


def _adam_inputs(case, gen):
    t, sizes = DT[case["dtype"]], _sizes(case)
    n = sum(sizes)
    p = (_randn(gen, n) * 0.04).to(t)
    g = (_randn(gen, n) * torch.exp(_randn(gen, n)) * 1e-3).to(t)
    blocks = [-(-k // BLOCK) for k in sizes]
    s = {"p": p, "g": g, "step": 0, "nblk": sum(blocks), "pos": None}
    if any(k % BLOCK for k in sizes):                         # where each element stands among its tensor's blocks
        per = torch.tensor(sizes, device=DEV)
        first = torch.cumsum(torch.tensor([0] + blocks[:-1], device=DEV), 0) * BLOCK
        start = torch.cumsum(per, 0) - per
        s["pos"] = torch.arange(n, device=DEV) + torch.repeat_interleave(first - start, per)
    if own:
        from neat_amd.optim import MultiTensorAdamW
        params = [torch.nn.Parameter(v) for v in torch.split(p, sizes)]
        for w, v in zip(params, torch.split(g, sizes)):
            w.grad = v
        s["opt"] = MultiTensorAdamW(params, lr=LR, betas=(B1, B2), eps=AEPS, weight_decay=WD, state_bits=case["bits"])
    else:
        s["m"] = torch.zeros(s["nblk"], BLOCK, device=DEV)
        s["v"] = torch.zeros(s["nblk"], BLOCK, device=DEV)
        if case["bits"] == 8:
            s["m"], s["v"] = s["m"].to(torch.float8_e4m3fn), s["v"].to(torch.float8_e4m3fn)
            s["ms"], s["vs"] = torch.ones(s["nblk"], device=DEV), torch.ones(s["nblk"], device=DEV)
    return s


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    make = {"norm": _norm_inputs, "logprob": _lp_inputs, "adamw": _adam_inputs}[case["op"]]
    return dict(make(case, gen), case=case)


# ---- the framework's operators ----
def _own_norm(s, case):
    from neat_amd import ops
    par = dict(post_w=s["post_w"], post_b=s["post_b"], scale=s["scale"], gate=s["gate"], cu=s["cu"], kind=case["kind"])
    x_out, y, stats = ops.res_norm_fwd(s["x"], s["h"], s["pre_w"], s["pre_b"], eps=EPS, save=case["train"], **par)
    if not case["train"]:
        return x_out, y
    dx, dh, grads = ops.res_norm_bwd(s["dy"], s["dres"], s["h"], x_out, stats, s["pre_w"], **par)
    return x_out, y, dx, dh, grads


def _own_lp(s, case):
    from neat_amd import ops
    if case["mode"] == "score":
        logp, ent, _, top, idx = ops.token_logprobs(s["z"], s["t"], scale=case["scale"], k=case["k"])
        return logp, ent, top, idx
    if case["mode"] == "step":
        logp, ent, dz = ops.token_logprobs_fwd_bwd(s["z"], s["t"], s["a"], s["b"], scale=case["scale"])
        return logp, ent, dz
    logp, ent, stats, _, _ = ops.token_logprobs(s["z"], s["t"], scale=case["scale"])
    return logp, ent, ops.token_logprobs_bwd(s["z"], s["t"], stats, s["a"], s["b"], scale=case["scale"])


def _own_adamw(s, case):
    opt = s["opt"]
    opt.step()
    if case["bits"] == 32:
        return s["p"], opt.exp_avg, opt.exp_avg_sq
    # what a block holds are e4m3 numbers and the power of two that they are multiplied with
    return s["p"], opt.exp_avg, opt.exp_avg_scale, opt.exp_avg_root, opt.exp_avg_root_scale


# ---- the plain forms ----
def _unit(u, kind):
    """(u normalised, 1 / its deviation) over the last axis."""
    c = u - u.mean(-1, keepdim=True) if kind == "ln" else u
    r = torch.rsqrt((c * c).mean(-1, keepdim=True) + EPS)
    return c * r, r


def _unit_bwd(z, uh, r, kind):
    d = z - uh * (z * uh).mean(-1, keepdim=True)
    return r * (d - z.mean(-1, keepdim=True)) if kind == "ln" else r * d


def _group_of_row(s, case):
    if s["cu"] is None:
        return torch.arange(case["rows"], device=DEV) // (case["rows"] // case["groups"])
    n = (s["cu"][1:] - s["cu"][:-1]).long()
    return torch.repeat_interleave(torch.arange(case["groups"], device=DEV), n, output_size=case["rows"])


def _norm(s, case):
    kind, t, h = case["kind"], DT[case["dtype"]], s["h"].float()
    hh, hr = _unit(h, kind) if case["post"] else (h, None)
    n = hh * s["post_w"] + s["post_b"] if case["post"] else h
    f = s["scale"]
    gid = _group_of_row(s, case) if case["groups"] else None
    if gid is not None:
        g = s["gate"][gid]
        f = g if f is None else g * f
    x = s["x"] + (n if f is None else n * f)
    xh, xr = _unit(x, kind)
    y = (xh * s["pre_w"] + s["pre_b"]).to(t)
    if not case["train"]:
        return x, y
    dy = s["dy"].float()
    e = s["dres"] + _unit_bwd(dy * s["pre_w"], xh, xr, kind)
    grads = {"pre_w": (dy * xh).sum(0), "pre_b": dy.sum(0)}
    a = e * n
    if gid is not None:
        per = torch.zeros_like(s["gate"]).index_add_(0, gid, a)
        grads["gate"] = per if s["scale"] is None else per * s["scale"]
        if case["scale"]:
            grads["scale"] = (per * s["gate"]).sum(0)
    elif case["scale"]:
        grads["scale"] = a.sum(0)
    dn = e if f is None else e * f
    dh = dn
    if case["post"]:
        grads["post_w"], grads["post_b"] = (dn * hh).sum(0), dn.sum(0)
        dh = _unit_bwd(dn * s["post_w"], hh, hr, kind)
    return x, y, e, dh.to(t), grads


def _lp(s, case):
    z, t, f = s["z"].float(), s["t"], case["scale"]
    m = z.amax(-1, keepdim=True)
    m0 = torch.where(m == -math.inf, torch.zeros_like(m), m)
    d = (z - m0) * f
    e = torch.exp(d)
    tot = e.sum(-1, keepdim=True)
    logs = torch.log(tot)
    lp = d - logs
    p = torch.where(e > 0, e / tot, torch.zeros_like(e))
    none = m == -math.inf                                     # nothing left of the row
    ent = torch.where(none, torch.zeros_like(m), logs - torch.where(e > 0, p * d, torch.zeros_like(e)).sum(-1, keepdim=True))
    has = t >= 0
    at = lp.gather(1, t.clamp(min=0)[:, None])
    at = torch.where(none, torch.full_like(at, -math.inf), at)
    logp = torch.where(has[:, None], at, torch.zeros_like(at))[:, 0]
    if case["mode"] == "score":
        val, idx = torch.sort(z, dim=-1, descending=True, stable=True)
        val, idx = val[:, :case["k"]], idx[:, :case["k"]]
        top = torch.where(none, torch.full_like(val, -math.inf), (val - m0) * f - logs)
        return logp, ent[:, 0], top, idx.to(torch.int32)
    a = torch.where(has, s["a"], torch.zeros_like(s["a"]))[:, None]
    a = torch.where(none, torch.zeros_like(a), a)
    dz = -p * (a + s["b"][:, None] * torch.where(e > 0, lp + ent, torch.zeros_like(lp)))
    dz.scatter_add_(1, t.clamp(min=0)[:, None], a)
    return logp, ent[:, 0], (dz * f).to(s["z"].dtype)


def _quantise(x, lowest):
    """(e4m3 numbers, powers of two [blocks]): each block's largest finite value lies in (224, 448] times its power of two;
    with ``lowest``, what is above zero stays above it."""
    a = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x)).amax(-1)
    f, ex = torch.frexp(a)
    ex = torch.where(a > 0, ex - 9 + (f > 0.875).to(ex.dtype), torch.full_like(ex, -126)).clamp(min=-126)
    q = x * torch.ldexp(torch.ones_like(a), -ex)[:, None]
    if lowest:
        q = torch.where(x > 0, q.clamp(min=2.0 ** -9), q)
    return q.to(torch.float8_e4m3fn), torch.ldexp(torch.ones_like(a), ex)


def _blocks(flat, s):
    out = flat.float()
    if s["pos"] is not None:
        out = torch.zeros(s["nblk"] * BLOCK, device=DEV).index_copy_(0, s["pos"], out)
    return out.view(-1, BLOCK)


def _adamw(s, case):
    s["step"] += 1
    step, small = s["step"], case["bits"] == 8
    p, g, m, v = _blocks(s["p"], s), _blocks(s["g"], s), s["m"], s["v"]
    if small:
        m = m.float() * s["ms"][:, None]
        r = v.float() * s["vs"][:, None]
        v = r * r
    m = m + (g - m) * (1.0 - B1)
    v = v * B2 + g * g * (1.0 - B2)
    r = torch.sqrt(v)
    p = p * (1.0 - LR * WD) - (m / (r / math.sqrt(1.0 - B2 ** step) + AEPS)) * (LR / (1.0 - B1 ** step))
    s["p"].copy_(p.view(-1) if s["pos"] is None else p.view(-1)[s["pos"]])
    if not small:
        s["m"], s["v"] = m, v
        return s["p"], m, v
    s["m"], s["ms"] = _quantise(m, False)
    s["v"], s["vs"] = _quantise(r, True)
    return s["p"], s["m"], s["ms"], s["v"], s["vs"]


def run(s):
    case = s["case"]
    if own:
        return {"norm": _own_norm, "logprob": _own_lp, "adamw": _own_adamw}[case["op"]](s, case)
    return {"norm": _norm, "logprob": _lp, "adamw": _adamw}[case["op"]](s, case)


# ---- what a pass cannot do without ----
def work(case):
    t = SIZE[case["dtype"]]
    if case["op"] == "norm":
        n, g = case["rows"] * case["cols"], case["groups"] * case["cols"]
        once = n * (8 + 2 * t) + 4 * g + 20 * case["cols"]
        if case["train"]:                                     # dy, dres, h and x_out come in again, dx and dh go out
            once += n * (12 + 3 * t) + 4 * g + 20 * case["cols"]
        return {"bytes": once, "flops": n * (60 if case["train"] else 20)}
    if case["op"] == "logprob":
        n = case["rows"] * case["vocab"]
        if case["mode"] == "score":
            return {"bytes": n * t + case["rows"] * (16 + 8 * case["k"]), "flops": 6 * n}
        return {"bytes": 2 * n * t + 24 * case["rows"], "flops": 12 * n}
    n = sum(_sizes(case))
    held = 16 if case["bits"] == 32 else 4 + 16 / BLOCK
    return {"bytes": n * (3 * t + held), "flops": 15 * n}


# ---- the definitions in 64 bits ----
def _exact_norm(s, case):
    D = torch.float64
    ln, C = case["kind"] == "ln", case["cols"]

    def norm(u, w, b):
        mean = u.sum(1, keepdim=True) / C if ln else torch.zeros(len(u), 1, dtype=D, device=DEV)
        dev = torch.sqrt(((u - mean) ** 2).sum(1, keepdim=True) / C + EPS)
        hat = (u - mean) / dev
        return hat, dev, hat * w.to(D) + b.to(D)

    def norm_grad(dz, hat, dev):
        out = dz - hat * ((dz * hat).sum(1, keepdim=True) / C)
        if ln:
            out = out - dz.sum(1, keepdim=True) / C
        return out / dev

    h = s["h"].to(D)
    hat_h, dev_h, n = norm(h, s["post_w"], s["post_b"]) if case["post"] else (None, None, h)
    scale = s["scale"].to(D) if case["scale"] else torch.ones(C, dtype=D, device=DEV)
    if case["groups"]:
        if case["ragged"]:
            of = [i for i, k in enumerate(_lengths(case)) for _ in range(k)]
        else:
            of = [r // (case["rows"] // case["groups"]) for r in range(case["rows"])]
        of = torch.tensor(of, device=DEV)
        gate = s["gate"].to(D)[of]
    else:
        of, gate = None, torch.ones(1, C, dtype=D, device=DEV)
    x = s["x"].to(D) + n * scale * gate
    hat, dev, y = norm(x, s["pre_w"], s["pre_b"])
    if not case["train"]:
        return x, y
    dy = s["dy"].to(D)
    e = s["dres"].to(D) + norm_grad(dy * s["pre_w"].to(D), hat, dev)
    grads = {"pre_w": (dy * hat).sum(0), "pre_b": dy.sum(0)}
    if of is not None:
        grads["gate"] = torch.zeros(case["groups"], C, dtype=D, device=DEV).index_add_(0, of, e * n * scale)
    if case["scale"]:
        grads["scale"] = (e * n * gate).sum(0)
    dh = dn = e * scale * gate
    if case["post"]:
        grads["post_w"], grads["post_b"] = (dn * hat_h).sum(0), dn.sum(0)
        dh = norm_grad(dn * s["post_w"].to(D), hat_h, dev_h)
    return x, y, e, dh, grads


def _exact_lp(s, case):
    z, t = s["z"].to(torch.float64) * case["scale"], s["t"]
    lse = torch.logsumexp(z, 1)
    empty = lse == -math.inf
    lp = z - torch.where(empty, torch.zeros_like(lse), lse)[:, None]
    p = torch.exp(lp)
    plp = torch.nan_to_num(p * lp, nan=0.0, posinf=0.0, neginf=0.0)     # a masked place adds nothing
    ent = -plp.sum(1)
    logp = torch.where(t < 0, torch.zeros_like(lse), lp[torch.arange(len(t), device=DEV), t.clamp(min=0)])
    if case["mode"] == "score":
        order = torch.argsort(s["z"].to(torch.float64), dim=1, descending=True, stable=True)[:, :case["k"]]
        return logp, ent, lp.gather(1, order), order.to(torch.int32)
    a = torch.where((t < 0) | empty, torch.zeros_like(lse), s["a"].to(torch.float64))
    dz = -a[:, None] * p - s["b"].to(torch.float64)[:, None] * (plp + p * ent[:, None])
    dz[torch.arange(len(t), device=DEV), t.clamp(min=0)] += a
    return logp, ent, dz * case["scale"]


def _exact_adamw(s, case):
    p, g = s["p"].to(torch.float64), s["g"].to(torch.float64)
    m, v = (1.0 - B1) * g, (1.0 - B2) * g ** 2                # the first step: both moments start at zero
    m_hat, v_hat = m / (1.0 - B1), v / (1.0 - B2)
    new = p - LR * WD * p - LR * m_hat / (torch.sqrt(v_hat) + AEPS)

    def held(u):
        out = torch.zeros(s["nblk"] * BLOCK, dtype=torch.float64, device=DEV)
        out[torch.arange(len(u), device=DEV) if s["pos"] is None else s["pos"]] = u
        return out.view(-1, BLOCK)

    def coded(u, lowest):
        u = held(u)
        top = u.abs().amax(1)
        e = torch.where(top > 0, torch.ceil(torch.log2(top.clamp(min=1e-300) / 448.0)), torch.full_like(top, -126.0)).clamp(min=-126.0)
        unit = torch.exp2(e)
        q = u / unit[:, None]
        step = torch.exp2(torch.floor(torch.log2(q.abs().clamp(min=2.0 ** -6))) - 3.0)   # e4m3: three bits behind the leading one
        r = torch.round(q / step) * step
        if lowest:
            r = torch.where((u > 0) & (r == 0), torch.full_like(r, 2.0 ** -9), r)
        return r, unit

    if case["bits"] == 32:
        return new, held(m), held(v)
    return (new, *coded(m, False), *coded(torch.sqrt(v), True))


def exact(case, seed):
    global own
    was, own = own, False                                     # the inputs alone, without the framework's handle
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return {"norm": _exact_norm, "logprob": _exact_lp, "adamw": _exact_adamw}[case["op"]](s, case)
