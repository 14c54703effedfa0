"""CPU: calls that the operators refuse are refused before anything is launched (no GPU is needed to see it)."""
import ctypes

import pytest
import torch

from neat_amd import lib, ops
from neat_amd.optim import MultiTensorAdamW


def _arr(kind, *v):
    return (kind * len(v))(*v)


def _adamw(count=1, p=64, g=64, n=10, block=0, step=1, dtype=0, m=64, v=64, ms=64, vs=64, bits=32):
    return lib.load().neat_adamw_multi(count, _arr(ctypes.c_void_p, p), _arr(ctypes.c_void_p, g), _arr(ctypes.c_int64, n),
                                       _arr(ctypes.c_int64, block), _arr(ctypes.c_int32, step), dtype, m, v, ms, vs, bits, 1e-3,
                                       0.9, 0.999, 1e-8, 0.0, None)


@pytest.mark.parametrize("bad, rc, says", [
    (dict(count=-1), -1, "count"), (dict(p=None), -2, "null"), (dict(g=None), -2, "null"), (dict(m=None), -2, "null"),
    (dict(n=-1), -1, "n=-1"), (dict(n=1 << 40), -1, "too large"), (dict(block=-1), -1, "state_block"),
    (dict(block=1 << 32), -1, "too large"), (dict(step=0), -1, "step=0"), (dict(dtype=7), -2, "dtype"),
    (dict(bits=4), -2, "state_bits"), (dict(bits=8, ms=None), -2, "scales"), (dict(m=68), -2, "aligned"),
    (dict(p=66), -2, "aligned"), (dict(p=65, dtype=1), -2, "aligned")])
def test_adamw_multi_checks_before_launching(bad, rc, says):
    assert _adamw(**bad) == rc
    assert says in lib.last_error()


def test_adamw_multi_without_tensors_is_nothing():
    assert _adamw(count=0) == 0
    assert _adamw(n=0, p=None, g=None) == 0


def test_adamw_multi_wrapper_refuses():
    p, m = torch.zeros(5), torch.zeros(1, 256)
    with pytest.raises(RuntimeError, match="GPU"):
        ops.adamw_multi([p], [p], [0], [1], m, m.clone())
    with pytest.raises(RuntimeError, match="one gradient"):
        ops.adamw_multi([p], [], [0], [1], m, m.clone())
    with pytest.raises(RuntimeError, match="float32 or bfloat16"):
        ops.adamw_multi([p.double()], [p.double()], [0], [1], m, m.clone())
    with pytest.raises(RuntimeError, match="all be"):
        ops.adamw_multi([p], [p.bfloat16()], [0], [1], m, m.clone())
    with pytest.raises(RuntimeError, match="contiguous"):
        ops.adamw_multi([torch.zeros(4, 3).t()], [torch.zeros(3, 4)], [0], [1], m, m.clone())
    with pytest.raises(RuntimeError, match="size"):
        ops.adamw_multi([p], [torch.zeros(6)], [0], [1], m, m.clone())
    with pytest.raises(RuntimeError, match="outside"):
        ops.adamw_multi([p], [p], [1], [1], m, m.clone())
    with pytest.raises(RuntimeError, match="m and v"):
        ops.adamw_multi([p], [p], [0], [1], m, torch.zeros(1, 128))
    with pytest.raises(RuntimeError, match="m_scale"):
        ops.adamw_multi([p], [p], [0], [1], m.to(torch.uint8), m.to(torch.uint8))
    with pytest.raises(RuntimeError, match="GPU"):
        MultiTensorAdamW([torch.nn.Parameter(p)])
    with pytest.raises(ValueError):
        MultiTensorAdamW([torch.nn.Parameter(p)], betas=(0.9, 1.0))
    with pytest.raises(ValueError):
        MultiTensorAdamW([torch.nn.Parameter(p)], lr=-1.0)


def _lp(z=64, ld=100, dtype=0, target=64, scale=1.0, k=0, logp=64, top=64, idx=64, R=4, V=100, ws=64):
    return lib.load().neat_token_logprobs(z, ld, dtype, target, scale, k, logp, 64, 64, top, idx, R, V, ws, None)


@pytest.mark.parametrize("bad, rc, says", [
    (dict(z=None), -2, "null"), (dict(target=None), -2, "targets"), (dict(dtype=2), -2, "dtype"), (dict(ld=99), -1, "pitch"),
    (dict(V=0), -1, "V=0"), (dict(R=-1), -1, "R=-1"), (dict(k=33), -1, "k=33"), (dict(k=5, V=4), -1, "k=5"),
    (dict(k=-1), -1, "k=-1"), (dict(k=2, top=None), -2, "alternatives"), (dict(z=66), -2, "aligned"),
    (dict(scale=0.0), -2, "scale"), (dict(scale=-1.0), -2, "scale"), (dict(scale=float("nan")), -2, "scale"),
    (dict(scale=float("inf")), -2, "scale"), (dict(V=3_000_000, ld=3_000_000), -1, "above"),
    (dict(V=100_000, ld=100_000, ws=None), -2, "workspace"), (dict(V=4_200_000, ld=4_200_000, dtype=1, k=32), -1, "above")])
def test_token_logprobs_checks_before_launching(bad, rc, says):
    assert _lp(**bad) == rc
    assert says in lib.last_error()


def test_token_logprobs_gradient_checks_before_launching():
    L = lib.load()
    assert L.neat_token_logprobs_bwd(64, 9, 0, 64, None, 64, 64, 1.0, 64, 9, 2, 9, None) == -2
    assert L.neat_token_logprobs_bwd(64, 9, 0, None, 64, 64, 64, 1.0, 64, 9, 2, 9, None) == -2
    assert L.neat_token_logprobs_bwd(64, 9, 0, 64, 64, 64, 64, 1.0, 64, 8, 2, 9, None) == -1
    assert L.neat_token_logprobs_bwd(64, 9, 0, 64, 64, 64, 64, 1.0, 65, 9, 2, 9, None) == -2
    assert L.neat_token_logprobs_fwd_bwd(64, 9, 0, None, 64, 64, 1.0, 64, 64, 64, 64, 9, 2, 9, None, None) == -2
    assert L.neat_token_logprobs_fwd_bwd(64, 90000, 0, 64, 64, 64, 1.0, 64, 64, None, 64, 90000, 2, 90000, 64, None) == -2
    assert L.neat_token_logprobs_ws_bytes(0, 4, 32768, 0) == 0
    assert L.neat_token_logprobs_ws_bytes(0, 4, 32769, 0) >= 4 * 2 * 16
    assert _lp(R=0) == 0


def test_token_logprobs_wrapper_refuses():
    z = torch.zeros(3, 7)
    for call in (lambda: ops.token_logprobs(z), lambda: ops.token_logprobs(z.half()), lambda: ops.token_logprobs(z[0]),
                 lambda: ops.token_logprobs_bwd(z, None, torch.zeros(3, 3)), lambda: ops.token_logprobs_fwd_bwd(z, None)):
        with pytest.raises(RuntimeError):
            call()


def _rn(x=64, h=64, dtype=0, kind=0, pre_w=64, pre_b=64, post_w=64, post_b=64, scale=64, gate=64, groups=2, cu=None, x_out=64, y=64,
        rows=4, cols=64):
    return lib.load().neat_res_norm_fwd(x, h, dtype, kind, pre_w, pre_b, post_w, post_b, scale, gate, groups, cu, x_out, y, 64, 0, rows,
                                        cols, 1e-5, None)


@pytest.mark.parametrize("bad, rc, says", [
    (dict(x=None), -2, "null"), (dict(h=None), -2, "null"), (dict(pre_w=None), -2, "null"), (dict(y=None), -2, "null"),
    (dict(dtype=5), -2, "dtype"), (dict(kind=2), -2, "kind"), (dict(cols=66), -1, "cols"), (dict(cols=4100), -1, "cols"),
    (dict(rows=-1), -1, "rows"), (dict(rows=5), -1, "divide"), (dict(groups=0), -2, "groups"), (dict(gate=None), -2, "groups"),
    (dict(gate=None, groups=0, cu=64), -2, "cu"), (dict(post_w=None), -2, "post_b"), (dict(x=72), -2, "aligned"),
    (dict(h=72), -2, "aligned"), (dict(h=68, dtype=1), -2, "aligned"), (dict(scale=68), -2, "aligned")])
def test_res_norm_checks_before_launching(bad, rc, says):
    assert _rn(**bad) == rc
    assert says in lib.last_error()


def test_res_norm_backward_checks_before_launching():
    L = lib.load()

    def call(**k):
        v = dict(dy=64, h=64, x_out=64, stats=64, post_w=64, scale=64, gate=64, groups=2, dpost_w=64, dscale=64, dgate=64, ws=64)
        v.update(k)
        return L.neat_res_norm_bwd(v["dy"], 64, v["h"], v["x_out"], v["stats"], 0, 0, 64, v["post_w"], None, v["scale"], v["gate"],
                                   v["groups"], None, 64, 64, 64, 64, v["dpost_w"], None, v["dscale"], v["dgate"], v["ws"], 0, 4, 64,
                                   None)
    for bad in (dict(dy=None), dict(stats=None), dict(ws=None), dict(post_w=None), dict(scale=None), dict(gate=None, groups=0),
                dict(ws=72)):
        assert call(**bad) == -2, bad
    assert L.neat_res_norm_ws_floats(0, 4, 64, 2) > 5 * 64
    assert _rn(rows=0) == 0
