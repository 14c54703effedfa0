"""GPU: outputs of the fused norms that lie exactly over an input of their element size give what buffers of their own give; other
overlaps are refused and leave everything alone."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from neat_amd import ops  # noqa: E402

DEV = "cuda"


def inputs(rows, cols, dtype, ragged):
    gen = torch.Generator(device=DEV).manual_seed(rows + cols)
    r = lambda *s: torch.randn(*s, generator=gen, device=DEV)  # noqa: E731
    cu = torch.tensor([0, rows // 3, rows // 3, rows - 1], dtype=torch.int32, device=DEV) if ragged else None
    par = dict(post_w=1 + 0.1 * r(cols), post_b=0.1 * r(cols), scale=r(cols), gate=r(3 if ragged else 1, cols), cu=cu)
    return r(rows, cols), r(rows, cols).to(dtype), 1 + 0.1 * r(cols), par, r(rows, cols).to(dtype), r(rows, cols)


@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,cols", [(5, 64), (2000, 512), (333, 1664), (50, 4096)])
def test_exactly_over_an_input(rows, cols, dtype, ragged):
    x, h, w, par, dy, dres = inputs(rows, cols, dtype, ragged)
    used = rows - 1 if ragged else rows                      # rows behind the last sequence stay as they are in given buffers
    want_x, want_y, stats = ops.res_norm_fwd(x, h, w, **par)
    over = [("x", None), (None, "h")] + ([("h", None), (None, "x"), ("x", "h"), ("h", "x")] if dtype == torch.float32 else [("x", "h")])
    for over_x, over_y in over:
        t = dict(x=x.clone(), h=h.clone())
        got_x, got_y, st = ops.res_norm_fwd(t["x"], t["h"], w, x_out=t.get(over_x), y=t.get(over_y), **par)
        assert torch.equal(got_x[:used], want_x[:used]) and torch.equal(got_y[:used], want_y[:used])
        assert torch.equal(st[:, :used], stats[:, :used])
    want_dx, want_dh, want = ops.res_norm_bwd(dy, dres, h, want_x, stats, w, **par)
    over = [("dres", None), ("xo", None), (None, "h"), (None, "dy"), ("dres", "h"), ("xo", "dy")]
    if dtype == torch.float32:
        over += [("dy", "dres"), ("h", "xo")]
    for over_x, over_h in over:
        t = dict(dy=dy.clone(), dres=dres.clone(), h=h.clone(), xo=want_x.clone())
        dx, dh, g = ops.res_norm_bwd(t["dy"], t["dres"], t["h"], t["xo"], stats, w, dx=t.get(over_x), dh=t.get(over_h), **par)
        assert torch.equal(dx[:used], want_dx[:used]) and torch.equal(dh[:used], want_dh[:used])
        assert all(torch.equal(g[n], want[n]) for n in want)


def test_other_overlaps_are_refused():
    rows, cols = 6, 64
    x, h, w, par, dy, dres = inputs(rows, cols, torch.float32, False)
    flat = torch.randn(rows * cols + 4 * cols, device=DEV)
    one, two, was = flat[:rows * cols].view(rows, cols), flat[cols:cols + rows * cols].view(rows, cols), flat.clone()
    x_out, y, stats = ops.res_norm_fwd(x, h, w, **par)
    for call in (lambda: ops.res_norm_fwd(one, h, w, x_out=two, **par), lambda: ops.res_norm_fwd(x, one, w, y=two, **par),
                 lambda: ops.res_norm_fwd(x, h, w, x_out=one, y=one, **par), lambda: ops.res_norm_fwd(x, h, w, x_out=one, y=two, **par),
                 lambda: ops.res_norm_fwd(x, h, flat[cols:2 * cols], x_out=one, **par),
                 lambda: ops.res_norm_bwd(dy, one, h, x_out, stats, w, dx=two, **par),
                 lambda: ops.res_norm_bwd(one, dres, h, x_out, stats, w, dh=two, **par),
                 lambda: ops.res_norm_bwd(dy, dres, h, x_out, stats, w, dx=one, dh=one, **par)):
        with pytest.raises(RuntimeError, match="overlap"):
            call()
    assert torch.equal(flat, was)
