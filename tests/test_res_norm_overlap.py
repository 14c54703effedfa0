"""CPU: outputs of the fused norms that overlap an input, or each other, in a way that spoils results are refused before anything is
launched.  Addresses are made up (64 KiB apart unless a test moves one), every call here is refused."""
import pytest

from neat_amd import lib

ROWS, COLS, GROUPS = 8, 64, 2
NAMES_F = ["x", "h", "pre_w", "pre_b", "post_w", "post_b", "scale", "gate", "cu", "x_out", "y", "stats"]
NAMES_B = ["dy", "dres", "h", "x_out", "stats", "pre_w", "post_w", "post_b", "scale", "gate", "cu", "dx", "dh", "dpre_w", "dpre_b",
           "dpost_w", "dpost_b", "dscale", "dgate", "ws"]


def fwd(dtype=0, **move):
    p = {n: (k + 1) << 16 for k, n in enumerate(NAMES_F)}
    p.update({n: p[of] + off for n, (of, off) in move.items()})
    return lib.load().neat_res_norm_fwd(p["x"], p["h"], dtype, 0, p["pre_w"], p["pre_b"], p["post_w"], p["post_b"], p["scale"],
                                        p["gate"], GROUPS, p["cu"], p["x_out"], p["y"], p["stats"], 0, ROWS, COLS, 1e-5, None)


def bwd(dtype=0, **move):
    p = {n: (k + 1) << 16 for k, n in enumerate(NAMES_B)}
    p["ws"] = 1 << 30
    p.update({n: p[of] + off for n, (of, off) in move.items()})
    return lib.load().neat_res_norm_bwd(p["dy"], p["dres"], p["h"], p["x_out"], p["stats"], dtype, 0, p["pre_w"], p["post_w"],
                                        p["post_b"], p["scale"], p["gate"], GROUPS, p["cu"], p["dx"], p["dh"], p["dpre_w"],
                                        p["dpre_b"], p["dpost_w"], p["dpost_b"], p["dscale"], p["dgate"], p["ws"], 0, ROWS, COLS,
                                        None)


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("move", [
    dict(x_out=("x", 256)), dict(x_out=("x", -256)), dict(x_out=("h", 16)), dict(y=("h", 16)), dict(y=("x_out", 0)), dict(y=("x_out", 64)),
    dict(x_out=("pre_w", 0)), dict(y=("gate", 256)), dict(x_out=("scale", -1024)), dict(y=("cu", 0)), dict(stats=("x", 0)),
    dict(stats=("y", 0)), dict(stats=("post_b", 128))])
def test_forward_overlaps_are_refused(move, dtype):
    assert fwd(dtype, **move) == -2
    assert "overlap" in lib.last_error()


def test_an_output_over_an_input_of_another_element_size_is_refused():
    for call, move in ((fwd, dict(x_out=("h", 0))), (fwd, dict(y=("x", 0))), (bwd, dict(dx=("dy", 0))), (bwd, dict(dx=("h", 0))),
                       (bwd, dict(dh=("dres", 0))), (bwd, dict(dh=("x_out", 0)))):
        assert call(1, **move) == -2, move
        assert "overlap" in lib.last_error()


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("move", [
    dict(dx=("dres", 256)), dict(dx=("x_out", -256)), dict(dh=("h", 16)), dict(dh=("dy", -16)), dict(dh=("dx", 0)), dict(dx=("gate", 0)),
    dict(dh=("stats", 16)), dict(ws=("h", 0)), dict(ws=("dx", 0)), dict(ws=("pre_w", 0)), dict(dpre_w=("dpre_b", 128)),
    dict(dscale=("scale", 0)), dict(dgate=("scale", 0)), dict(dgate=("cu", -16)), dict(dpost_w=("dx", 512)), dict(dgate=("ws", 256)),
    dict(dpost_b=("dgate", 256))])
def test_backward_overlaps_are_refused(move, dtype):
    assert bwd(dtype, **move) == -2
    assert "overlap" in lib.last_error()
