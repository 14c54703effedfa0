"""CPU: a gate whose gradient would take more than one launch can hold is refused before anything is launched (addresses are made up)."""
import pytest

from neat_amd import lib

G = 1 << 40


@pytest.mark.parametrize("groups,cols", [(1 << 26, 4096), (1 << 20, 4096), (1 << 30, 4), ((1 << 26) + 1, 64)])
def test_a_gate_too_large_for_one_launch_is_refused(groups, cols):
    rc = lib.load().neat_res_norm_bwd(G, 2 * G, 3 * G, 4 * G, 5 * G, 0, 0, 6 * G, None, None, None, 7 * G, groups, 9 * G, 10 * G,
                                      11 * G, None, None, None, None, None, 12 * G, 14 * G, 0, 4, cols, None)
    assert rc == -1 and "too large" in lib.last_error()


def test_more_groups_than_indices_hold_are_refused():
    L = lib.load()
    for groups in ((1 << 30) + 1, (1 << 31) - 1):
        assert L.neat_res_norm_fwd(G, 2 * G, 0, 0, 3 * G, None, None, None, None, 4 * G, groups, 6 * G, 7 * G, 8 * G, None, 0, 4, 4, 1e-5,
                                   None) == -1
        assert "too large" in lib.last_error()
