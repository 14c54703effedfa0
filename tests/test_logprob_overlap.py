"""CPU: a gradient that overlaps the logits in another way than element by element is refused before anything is launched.  Addresses
are made up: every call here is refused.  What may lie between the logits' rows is checked with numbers of rows that share no byte."""
import random

import pytest

from neat_amd import lib

A = 1 << 20


def bwd(z, ld, dz, ldz, R=4, V=100, dtype=0):
    return lib.load().neat_token_logprobs_bwd(z, ld, dtype, 64, 64, 64, 64, 1.0, dz, ldz, R, V, None)


def both(z, ld, dz, ldz, R=4, V=100, dtype=0):
    return lib.load().neat_token_logprobs_fwd_bwd(z, ld, dtype, 64, 64, 64, 1.0, 64, 64, 64, dz, ldz, R, V, 64, None)


def meet(z, ld, dz, ldz, R, V, t):
    """The definition: some row of one shares a byte with some row of the other."""
    return any(z + i * ld * t < dz + j * ldz * t + V * t and dz + j * ldz * t < z + i * ld * t + V * t for i in range(R) for j in range(R))


@pytest.mark.parametrize("call", [bwd, both])
@pytest.mark.parametrize("dtype,t", [(0, 4), (1, 2)])
@pytest.mark.parametrize("ld,off,ldz", [(100, 1, 100), (100, -1, 100), (100, 100, 100), (100, -300, 100), (100, 399, 100),
                                        (250, 99, 250), (250, -99, 250), (250, 151, 250), (250, 250, 250), (250, 849, 250),
                                        (100, 0, 101), (250, 0, 100), (250, 100, 130), (101, 3, 100)])
def test_overlaps_are_refused(call, dtype, t, ld, off, ldz):
    assert meet(A, ld, A + off * t, ldz, 4, 100, t)
    assert call(A, ld, A + off * t, ldz, dtype=dtype) == -2
    assert "overlaps" in lib.last_error()


def test_overlaps_of_random_layouts_are_refused():
    r = random.Random(1)
    seen = 0
    for _ in range(4000):
        R, V = r.randint(1, 6), r.randint(1, 9)
        ld, ldz, off = V + r.randint(0, 12), V + r.randint(0, 12), r.randint(-70, 70)
        if r.random() < 0.5:
            ldz = ld
        if (off == 0 and (ld == ldz or R == 1)) or not meet(A, ld, A + 4 * off, ldz, R, V, 4):
            continue
        seen += 1
        assert bwd(A, ld, A + 4 * off, ldz, R, V) == -2, (R, V, ld, ldz, off)
    assert seen > 500
