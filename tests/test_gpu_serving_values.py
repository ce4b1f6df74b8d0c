"""Attention over pages where values are not finite.

What is infinite or NaN by the definition (64 bits) is the same infinity or NaN in the result, and nothing else is.  The rest is held to the
tolerances of the ready-query form: 2^-8 |o| for the rounding of the output and 2^-13 of the largest |v|.
"""
import numpy as np
import pytest

from bunker_b200 import ops
from bunker_b200 import runtime as R
from tests.test_gpu_serving import Case, bf16, val

pytestmark = pytest.mark.gpu

INF, NINF, NAN = 0x7F80, 0xFF80, 0x7FC0


def as_defined(c):
    with np.errstate(invalid="ignore", over="ignore"):
        want, kp, vp = c.want()
    for _ in range(2):
        ops.paged_attn(c.args())
        assert R.cuSync() == 0, R.last_error()
        got = val(c.out.download(np.uint16, (c.T * c.B, c.Hq, c.HD)))
        assert np.array_equal(np.isnan(got), np.isnan(want)), (np.argwhere(np.isnan(got) != np.isnan(want))[:5], got[np.isnan(want)][:5])
        assert np.array_equal(got == np.inf, want == np.inf) and np.array_equal(got == -np.inf, want == -np.inf)
        fine = np.isfinite(want)
        vmax = np.abs(val(vp)[np.isfinite(val(vp))]).max()
        assert (np.abs(got[fine] - want[fine]) <= 2.0 ** -8 * np.abs(want[fine]) + 2.0 ** -13 * vmax).all()
    return want


# ---- scores that are not numbers ------------------------------------------------------------

@pytest.mark.parametrize("HD,rows", [(128, 16), (256, 64)])
def test_a_query_that_is_nan_gives_nan(bk, HD, rows):
    for prefix, own_rows, T, new in ((0, [1, 70, 33], 1, None), (200, [1, 0, 150], 1, None), (70, [20, 9, 40], 9, [9, 2, 5])):
        c = Case(101 + prefix, 3, T, prefix, own_rows, new=new, HD=HD, Hq=6, Hkv=2, rows=rows, fused=False)
        for e, h in ((0, 2), (1, 5), (3 * T - 1, 0)):
            c.q[e, h, HD // 2] = NAN
        assert np.isnan(as_defined(c)).any()


def test_a_query_that_is_nan_gives_nan_behind_the_norm(bk):
    c = Case(111, 2, 1, 64, [30, 5], HD=128, Hq=4, Hkv=1)
    c.q[1, 3, 7] = NAN
    ops.paged_attn(c.args())
    assert R.cuSync() == 0, R.last_error()
    got = val(c.out.download(np.uint16, (2, 4, 128)))
    odd = np.zeros(got.shape, bool)
    odd[1, 3] = True
    assert np.array_equal(np.isnan(got), odd) and np.isfinite(got[~odd]).all()


@pytest.mark.parametrize("HD", [128, 256])
def test_keys_that_are_all_nan_give_nan(bk, HD):
    # the only key of a sequence
    c = Case(121, 2, 1, 0, [1, 5], HD=HD, fused=False)
    c.k[0, 0, 3] = NAN
    assert np.isnan(as_defined(c)[0]).all()
    # the only own key behind a prefix: a piece of the work with nothing else in it
    c = Case(122, 3, 1, 128, [1, 2, 60], HD=HD, Hq=8, Hkv=2, fused=False)
    c.k[0, 1, HD - 1] = NAN
    assert np.isnan(as_defined(c)[0, 4:]).all()
    # all keys of a sequence's own part, more than a tile of them
    c = Case(123, 2, 1, 64, [100, 100], HD=HD, fused=False)
    j = np.arange(64, 164)
    c.kp[c.table[1, j // c.rows], :, j % c.rows] = NAN
    c.k[1] = NAN
    assert np.isnan(as_defined(c)[1]).all()


@pytest.mark.parametrize("HD", [128, 256])
def test_infinite_scores(bk, HD):
    """A key at minus infinity has no weight beside others, and is 0 / 0 alone; one at plus infinity is inf / inf."""
    for own_rows, at in (([1, 40], None), ([30, 40], 5), ([200, 3], 100)):
        c = Case(131 + own_rows[0], 2, 1, 0, own_rows, HD=HD, Hq=2, Hkv=1, fused=False)
        c.q[:] = bf16(np.full(c.q.shape, 0.25))
        if at is None:
            c.k[0, 0, 4] = NINF
        else:
            c.kp[c.table[0, at // c.rows], 0, at % c.rows, 4] = NINF
        assert np.isnan(as_defined(c)).any() == (at is None)
    c = Case(137, 2, 1, 0, [50, 10], HD=HD, Hq=2, Hkv=1, fused=False)
    c.q[:] = bf16(np.full(c.q.shape, 0.25))
    c.kp[c.table[1, 0], 0, 3, 9] = INF
    assert np.isnan(as_defined(c)[1]).all()
