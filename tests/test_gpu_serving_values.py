"""Attention over pages and adapters where values are not finite, and where many row tiles share a long prefix.

What is infinite or NaN by the definition (64 bits) is the same infinity or NaN in the result, and nothing else is.  The rest is held to the
tolerances of the ready-query form: 2^-8 |o| for the rounding of the output and 2^-13 of the largest |v|.  Two results from the same
bits of q, k and v by two plans are each within that of the exact one: 2^-7 |o| + 2^-12 of the largest |v| of one another.
"""
import numpy as np
import pytest

from bunker_b200 import ops
from bunker_b200 import runtime as R
from tests.test_gpu_serving import Case, bf16, lora_case, val

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


# ---- values that are not finite, seen by every row of a tile ---------------------------------------

def put(c, b, key, dim, what):
    c.vp[c.table[b, key // c.rows], :, key % c.rows, dim] = what


@pytest.mark.parametrize("HD,rows", [(128, 16), (256, 64)])
@pytest.mark.parametrize("std", [1.0, 16.0])     # (16: one key has nearly all of the weight, and some have none in 32 bits)
def test_values_that_are_infinite_for_single_tokens(bk, HD, rows, std):
    # one sequence, keys in the first, a middle and the last tile, and the new row itself
    c = Case(141, 1, 1, 0, [700], HD=HD, Hq=8, Hkv=1, rows=rows, fused=False, std=std)
    for key, dim, what in ((0, 0, INF), (33, 1, NINF), (300, 2, INF), (301, 2, INF), (640, HD - 1, NINF), (10, 40, INF), (600, 40, NINF), (77, 64, NAN), (698, 65, INF)):
        put(c, 0, key, dim, what)
    c.v[0, 0, 70] = INF
    for key in (33, 300, 640):                      # scores of four times the size: far below or far above the others
        at = c.table[0, key // rows], slice(None), key % rows
        c.kp[at] = bf16(4 * val(c.kp[at]))
    w = as_defined(c)
    assert (w[:, :, [0, 2, 65, 70]] == np.inf).all() and (w[:, :, [1, HD - 1]] == -np.inf).all() and np.isnan(w[:, :, [40, 64]]).all()
    # common rows of several sequences, rows of one sequence, and both at once
    c = Case(142, 5, 1, 450, [1, 100, 20, 0, 64], HD=HD, Hq=12, Hkv=2, rows=rows, fused=False, std=std)
    for b, key, dim, what in ((0, 5, 3, INF), (0, 200, 4, NINF), (0, 430, 60, NAN), (1, 500, 3, INF), (1, 460, 4, INF), (4, 455, 9, NINF)):
        put(c, b, key, dim, what)
    w = as_defined(c)
    assert (w[1, :, 3] == np.inf).all() and np.isnan(w[1, :, 4]).all() and (w[4, :, 9] == -np.inf).all()


@pytest.mark.parametrize("HD", [128, 256])
def test_values_that_are_infinite_for_pieces_of_prompts(bk, HD):
    """The same row of V does the same in tiles that all rows see and in those that some see."""
    T = 12
    c = Case(151, 2, T, 300, [140, 12], HD=HD, Hq=6, Hkv=1, rows=32, fused=False)
    for key, dim, what in ((3, 0, INF), (299, 1, NINF), (330, 2, INF), (420, 3, NINF), (3, 5, INF), (425, 5, NINF)):
        put(c, 0, key, dim, what)
    c.v[7 * 2, 0, 8], c.v[9 * 2 + 1, 0, 9] = NINF, INF
    assert not np.isfinite(as_defined(c)).all()


def test_values_that_are_infinite_in_row_tiles_cut_at_the_same_keys(bk):
    c = Case(161, 2, 70, 1300, [70, 75], new=[70, 31], Hq=16, Hkv=2, HD=256, rows=128, fused=False)
    for key, dim, what in ((0, 0, INF), (640, 1, NINF), (1200, 2, INF), (1310, 3, INF), (64, 200, NINF)):
        put(c, 0, key, dim, what)
    as_defined(c)


# ---- adapters -------------------------------------------------------------------------------

@pytest.mark.parametrize("B,n_adapters,ids", [(1, 2, [1]), (2, 2, [1, 1]), (3, 5, [1, 4, 1]), (4, 2, [1, 0, 1, 1]), (13, 3, [1] * 11 + [0, -1])])
@pytest.mark.parametrize("rank", [8, 24, 32, 64, 72, 128])
@pytest.mark.parametrize("f32", [True, False])
def test_a_weight_that_is_infinite_makes_its_row_infinite(bk, B, n_adapters, ids, rank, f32):
    K, rows = 264, [300]
    args, keep, want, (dx, di, ds, scratch) = lora_case(rank + B, B, K, rows, rank, n_adapters, ids, f32)
    (dA, dM, dbase), out, ld, n = keep[0]
    A, M, x = dA.download(np.uint16, (n_adapters, rank, K)), dM.download(np.uint16, (n_adapters, n, rank)), dx.download(np.uint16, (B, K))
    A[1, rank - 1] = bf16(np.full(K, 0.5))
    x[0] = bf16(np.ones(K) * 0.25)               # u of the last row of A is 33 exactly: a bf16 value, whose other parts are zeros
    M[1, 0, rank - 1], M[1, 17, 3], M[1, 299, 0], M[1, 299, rank - 1], M[1, 40, 5] = INF, NINF, INF, NINF, NAN
    for d, a in ((dA, A), (dM, M), (dx, x)):
        d.upload(a)
    base = dbase.download(np.float32 if f32 else np.uint16, (B, ld))
    scale = ds.download(np.float32, (n_adapters,))
    y = base.astype(np.float64) if f32 else val(base)
    mag = np.abs(y)
    with np.errstate(invalid="ignore"):
        for b, a in enumerate(ids):
            if a >= 0:
                y[b] += float(scale[a]) * (val(M[a]) @ (val(A[a]) @ val(x[b])))
                mag[b] += float(scale[a]) * (np.abs(val(M[a])) @ (np.abs(val(A[a])) @ np.abs(val(x[b]))))
    assert y[0, 0] == np.inf and np.isnan(y[0, 40])
    ops.lora(args)
    assert R.cuSync() == 0, R.last_error()
    raw = out.download(np.uint32 if f32 else np.uint16, (B, ld))
    got = raw.view(np.float32).astype(np.float64) if f32 else val(raw)
    assert np.array_equal(np.isnan(got), np.isnan(y))
    fine = np.isfinite(y)
    assert np.array_equal(got[~fine & ~np.isnan(y)], y[~fine & ~np.isnan(y)]) and np.isfinite(got[fine]).all()
    got, y, mag = got[fine], y[fine], mag[fine]
    assert (np.abs(got - y) <= (K + rank + 4) * 2.0 ** -24 * mag + (0 if f32 else 2.0 ** -8 * np.abs(y))).all()


# ---- row tiles that are cut at the same common keys ----------------------------------------------

LONG = [(64, 1, 150, 2000, [150], None, 8, 1, 128, 64), (65, 2, 70, 1300, [70, 75], [70, 31], 16, 2, 256, 128), (63, 1, 150, 0, [600], None, 8, 1, 128, 16),
        (67, 40, 1, 2500, [1 + 7 * (i % 11) for i in range(40)], None, 8, 1, 256, 64)]


@pytest.mark.parametrize("seed,B,T,prefix,own_rows,new,Hq,Hkv,HD,rows", LONG)
def test_attention_of_many_row_tiles_with_ready_queries(bk, seed, B, T, prefix, own_rows, new, Hq, Hkv, HD, rows):
    """The plan that cuts several row tiles at the same keys, held to the bound without the norm's roundings: a tile of keys left out or taken
    twice moves the result by many times that (tests/test_serving_cpu.py)."""
    Case(seed, B, T, prefix, own_rows, new=new, Hq=Hq, Hkv=Hkv, HD=HD, rows=rows, fused=False).check()


@pytest.mark.parametrize("seed,B,T,prefix,own_rows,new,Hq,Hkv,HD,rows", [c for c in LONG if c[3]])
def test_attention_of_many_row_tiles_is_the_same_whatever_is_shared(bk, seed, B, T, prefix, own_rows, new, Hq, Hkv, HD, rows):
    """The same with norm and rotation: both ways read the same bits of q, k and v."""
    c = Case(seed, B, T, prefix, own_rows, new=new, Hq=Hq, Hkv=Hkv, HD=HD, rows=rows)
    got = []
    for P in (prefix, 0, prefix // 2):
        ops.paged_attn(c.args(prefix_rows=P))
        assert R.cuSync() == 0, R.last_error()
        got.append(val(c.out.download(np.uint16, (T * B, Hq, HD))))
    vmax = np.abs(val(c.vp)[np.isfinite(val(c.vp))]).max()
    vmax = max(vmax, np.abs(val(c.v)).max())
    for g in got[1:]:
        assert (np.abs(g - got[0]) <= 2.0 ** -7 * np.abs(got[0]) + 2.0 ** -12 * vmax).all()
