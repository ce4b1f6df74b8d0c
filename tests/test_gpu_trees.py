"""Drafted trees on the paged cache -- maps of a step, attention, logits, commit -- against plain implementations in 64 bits.

Tolerances.  Attention: those of attention over pages (2^-8 |o| for the one rounding of out, 2^-13 of the largest |v| for 16 bits of probabilities; with
the fused norm 2^-7 of it for values of q that may be rounded the other way).  Logits: every operation of x / r, f n, f n + p, x - y and x + bias rounds by at most 2^-24 of
what it gives, so the result is off by at most 2^-24 (3 |x'| + 3 f n + 2 p + |sum of biases|), x' the penalised logit, and each of the sums of a bias by 2^-24 of the sum of
magnitudes; twice that is allowed.  Tables, lists, masks and moved rows are equal bit for bit.
"""
import ctypes as C
import math

import numpy as np
import pytest

from bunker_b200 import ops
from bunker_b200 import runtime as R
from tests.test_gpu_serving import Case, Pool, bf16, i32, rnd, val
from tests.util import dev

pytestmark = pytest.mark.gpu


def random_tree(rng, T, wide=False):
    """parents of T nodes; now and then a second root"""
    p = [-1]
    for t in range(1, T):
        p.append(-1 if rng.random() < 0.05 else int(rng.integers(0, t)) if wide or rng.random() < 0.5 else t - 1)
    return p


def paths(parent):
    """[node][node]: whether u is t or an ancestor of t"""
    T = len(parent)
    m = np.zeros((T, T), bool)
    for t, u in enumerate(parent):
        if 0 <= u < t:
            m[t] = m[u]
        m[t, t] = True
    return m


def words(m, n_words):
    """bool [...][T] -> uint32 [...][n_words]"""
    bits = np.zeros(m.shape[:-1] + (32 * n_words,), np.uint64)
    bits[..., :m.shape[-1]] = m
    return (bits.reshape(m.shape[:-1] + (n_words, 32)) << np.arange(32, dtype=np.uint64)).sum(-1).astype(np.uint32)


def by_node(rows, T):
    """[sequence][node] -> [node][sequence]"""
    return np.ascontiguousarray(np.array(rows, np.int32).reshape(len(rows), T).T)


# ---- maps of a step -----------------------------------------------------------------

@pytest.mark.parametrize("T,rows,extra", [(1, 16, 0), (7, 5, 0), (32, 64, 1), (33, 16, 0), (64, 1, 0), (100, 32, 2), (1024, 16, 0)])
def test_batch_maps_of_lists_and_trees(bk, T, rows, extra):
    rng = np.random.default_rng(T)
    p = Pool(rng, planes=1, n_pages=max(40, 5 * -(-(T + 70) // rows)), heads=1, rows=rows, row_vals=8, seqs=7, max_pages=-(-(T + 70) // rows))
    order = list(rng.permutation(p.n_pages))
    for s, length in enumerate([T + 3, T, T + 61, max(1, T - 1), 0]):
        p.own(s, length, order)
    if p.table[2, 0] >= 0:
        p.table[2, (T + 60) // rows] = p.n_pages        # names no page
    pool = p.upload()
    seqs = i32(2, 0, 7, -1, 4, 0, 3, 1)
    new = i32(T, max(1, T // 2), T, 1, T, T + 5, T, -2)
    n, W = len(seqs), (T + 31) // 32 + extra
    trees = [random_tree(rng, T, b % 2 == 0) for b in range(n)]
    trees[1][T - 1] = T + 3                              # not an earlier node
    trees[5][T // 2] = -7
    served = i32(1, 1, 1, 1, 1, 1, 0, 1)
    for parent, counts, ok in ((trees, new, None), (None, new, served), (trees, None, served)):
        out = {k: R.DeviceBuffer.from_numpy(np.full(size, 0x5A5A5A5A, np.uint32)) for k, size in
               (("table", n * p.max_pages), ("lens", n), ("pos", T * n), ("slot", T * n), ("mask", T * n * W), ("count", n))}
        d = [dev(seqs), dev(new), dev(by_node(trees, T)), dev(served)]
        pool.batch(d[0].ptr, n, T=T, n_new=d[1].ptr if counts is not None else 0, parent=d[2].ptr if parent else 0, ok=d[3].ptr if ok is not None else 0, mask_words=W, **{k: b.ptr for k, b in out.items()})
        p.check("unchanged")
        table, lens, count = np.full((n, p.max_pages), -1, np.int32), np.zeros(n, np.int32), np.zeros(n, np.int32)
        pos, slot, mask = np.full((T, n), -1, np.int32), np.full((T, n), -1, np.int32), np.zeros((T, n, W), np.uint32)
        for i, s in enumerate(seqs):
            if not 0 <= s < p.seqs:
                continue
            lens[i] = p.lens[s]
            held = p.np_pages(lens[i])
            table[i, :held] = p.table[s, :held]
            m = T if counts is None else min(max(int(new[i]), 0), T)
            if ok is not None and not ok[i]:
                m = 0
            base = int(lens[i]) - m
            if base < 0:
                continue
            count[i] = m
            path = paths(parent[i] if parent else list(range(-1, T - 1)))
            for t in range(m):
                pos[t, i] = base + path[t].sum() - 1
                page = p.table[s, (base + t) // rows]
                slot[t, i] = page * rows + (base + t) % rows if 0 <= page < p.n_pages else -1
                mask[t, i] = words(path[t], W)
        for name, want in (("table", table), ("lens", lens), ("pos", pos), ("slot", slot), ("mask", mask), ("count", count)):
            assert np.array_equal(out[name].download(want.dtype, want.shape), want), name


def test_batch_gives_what_is_asked_for(bk):
    rng = np.random.default_rng(5)
    p = Pool(rng)
    p.own(1, 40, [3, 8, 1])
    pool = p.upload()
    seqs, pos, lens = dev(i32(1)), dev(i32(9, 9)), dev(i32(9))
    pool.batch(seqs.ptr, 1, T=2, pos=pos.ptr)
    pool.batch(seqs.ptr, 1, lens=lens.ptr)
    pool.batch(seqs.ptr, 1)
    pool.batch(0, 0)
    p.check()
    assert pos.download(np.int32, (2,)).tolist() == [38, 39] and lens.download(np.int32, (1,)).tolist() == [40]


@pytest.mark.parametrize("place", ["n_new", "ok"])
def test_batch_counts_in_place(bk, place):
    rng = np.random.default_rng(6)
    p = Pool(rng, n_pages=600, seqs=8, max_pages=66)
    order = list(rng.permutation(600))
    for s in range(8):
        p.own(s, 150 * s, order)
    pool = p.upload()
    seqs = dev(np.tile(np.arange(8, dtype=np.int32), 32))
    for _ in range(20):
        d = {"n_new": dev(np.full(256, 2000, np.int32)), "ok": dev(np.full(256, 3, np.int32))}
        slot = R.DeviceBuffer.from_numpy(np.full(300 * 256, 77, np.int32))
        pool.batch(seqs.ptr, 256, T=300, n_new=d["n_new"].ptr, ok=d["ok"].ptr, count=d[place].ptr, slot=slot.ptr)
        want = np.where(150 * (np.arange(256) % 8) >= 300, 300, 0)
        assert np.array_equal(d[place].download(np.int32, (256,)), want)
        assert np.array_equal((slot.download(np.int32, (300, 256)) >= 0).sum(0), want)
    p.check("unchanged")


def test_batch_of_a_full_list_with_long_tables(bk):
    rng = np.random.default_rng(6)
    p = Pool(rng, planes=1, n_pages=5000, heads=1, rows=2, row_vals=8, seqs=1100, max_pages=3001)
    p.lens[:] = rng.integers(0, 6003, 1100)
    p.table[:] = rng.integers(-1, 5001, p.table.shape)
    pool = p.upload()
    for n in (1, 3, 1024):
        seqs = rng.integers(0, 1100, n).astype(np.int32)
        d, table, lens = dev(seqs), R.DeviceBuffer(4 * n * 3001), R.DeviceBuffer(4 * n)
        pool.batch(d.ptr, n, table=table.ptr, lens=lens.ptr)
        p.check()
        length = np.where(p.lens[seqs] <= 6002, p.lens[seqs], 0)
        assert np.array_equal(lens.download(np.int32, (n,)), length)
        want = np.where(np.arange(3001)[None] < -(-length[:, None] // 2), p.table[seqs], -1)
        assert np.array_equal(table.download(np.int32, (n, 3001)), want)


# ---- attention ----------------------------------------------------------------------

class TreeCase(Case):
    """Trees instead of chains.  ``tree``: "tree", "chain" or "any" (any bits at all, rows that see nothing among them)."""

    def __init__(self, seed, B, T, prefix, own_rows, tree="tree", extra_words=0, **kw):
        super().__init__(seed, B, T, prefix, own_rows, **kw)
        rng = np.random.default_rng(seed + 1000)
        self.W = (T + 31) // 32 + extra_words
        self.sees = np.zeros((T, B, T), bool)
        self.pos = np.full((T, B), -1, np.int32)
        self.slot = np.full((T, B), -1, np.int32)
        for b in range(B):
            n, base = self.n_base(b)
            m = paths(random_tree(rng, T, b % 2 == 1)) if tree == "tree" else np.tril(np.ones((T, T), bool))
            if tree == "any":
                m = rng.random((T, T)) < 0.3
                m[T // 2] = False
            self.sees[:, b] = m
            for t in range(n):
                self.pos[t, b] = base + (m[t].sum() - 1 if tree == "tree" else t)
                self.slot[t, b] = self.table[b, (base + t) // self.rows] * self.rows + (base + t) % self.rows

    def n_base(self, b):
        n = min(max(int(self.new[b]), 0), self.T)
        base = int(self.lens[b]) - n
        return (n, base) if base >= 0 and self.lens[b] <= min(self.max_len, self.max_pages * self.rows) else (0, 0)

    def positions(self):
        """row of (t, b) in its sequence, -1 where it is not there"""
        at = np.full((self.T, self.B), -1)
        for b in range(self.B):
            n, base = self.n_base(b)
            for t in range(n):
                if not self.fused or 0 <= self.pos[t, b] < self.max_len:
                    at[t, b] = base + t
        return at

    def want(self):
        at, kp, vp = self.positions(), self.kp.copy(), self.vp.copy()
        G, out = self.Hq // self.Hkv, np.zeros((self.T * self.B, self.Hq, self.HD))
        for b in range(self.B):
            for t in range(self.T):
                e, slot = t * self.B + b, int(self.slot[t, b])
                if at[t, b] >= 0 and 0 <= slot < self.n_pages * self.rows:
                    page = slot // self.rows, slice(None), slot % self.rows
                    kp[page] = bf16(self.turned(self.k[e], self.kw, self.pos[t, b])) if self.fused else self.k[e]
                    vp[page] = self.v[e]
        for b in range(self.B):
            n, base = self.n_base(b)
            for t in range(self.T):
                e = t * self.B + b
                j = np.concatenate([np.arange(base), base + np.nonzero(self.sees[t, b, :n])[0]])
                if at[t, b] < 0 or not len(j):
                    continue
                K, V = (val(x[self.table[b, j // self.rows], :, j % self.rows]) for x in (kp, vp))
                q = val(bf16(self.turned(self.q[e], self.qw, self.pos[t, b]))) if self.fused else val(self.q[e])
                for h in range(self.Hq):
                    s = K[:, h // G] @ q[h] * float(self.scale)
                    w = np.exp(s - s.max())
                    out[e, h] = w @ V[:, h // G] / w.sum()
                if self.g is not None:
                    out[e] /= 1 + np.exp(-val(self.g[e]))
        return out, kp, vp

    def nothing_seen(self):
        """rows that get zeros"""
        at, none = self.positions(), np.zeros((self.T, self.B), bool)
        for b in range(self.B):
            n, base = self.n_base(b)
            none[:, b] = (at[:, b] < 0) | ((base == 0) & ~self.sees[:, b, :n].any(-1))
        return none.reshape(-1)

    def tree_args(self, **change):
        a = self.args()
        nb = ops.tree_attn_scratch_bytes(self.B, self.T, self.Hq, self.Hkv, self.HD, self.P)
        self.scratch = R.DeviceBuffer.from_numpy(np.full(nb // 4 + 1, 0x7FC00000, np.uint32))
        a.scratch, a.scratch_bytes = self.scratch.ptr, nb
        for name, x in (("pos", self.pos), ("slot", self.slot), ("mask", words(self.sees, self.W))):
            self.keep[name] = dev(x)
        return R.bkTreeAttnArgs(**{**dict(attn=a, pos=self.keep["pos"].ptr, slot=self.keep["slot"].ptr, mask=self.keep["mask"].ptr, mask_words=self.W), **change})

    def run(self, a):
        ops.tree_attn(a)
        assert R.cuSync() == 0, R.last_error()
        return self.out.download(np.uint16, (self.T * self.B, self.Hq, self.HD))

    def check(self, times=2):
        a = self.tree_args()
        want, kp, vp = self.want()
        vmax = np.nanmax(np.abs(np.where(np.isfinite(val(vp)), val(vp), 0)))
        first = None
        for _ in range(times):
            bits = self.run(a)
            got = val(bits)
            assert np.isfinite(got).all()
            tol = 2.0 ** -8 * np.abs(want) + (2.0 ** -7 if self.fused else 2.0 ** -13) * vmax
            bad = np.abs(got - want) > tol
            assert not bad.any(), (np.argwhere(bad)[:5], np.abs(got - want).max(), got[bad][:5], want[bad][:5])
            assert not bits[self.nothing_seen()].any()
            assert first is None or np.array_equal(first, bits)
            first = bits
        k, v = self.keep["kp"].download(np.uint16, self.kp.shape), self.keep["vp"].download(np.uint16, self.vp.shape)
        assert np.array_equal(v, vp)
        changed = kp != self.kp
        assert np.array_equal(k[~changed], kp[~changed])
        assert (np.abs(val(k[changed]) - val(kp[changed])) <= 2.0 ** -7 * np.abs(val(kp[changed])) + 2.0 ** -16).all()


@pytest.mark.parametrize("HD", [128, 256])
@pytest.mark.parametrize("T,before", [(1, 0), (1, 1), (2, 0), (5, 60), (8, 64), (31, 1), (32, 33), (33, 31), (40, 100), (64, 0), (64, 64), (65, 127), (100, 17)])
def test_a_tree_of_one_sequence(bk, T, before, HD):
    TreeCase(T + before, 1, T, 0, [T + before], HD=HD, Hq=4, Hkv=1, fused=T % 2 == 0).check()


@pytest.mark.parametrize("fused", [True, False])
@pytest.mark.parametrize("Hq,Hkv,HD,rows", [(16, 2, 256, 64), (24, 4, 256, 32), (3, 3, 128, 128), (16, 1, 128, 16), (14, 2, 128, 1024)])
def test_trees_behind_a_prefix_by_heads_and_page_sizes(bk, fused, Hq, Hkv, HD, rows):
    TreeCase(Hq + rows, 4, 12, 150, [12, 40, 77, 13], new=[12, 5, 1, 12], Hq=Hq, Hkv=Hkv, HD=HD, rows=rows, fused=fused).check()


@pytest.mark.parametrize("T,new", [(9, [9, 0, 4]), (40, [40, 33, 1]), (130, [130, 64, 97])])
@pytest.mark.parametrize("prefix", [0, 16, 70, 500])
def test_any_mask_over_the_new_rows(bk, T, new, prefix):
    """Bits of later rows, own bits that are not set, rows that see nothing, bits behind the last row."""
    TreeCase(T + prefix, 3, T, prefix, [max(n, 1) + 11 * i for i, n in enumerate(new)], new=new, tree="any", extra_words=T % 2, Hq=6, Hkv=1, HD=128, fused=False).check()


def test_trees_of_many_row_tiles(bk):
    TreeCase(71, 20, 16, 260, [16 + 3 * (i % 5) for i in range(20)], new=[16 - i % 7 for i in range(20)], Hq=8, Hkv=1, HD=256, fused=False).check()   # 2,560 rows behind the prefix
    TreeCase(72, 2, 130, 1300, [200, 131], new=[130, 70], Hq=16, Hkv=2, HD=256, rows=64).check()
    TreeCase(73, 300, 3, 64, [3 + i % 40 for i in range(300)], Hq=4, Hkv=4, HD=128, fused=False).check(1)                                             # 1,200 jobs and more


def test_trees_of_more_sequences_than_are_packed(bk):
    """From 1,025 sequences on ready queries lie T to a sequence."""
    TreeCase(74, 1100, 2, 0, [2 + i % 7 for i in range(1100)], new=[2 - (i % 5 == 0) - (i % 11 == 0) for i in range(1100)], Hq=1, Hkv=1, HD=128, fused=False).check(1)
    TreeCase(75, 1030, 1, 48, [1 + i % 3 for i in range(1030)], new=[int(i % 4 != 1) for i in range(1030)], Hq=2, Hkv=1, HD=128, fused=True).check(1)
    TreeCase(76, 1024, 2, 32, [2 + i % 3 for i in range(1024)], new=[2 - i % 3 for i in range(1024)], Hq=1, Hkv=1, HD=128, fused=False, tree="any").check(1)


def test_a_chain_is_what_attention_over_pages_gives(bk):
    """The same rows in the pages, and the same ready queries: each result is within 2^-8 |o| and 2^-13 of the largest |v| of the exact one for these queries."""
    for seed, prefix, fused in ((81, 0, True), (82, 100, True), (83, 64, False)):
        c = TreeCase(seed, 3, 9, prefix, [9, 50, 20], new=[9, 4, 9], tree="chain", Hq=8, Hkv=1, HD=256, fused=fused)
        tree = val(c.run(c.tree_args()))
        k, v = c.keep["kp"].download(np.uint16, c.kp.shape), c.keep["vp"].download(np.uint16, c.vp.shape)
        ops.paged_attn(c.args())
        assert R.cuSync() == 0
        chain = val(c.out.download(np.uint16, tree.shape))
        vmax = np.abs(val(v)[np.isfinite(val(v))]).max()
        assert (np.abs(chain - tree) <= 2.0 ** -7 * np.maximum(np.abs(chain), np.abs(tree)) + 2.0 ** -12 * vmax).all()
        assert np.array_equal(c.keep["kp"].download(np.uint16, c.kp.shape), k) and np.array_equal(c.keep["vp"].download(np.uint16, c.vp.shape), v)


def test_trees_where_nothing_is_there(bk):
    TreeCase(1, 3, 4, 0, [0, 5, 0], new=[0, 4, 0], HD=128).check()
    TreeCase(2, 2, 3, 0, [2, 1], HD=256, tree="any").check()                    # fewer rows than nodes: none of the sequence's is there
    TreeCase(3, 2, 4, 32, [4, 2], new=[9, -3], HD=128).check()                  # counts outside 0..T
    TreeCase(4, 2, 3, 0, [40, 20], HD=128, max_len=30).check()                  # a sequence longer than the call allows
    c = TreeCase(5, 3, 6, 64, [10, 6, 9], HD=128)                               # sequences shorter than the prefix see only their own part of it
    c.lens = np.array([74, 20, 67], np.int32)
    c.slot[:] = -1                                                              # (and their rows are in the pages already)
    c.kp[c.table[0, :4]], c.vp[c.table[0, :4]] = rnd(np.random.default_rng(1), 2, 4, 1, 16, 128)
    c.check()
    c = TreeCase(6, 2, 5, 0, [30, 25], HD=128)                                  # positions outside the tables, slots in no page
    c.pos[1, 0], c.pos[4, 1] = c.max_len, -1
    for t, b in ((1, 0), (4, 1)):
        c.sees[:, b, t] = False
    c.check()
    c = TreeCase(7, 2, 5, 0, [30, 25], HD=128, fused=False)
    c.slot[2, 0], c.slot[3, 1] = c.n_pages * 16, -5
    for t, b in ((2, 0), (3, 1)):
        c.sees[:, b, t] = False                                                 # (those rows of the pages hold NaN or what was there)
    at = c.table[0, 27 // 16], slice(None), 27 % 16
    c.kp[at] = c.vp[at] = 0
    at = c.table[1, 23 // 16], slice(None), 23 % 16
    c.kp[at] = c.vp[at] = 0
    c.check()


@pytest.mark.parametrize("HD,rows", [(128, 16), (256, 64)])
def test_what_is_not_finite_stays_with_the_nodes_that_see_it(bk, HD, rows):
    T = 12
    c = TreeCase(51, 2, T, 40, [30, 12], HD=HD, Hq=6, Hkv=1, rows=rows, fused=False, gate=False)
    c.v[7 * 2, 0, 3], c.v[7 * 2, 0, HD - 1], c.v[10 * 2, 0, 5], c.k[4 * 2 + 1, 0, 1] = 0x7F80, 0xFF80, 0x7FC0, 0x7FC0
    with np.errstate(invalid="ignore"):
        want, kp, vp = c.want()
    got = val(c.run(c.tree_args())).reshape(T, 2, c.Hq, HD)
    want = want.reshape(T, 2, c.Hq, HD)
    odd = np.zeros(want.shape, bool)
    odd[c.sees[:, 0, 7]][:, 0] = True
    for t in range(T):
        odd[t, 0, :, [3, HD - 1]] |= c.sees[t, 0, 7]
        odd[t, 0, :, 5] |= c.sees[t, 0, 10]
        odd[t, 1] |= c.sees[t, 1, 4]
    assert np.array_equal(~np.isfinite(want), odd)
    assert np.array_equal(~np.isfinite(got), odd)
    assert np.array_equal(np.isnan(got[odd]), np.isnan(want[odd]))
    assert odd.any() and not odd.all(axis=(1, 2, 3)).any()
    vmax = np.abs(val(vp)[np.isfinite(val(vp))]).max()
    assert (np.abs(got[~odd] - want[~odd]) <= 2.0 ** -8 * np.abs(want[~odd]) + 2.0 ** -13 * vmax).all()
    # scores that are all -inf give NaN, none at all zeros
    c = TreeCase(53, 1, 3, 0, [3], HD=HD, Hq=2, Hkv=1, rows=rows, fused=False, gate=False, tree="any")
    c.sees[:] = np.array([[1, 0, 0], [0, 0, 0], [1, 1, 0]], bool)[:, None]
    c.q[:] = bf16(np.ones(c.q.shape))
    c.k[0], c.k[1] = 0xFF80, 0x3F80
    got = val(c.run(c.tree_args()))
    assert np.isnan(got[0]).all() and not got[1].any() and (np.abs(got[2] - val(c.v[1])) <= 2.0 ** -8 * np.abs(val(c.v[1]))).all()


def test_trees_over_pages_beyond_32_bits(bk):
    """Pools of 5 GB of keys and of values: the pages in use lie at their end."""
    c = TreeCase(66, 2, 6, 80, [40, 100], Hq=8, Hkv=2, HD=256, rows=64)
    page = 2 * 64 * 256 * 2
    far = (5 << 30) // page
    shift = far - c.n_pages
    want, kp, vp = c.want()
    big = [R.DeviceBuffer(5 << 30) for _ in range(2)]
    for b, host in zip(big, (c.kp, c.vp)):
        R.cuHtoD(b.ptr + shift * page, host)
    a = c.tree_args()
    table, slot = dev(np.where(c.table >= 0, c.table + shift, -1).astype(np.int32)), dev((c.slot + shift * 64).astype(np.int32))
    a.attn.k_pages, a.attn.v_pages, a.attn.table, a.attn.n_pages, a.slot = big[0].ptr, big[1].ptr, table.ptr, far, slot.ptr
    got = val(c.run(a))
    vmax = np.abs(val(vp)[np.isfinite(val(vp))]).max()
    assert (np.abs(got - want) <= 2.0 ** -8 * np.abs(want) + 2.0 ** -7 * vmax).all()
    back = np.empty_like(c.vp)
    R.cuDtoH(back, big[1].ptr + shift * page)
    assert np.array_equal(back, vp)
    for b in big:
        b.free()


def test_attention_of_trees_refuses_what_it_cannot_do(bk):
    c = TreeCase(9, 2, 40, 0, [50, 41], HD=128)
    lib = R.cu()

    def refused(word, **change):
        a = c.tree_args()
        for k, v in change.items():
            setattr(a.attn if hasattr(a.attn, k) else a, k, v)
        assert lib.bkTreeAttn(C.byref(a)) == R.BK_ERR_ARG and word in R.last_error(), (change, R.last_error())

    refused("mask", mask=0)
    refused("mask", mask_words=1)
    refused("mask", mask=c.tree_args().mask + 2)
    refused("pos", pos=0)
    refused("pos", pos=6)
    refused("slot", slot=0)
    refused("slot", slot=5)
    refused("head_dim", HD=64)
    refused("page_rows", page_rows=24)
    refused("scratch", scratch_bytes=16)
    refused("null", out=0)
    refused("go together", v=0)
    refused("scale", scale=0.0)
    refused("prefix", prefix_rows=-1)
    assert lib.bkTreeAttn(None) == R.BK_ERR_ARG


# ---- logits --------------------------------------------------------------------------

class Logits:
    """Requests, their histories, biases and masks, and the adjusted logits in 64 bits."""

    def __init__(self, seed, B, T, V, history=0, n_bias=0, n_masks=0, allow=0.5, seqs=None, n_seqs=None, tree=False, ld=0, penalties=True, prompts=True, same=False):
        rng = np.random.default_rng(seed)
        n = B if n_seqs is None else n_seqs
        self.B, self.T, self.V, self.ld, self.n_seqs = B, T, V, ld or V, n
        self.x = rng.normal(0, 3, (T * B, self.ld)).astype(np.float32)
        self.seqs = None if seqs is None else np.array(seqs, np.int32)
        self.hist = rng.integers(-2 if not same else 0, min(V, 50 if same else V) + 2, (n, max(history, 1))).astype(np.int32) if history else None
        self.hist_len = rng.integers(0, history + 1, n).astype(np.int32)
        self.hist_len[0] = history
        self.prompt = (self.hist_len // 3).astype(np.int32) if prompts else None
        self.rep, self.pres, self.freq = ((1 + rng.random(n)).astype(np.float32), rng.random(n).astype(np.float32), rng.random(n).astype(np.float32)) if penalties else (None,) * 3
        self.bt = rng.integers(-3, V + 3, (n, n_bias)).astype(np.int32) if n_bias else None
        self.bv = rng.normal(0, 2, (n, n_bias)).astype(np.float32) if n_bias else None
        self.bn = np.array([max(0, n_bias - i) for i in range(n)], np.int32)
        self.W = (V + 31) // 32 + 1
        self.allowed = words(rng.random((n_masks, V)) < allow, self.W) if n_masks else None
        self.mask_id = rng.integers(-1, n_masks + 1, T * B).astype(np.int32)
        self.draft = rng.integers(-1, min(V, 20) + 1, T * B).astype(np.int32) if tree else None
        self.sees = np.stack([paths(random_tree(rng, T)) for _ in range(B)], 1) if tree else None      # [T][B][T]

    def want(self):
        """(logits, how far they may be off, which tokens something names or hides)"""
        y, tol, named = self.x.astype(np.float64), np.zeros(self.x.shape), np.zeros(self.x.shape, bool)
        for b in range(self.B):
            s = b if self.seqs is None else int(self.seqs[b])
            known = 0 <= s < self.n_seqs
            for t in range(self.T):
                r = t * self.B + b
                count, inp = np.zeros(self.V, np.int64), np.zeros(self.V, bool)
                if known and self.hist is not None:
                    m = min(max(int(self.hist_len[s]), 0), self.hist.shape[1])
                    h = self.hist[s, :m]
                    k = 0 if self.prompt is None else min(max(int(self.prompt[s]), 0), m)
                    inp[h[:k][(h[:k] >= 0) & (h[:k] < self.V)]] = True
                    np.add.at(count, h[k:][(h[k:] >= 0) & (h[k:] < self.V)], 1)
                if self.draft is not None:
                    d = self.draft.reshape(self.T, self.B)[self.sees[t, b], b]
                    np.add.at(count, d[(d >= 0) & (d < self.V)], 1)
                x = self.x[r, :self.V].astype(np.float64)
                if known and self.rep is not None:
                    rep, pres, freq = float(self.rep[s]), float(self.pres[s]), float(self.freq[s])
                else:
                    rep, pres, freq = 1.0, 0.0, 0.0
                hit = inp | (count > 0)
                z = np.where(hit, np.where(x > 0, x / rep, x * rep) - (freq * count + pres * (count > 0)), x)
                bias, size = np.zeros(self.V), np.zeros(self.V)
                if known and self.bt is not None:
                    for v, f in zip(self.bt[s, :self.bn[s]], self.bv[s, :self.bn[s]]):
                        if 0 <= v < self.V:
                            bias[v] += f
                            size[v] += abs(f)
                            hit[v] = True
                with np.errstate(invalid="ignore"):
                    tol[r, :self.V] = np.where(hit, 2.0 ** -23 * (3 * np.abs(z) + 3 * freq * count + 2 * pres + 4 * size), 0)
                    z = z + bias
                if self.allowed is not None and 0 <= self.mask_id[r] < len(self.allowed):
                    off = ~((self.allowed[self.mask_id[r]][np.arange(self.V) // 32] >> np.arange(self.V) % 32 & 1).astype(bool))
                    z[off], hit[off] = -np.inf, True
                y[r, :self.V], named[r, :self.V] = z, hit
        return y, tol, named

    def args(self, offset=0, **change):
        self.keep = {}
        raw = np.zeros(self.x.size + 8, np.float32)
        raw[offset:offset + self.x.size] = self.x.reshape(-1)
        self.keep["logits"] = dev(raw)
        kw = dict(logits=self.keep["logits"].ptr + 4 * offset, B=self.B, T=self.T, V=self.V, ld=0 if self.ld == self.V else self.ld, n_seqs=self.n_seqs)
        every = [("seqs", self.seqs), ("history", self.hist), ("hist_len", self.hist_len), ("prompt_len", self.prompt), ("repetition", self.rep), ("presence", self.pres),
                 ("frequency", self.freq), ("bias_token", self.bt), ("bias_value", self.bv), ("allowed", self.allowed), ("draft", self.draft)]
        if self.bt is not None:
            every.append(("bias_n", self.bn))
            kw["bias_ld"] = self.bt.shape[1]
        if self.allowed is not None:
            every.append(("mask_id", self.mask_id))
            kw.update(n_masks=len(self.allowed), allowed_words=self.W)
        if self.hist is not None:
            kw["history_ld"] = self.hist.shape[1]
        if self.draft is not None:
            every.append(("path", words(self.sees, (self.T + 31) // 32)))
            kw["path_words"] = (self.T + 31) // 32
        for k, a in every:
            if a is not None:
                self.keep[k] = dev(a)
                kw[k] = self.keep[k].ptr
        kw.update(change)
        return ops.adjust_logits_args(**kw)

    def check(self, offset=0):
        ops.adjust_logits(self.args(offset))
        assert R.cuSync() == 0, R.last_error()
        got = self.keep["logits"].download(np.float32, (self.x.size + 8,))[offset:offset + self.x.size].reshape(self.x.shape)
        y, tol, named = self.want()
        assert np.array_equal(got.view(np.uint32)[~named], self.x.view(np.uint32)[~named])
        fin = np.isfinite(y)
        assert np.array_equal(np.isnan(got), np.isnan(y)) and np.array_equal(got[~fin & ~np.isnan(y)], y[~fin & ~np.isnan(y)].astype(np.float32))
        bad = np.abs(got[fin] - y[fin]) > tol[fin]
        assert not bad.any(), (np.argwhere(bad)[:4], got[fin][bad][:4], y[fin][bad][:4])
        return got


    def check_bits(self):
        """what nothing names or hides has the bits that it had"""
        ops.adjust_logits(self.args())
        assert R.cuSync() == 0, R.last_error()
        got = self.keep["logits"].download(np.uint32, (self.x.size + 8,))[:self.x.size].reshape(self.x.shape)
        _, _, named = self.want()
        assert np.array_equal(got[~named], self.x.view(np.uint32)[~named])
        return got


@pytest.mark.parametrize("V", [1, 2, 31, 33, 127, 1001, 4096, 8191, 8193, 40000, 151936])
@pytest.mark.parametrize("what", ["history", "bias", "mask", "all"])
def test_logits_by_vocabulary(bk, V, what):
    on = lambda k: what in (k, "all")  # noqa: E731
    Logits(V, 3, 1, V, history=200 if on("history") else 0, n_bias=40 if on("bias") else 0, n_masks=3 if on("mask") else 0).check()


@pytest.mark.parametrize("B,T,V", [(1, 2, 500), (2, 33, 1500), (3, 100, 700), (16, 16, 9001), (1, 64, 20000), (40, 3, 8192)])
@pytest.mark.parametrize("masks", [0, 5])
def test_logits_of_trees(bk, B, T, V, masks):
    Logits(B + T, B, T, V, history=300, n_bias=7, n_masks=masks, tree=True).check()


def test_logits_of_paths_alone_and_of_no_history(bk):
    Logits(1, 2, 9, 900, tree=True).check()
    Logits(2, 2, 1, 900).check()                                              # nothing names anything
    Logits(3, 2, 1, 900, history=50, penalties=False).check()                 # penalties of 1, 0, 0
    Logits(4, 2, 1, 900, history=50, prompts=False).check()


@pytest.mark.parametrize("offset,ld", [(0, 1008), (1, 0), (2, 1003), (3, 1001), (4, 1024)])
def test_logits_rows_anywhere(bk, offset, ld):
    """Rows that start on no multiple of 16 bytes, rows apart: what lies between is left as it is."""
    Logits(offset, 5, 2, 1001, history=100, n_bias=5, n_masks=2, tree=True, ld=ld).check(offset)


def test_logits_of_requests_in_any_order(bk):
    Logits(7, 6, 1, 3000, history=400, n_bias=20, n_masks=4, seqs=[5, 0, 5, 9, -1, 2], n_seqs=9).check()


def test_logits_of_long_histories_of_few_tokens(bk):
    """Counts in the thousands, histories of odd lengths (rows on no multiple of 16 bytes)."""
    Logits(8, 3, 1, 2000, history=70001, same=True).check()
    Logits(9, 2, 4, 151936, history=33333, n_bias=300, n_masks=2, tree=True).check()


@pytest.mark.parametrize("B,T,V,history,n_bias", [(64, 1, 30000, 1, 0), (64, 1, 30000, 300, 5), (160, 1, 9000, 6000, 40), (150, 1, 16500, 6143, 1), (150, 1, 16500, 6145, 0),
                                                  (20, 8, 20000, 5000, 1024), (150, 1, 40000, 9000, 3), (8, 40, 33000, 2000, 0)])
def test_logits_of_many_requests(bk, B, T, V, history, n_bias):
    """Slices of words and tables, histories around what a table holds, repeated tokens."""
    c = Logits(B + history, B, T, V, history=history, n_bias=n_bias, n_masks=3, tree=T > 1)
    c.hist[:, ::3] = c.hist[:, :1]
    c.check()


def test_logits_of_a_token_that_a_request_names_often(bk):
    c = Logits(10, 2, 1, 5000, history=30, n_bias=1024)
    c.bt[0, ::2], c.bt[1, 1000:] = 17, 4999
    c.check()
    c.bn[:] = [2000, -4]            # clamped: all, none
    a = c.args()
    ops.adjust_logits(a)
    assert R.cuSync() == 0
    got = c.keep["logits"].download(np.float32, (c.x.size + 8,))[:c.x.size].reshape(c.x.shape)
    c.bn[:] = [1024, 0]
    y, tol, _ = c.want()
    assert (np.abs(got - y) <= tol).all()


def test_logits_that_are_not_finite(bk):
    c = Logits(11, 2, 1, 600, history=100, n_bias=10, n_masks=2)
    c.x[0, ::7], c.x[0, 1::7], c.x[1, ::5], c.x[1, 1::5] = np.nan, np.inf, -np.inf, np.finfo(np.float32).min
    c.mask_id[:] = [0, -1]
    c.bv[1, 0] = np.inf
    c.rep[1] = 1.0                   # (the lowest value times a penalty is -inf in 32 bits)
    c.pres[1] = c.freq[1] = 0
    c.bt[1, 1:] = -1
    c.check()


def test_a_token_drafted_elsewhere_is_left_as_it_is(bk):
    """A NaN's own bits, a zero's sign: rows whose path does not hold the token do not touch it."""
    c = Logits(16, 1, 3, 300, tree=True)
    c.draft[:] = [7, 8, 9]
    c.sees[:, 0] = np.array([[1, 0, 0], [1, 1, 0], [1, 0, 1]], bool)
    c.x.view(np.uint32)[:, 7:10] = [0x7FC12345, 0x80000000, 0xFFC00001]
    got = c.check_bits()
    assert (got[[0, 2], 8] == 0x80000000).all() and (got[[0, 1], 9] == 0xFFC00001).all()


def test_logits_then_the_argmax_and_a_sample(bk):
    """As a server calls them: what a mask hides is never chosen, a bias of a hundred is."""
    B, V = 4, 151936
    c = Logits(12, B, 1, V, history=500, n_bias=3, n_masks=2, allow=0.001)
    c.mask_id[:] = [0, 1, -1, -1]
    c.bt[3, 0], c.bv[3, 0], c.bn[3] = 4242, 100.0, 1
    a = c.args()
    ops.adjust_logits(a)
    idx, val_, scratch = R.DeviceBuffer(4 * B), R.DeviceBuffer(4 * B), R.DeviceBuffer.zeros(ops.argmax_scratch_bytes(B))
    y, _, _ = c.want()
    ops.argmax(a.logits, V, B, idx.ptr, val_.ptr, scratch.ptr)
    assert np.array_equal(idx.download(np.int32, (B,)), y.argmax(1)) and idx.download(np.int32, (B,))[3] == 4242
    for step in range(5):
        ops.sample(a.logits, V, B, idx.ptr, temperature=1.5, top_k=40, seed=7, step_add=step)
        got = idx.download(np.int32, (B,))
        assert np.isfinite(y[np.arange(B), got]).all()


def test_logits_refuse_what_they_cannot_do(bk):
    c = Logits(13, 2, 3, 100, history=10, n_bias=4, n_masks=2, tree=True)
    lib = R.cu()

    def refused(word, **change):
        a = c.args(**change)
        assert lib.bkAdjustLogits(C.byref(a)) == R.BK_ERR_ARG and word in R.last_error(), (change, R.last_error())

    for change in (dict(logits=0), dict(logits=6)):
        refused("logits", **change)
    for change in (dict(B=0), dict(B=65536), dict(T=0), dict(T=1025), dict(V=0), dict(V=(1 << 30) + 1)):
        refused("B=", **change)
    refused("ld=", ld=99)
    refused("n_seqs", n_seqs=-1)
    refused("32-bit", draft=c.args().draft + 1)
    for change in (dict(hist_len=0), dict(history_ld=0), dict(history_ld=(1 << 29) + 1)):
        refused("history", **change)
    for change in (dict(draft=0), dict(path=0), dict(path_words=0)):
        refused("path", **change)
    for change in (dict(bias_token=0), dict(bias_value=0), dict(bias_n=0), dict(bias_ld=0), dict(bias_ld=1025)):
        refused("bias", **change)
    for change in (dict(allowed=0), dict(mask_id=0), dict(n_masks=0), dict(allowed_words=3)):
        refused("allowed", **change)
    assert lib.bkAdjustLogits(None) == R.BK_ERR_ARG
    assert R.cuSync() == 0


# ---- what stays ----------------------------------------------------------------------

class Draft(Pool):
    """A pool whose sequences end with drafted trees, and the same in numpy."""

    def grown(self, rng, T, new, tokens=12):
        self.T, self.new = T, np.array(new, np.int32)
        n = len(new)
        self.parent = by_node([random_tree(rng, T) for _ in range(n)], T)
        self.token, self.target = rng.integers(0, tokens, (T, n)).astype(np.int32), rng.integers(0, tokens, (T, n)).astype(np.int32)

    def agree(self, rng, i, node):
        """the model agrees with the path to `node` of entry i"""
        t = int(node)
        while self.parent[t, i] >= 0:
            self.target[self.parent[t, i], i] = self.token[t, i]
            t = self.parent[t, i]

    def commit(self, seqs, history=None, hist_len=None):
        n, seen = len(seqs), set()
        path, n_path, nxt, ok = np.full((self.T, n), -1, np.int32), np.zeros(n, np.int32), np.full(n, -1, np.int32), np.zeros(n, np.int32)
        ref0 = self.ref.copy()
        for i, s in enumerate(seqs):
            m = int(self.new[i])
            first = s not in seen
            seen.add(s)
            if not first or not 0 <= s < self.seqs or not 1 <= m <= self.T or self.lens[s] < m:
                continue
            base, end = int(self.lens[s]) - m, self.np_pages(self.lens[s])
            pages = self.table[s, base // self.rows:end]
            if (pages < 0).any() or (pages >= self.n_pages).any() or (ref0[pages] != 1).any():
                continue
            walk = [0]
            while True:
                kids = [t for t in range(walk[-1] + 1, m) if self.parent[t, i] == walk[-1] and self.token[t, i] == self.target[walk[-1], i]]
                if not kids:
                    break
                walk.append(kids[0])
            if history is not None:
                h = int(hist_len[s])
                if h < 0 or h + len(walk) > history.shape[1]:
                    continue
                history[s, h:h + len(walk)] = [self.token[t, i] for t in walk]
                hist_len[s] += len(walk)
            ok[i], n_path[i], nxt[i] = 1, len(walk), self.target[walk[-1], i]
            path[:len(walk), i] = walk
            src = [(self.table[s, (base + t) // self.rows], (base + t) % self.rows) for t in walk]
            rows = [self.data[:, pg, :, r].copy() for pg, r in src]
            for k, x in enumerate(rows):
                self.data[:, self.table[s, (base + k) // self.rows], :, (base + k) % self.rows] = x
            keep = self.np_pages(base + len(walk))
            self.ref[self.table[s, keep:end]] -= 1
            self.table[s, keep:end] = -1
            self.lens[s] = base + len(walk)
        return path, n_path, nxt, ok

    def run(self, seqs, history=None, hist_len=None, n_new=True):
        n = len(seqs)
        pool = self.upload()
        d = {k: dev(x) for k, x in (("seqs", seqs), ("parent", self.parent), ("token", self.token), ("target", self.target), ("n_new", self.new))}
        if not n_new:
            d.pop("n_new")
        o = {k: R.DeviceBuffer.from_numpy(np.full(size, 77, np.int32)) for k, size in (("path", self.T * n), ("n_path", n), ("next", n), ("ok", n))}
        hist = {}
        if history is not None:
            d["history"], d["hist_len"] = dev(history), dev(hist_len)
            hist = dict(history_ld=history.shape[1])
        pool.commit(n=n, T=self.T, **{k: b.ptr for k, b in {**d, **o}.items()}, **hist)
        want = self.commit(seqs, history, hist_len)
        self.check("commit")
        for (name, b), w in zip(o.items(), want):
            assert np.array_equal(b.download(np.int32, w.shape), w), name
        if history is not None:
            assert np.array_equal(d["history"].download(np.int32, history.shape), history)
            assert np.array_equal(d["hist_len"].download(np.int32, hist_len.shape), hist_len)
        return want


@pytest.mark.parametrize("T,rows,row_vals,planes,heads", [(1, 16, 8, 1, 1), (2, 1, 8, 2, 3), (8, 16, 128, 2, 1), (24, 16, 256, 3, 2), (64, 5, 264, 1, 1), (64, 64, 256, 6, 4), (200, 16, 16, 2, 1),
                                                          (1024, 32, 8, 1, 1)])
def test_commit_keeps_the_path_that_the_model_agrees_with(bk, T, rows, row_vals, planes, heads):
    rng = np.random.default_rng(T + rows)
    before = [0, 3, rows, 2 * rows - 1, 40]
    seqs = i32(3, 0, 4, 1, 2)
    need = sum(-(-(b + T) // rows) for b in before)
    p = Draft(rng, planes, need + 4, heads, rows, row_vals, seqs=6, max_pages=-(-(40 + 2 * rows + T) // rows) + 1)
    order = list(rng.permutation(need + 4))
    new = [T, max(1, T - 1), T, max(1, T // 2), T]
    for i, s in enumerate(seqs):
        p.own(int(s), before[i] + new[i], order)
    p.grown(rng, T, new, tokens=T + 5)
    p.agree(rng, 0, T - 1)
    p.agree(rng, 2, T // 2)
    p.parent[1:, 4] = np.arange(T - 1)                        # a chain, all of it agreed with
    p.agree(rng, 4, T - 1)
    history, hist_len = rng.integers(0, 99, (6, T + 9)).astype(np.int32), i32(0, 5, 8, 9, 2, 1)
    path, n_path, nxt, ok = p.run(seqs, history, hist_len)
    assert ok.all() and n_path[4] == T


def test_commit_takes_the_lowest_child_and_ignores_bad_parents(bk):
    rng = np.random.default_rng(2)
    p = Draft(rng, seqs=3)
    p.own(1, 30, [4, 9])
    p.grown(rng, 8, [8])
    p.parent[:, 0] = [5, 0, 0, 9, -3, 2, 1, 4]               # (node 0 has no parent, whatever is there)
    p.token[:, 0] = [1, 7, 7, 7, 7, 6, 6, 6]
    p.target[:, 0] = 7
    p.target[1, 0] = 6
    path, n_path, nxt, ok = p.run(i32(1))
    assert path[:, 0].tolist() == [0, 1, 6, -1, -1, -1, -1, -1] and nxt[0] == 7
    p = Draft(rng, seqs=3)                                    # all of T without counts
    p.own(1, 30, [4, 9])
    p.grown(rng, 8, [8])
    p.run(i32(1), n_new=False)


def test_commit_refuses_a_sequence_and_serves_the_others(bk):
    rng = np.random.default_rng(3)
    p = Draft(rng, n_pages=40, seqs=10, max_pages=4)
    order = list(rng.permutation(40))
    for s, length in enumerate([20, 20, 3, 33, 33, 20, 20, 20, 50]):
        p.own(s, length, order)
    p.ref[p.table[1, 1]] = 2                                  # its last page is shared: in sequence 9 too
    p.table[9, :2], p.lens[9] = p.table[1, :2], 20
    p.ref[p.table[1, 0]] = 2
    p.ref[p.table[3, 0]] = 2                                  # a shared page before the tree
    p.table[6, 1] = 40                                        # no page of the pool
    seqs = i32(0, 1, 2, 3, 4, 5, 6, 10, -1, 0, 7, 8, 9)
    p.grown(rng, 6, [6, 4, 6, 6, 0, 7, 4, 3, 3, 6, -1, 6, 4])
    history, hist_len = np.zeros((10, 40), np.int32), i32(0, 0, 0, 34, 0, 0, 0, 0, 40, 0)
    for i in range(len(seqs)):
        p.agree(rng, i, 3)
    table6 = p.table[6].copy()
    path, n_path, nxt, ok = p.run(seqs, history, hist_len)
    assert ok.tolist() == [1, 0, 0, 1, 0, 0, 0, 0, 0, 0, 0, 0, 0] and np.array_equal(p.table[6], table6)


def test_commit_of_planes_apart_by_more_than_32_bits(bk):
    rng = np.random.default_rng(8)
    p = Draft(rng, 2, 4, 1, 16, 16, seqs=2, max_pages=2)
    p.own(0, 30, [2, 1])
    p.grown(rng, 12, [12], tokens=1000)
    p.parent[1:, 0] = [0, 0, 2, 3, 3, 5, 5, 7, 8, 8, 10]
    p.agree(rng, 0, 11)
    gap, size = 5 << 30, 4 * 16 * 16 * 2
    big = R.DeviceBuffer(gap + size)
    pool = p.upload()
    for i in range(2):
        R.cuHtoD(big.ptr + i * gap, p.data[i])
    pool.desc.base, pool.desc.plane_bytes = big.ptr, gap
    d = {k: dev(x) for k, x in (("seqs", i32(0)), ("parent", p.parent), ("token", p.token), ("target", p.target))}
    pool.commit(n=1, T=12, **{k: b.ptr for k, b in d.items()})
    _, n_path, _, _ = p.commit(i32(0))
    assert R.cuSync() == 0 and n_path[0] == 8      # 0, 2, 3, 5, 7, 8, 10, 11
    got = np.empty_like(p.data)
    for i in range(2):
        R.cuDtoH(got[i], big.ptr + i * gap)
    assert np.array_equal(got, p.data)
    big.free()


def test_maps_and_commit_refuse_what_they_cannot_do(bk):
    rng = np.random.default_rng(4)
    p = Draft(rng)
    p.own(0, 20, [3, 4])
    p.grown(rng, 4, [4])
    pool = p.upload()
    a = dev(np.zeros(64, np.int32))
    lib = R.cu()

    def batch(word, **change):
        x = R.bkPagesBatchArgs(**{**dict(seqs=a.ptr, n=1, T=4, mask=a.ptr, mask_words=1), **change})
        assert lib.bkPagesBatch(C.byref(pool.desc), C.byref(x)) == R.BK_ERR_ARG and word in R.last_error(), (change, R.last_error())

    def commit(word, **change):
        x = R.bkPagesCommitArgs(**{**dict(seqs=a.ptr, parent=a.ptr, token=a.ptr, target=a.ptr, n=1, T=4), **change})
        assert lib.bkPagesCommit(C.byref(pool.desc), C.byref(x)) == R.BK_ERR_ARG and word in R.last_error(), (change, R.last_error())

    for call in (batch, commit):
        call("list", n=-1)
        call("list", n=1025)
        call("list", seqs=0)
        call("list", seqs=a.ptr + 2)
        call("T=", T=0)
        call("T=", T=1025)
        call("arrays", parent=a.ptr + 1)
    batch("mask_words", mask_words=0)
    batch("mask_words", T=33)
    batch("arrays", slot=a.ptr + 2)
    commit("parent", parent=0)
    commit("parent", token=0)
    commit("parent", target=0)
    commit("arrays", ok=a.ptr + 1)
    for result in ("path", "n_path", "next", "ok"):
        commit("apart", **{result: a.ptr})
        commit("apart", **{result: a.ptr + 64, "n_new": a.ptr + 64})
    commit("history", history=a.ptr)
    commit("history", hist_len=a.ptr)
    commit("history", history=a.ptr, hist_len=a.ptr)
    desc = type(pool.desc).from_buffer_copy(pool.desc)
    desc.scratch_bytes = 16
    for fn, x in ((lib.bkPagesBatch, R.bkPagesBatchArgs(seqs=a.ptr, n=1, T=1)), (lib.bkPagesCommit, R.bkPagesCommitArgs(seqs=a.ptr, parent=a.ptr, token=a.ptr, target=a.ptr, n=1, T=1))):
        assert fn(C.byref(pool.desc), None) == R.BK_ERR_ARG and fn(None, C.byref(x)) == R.BK_ERR_ARG
        assert fn(C.byref(desc), C.byref(x)) == R.BK_ERR_ARG
    p.check("nothing changed")


# ---- all of it together ----------------------------------------------------------------

def test_drafted_trees_give_the_tokens_of_single_steps(bk):
    """A one-layer model served to four requests behind a prompt, greedy under penalties, biases and a grammar: token by token, then with drafted trees whose branches hold those
    tokens and others.  Wherever the best logit is clear of the second, the same tokens come out, as many at once as were drafted right."""
    from bunker_b200 import shared_prompt as S
    from bunker_b200.model import CONFIG_TINY as cfg
    rng = np.random.default_rng(77)
    N, P, STEPS, T, H, V = 4, 83, 25, 9, cfg.hidden, cfg.vocab
    w, lora = S.random_layer(cfg, seed=3)
    f = dev(rng.normal(0, 1, (V, H)).astype(np.float32))
    table = R.DeviceBuffer(V * H // 256 * 144)
    ops.quantize_q4k(f.ptr, V, H, table.ptr)
    adapters = [0, -1, 2, 1]
    history = np.zeros((N, P + STEPS + 40), np.int32)
    history[:, :P] = rng.integers(0, V, P)
    history[:, P] = [5, 6, 7, 8]                                          # the first token of each
    rules = dict(rep=np.array([1.3, 1.0, 1.1, 2.0], np.float32), pres=np.array([0.5, 0, 0.2, 0], np.float32), freq=np.array([0.1, 0.3, 0, 0], np.float32))
    d_rules = {k: dev(v) for k, v in rules.items()}
    prompt_len = dev(np.full(N, P, np.int32))
    allowed = dev(words(rng.random((2, V)) < 0.5, V // 32))
    bias_t, bias_v, bias_n = dev(rng.integers(0, V, (N, 3)).astype(np.int32)), dev(rng.normal(0, 3, (N, 3)).astype(np.float32)), dev(i32(3, 0, 2, 1))
    ids, x, hq = R.DeviceBuffer(4 * 64), R.DeviceBuffer(64 * H * 2), R.DeviceBuffer(64 * H // 32 * 36)
    logits, best, top = R.DeviceBuffer(64 * V * 4), R.DeviceBuffer(4 * 64), R.DeviceBuffer(4 * 64)
    scratch = R.DeviceBuffer.zeros(ops.argmax_scratch_bytes(64))

    def layer():
        s = S.SharedPrompt(cfg, w, lora, N, P + STEPS + 60, 60)
        ids_p, xp = dev(history[0, :P]), R.DeviceBuffer(P * H * 2)
        for at in range(0, P, 64):
            ops.embed(table.ptr, H, ids_p.ptr + 4 * at, min(64, P - at), xp.ptr + at * H * 2)
        s.prompt(xp.ptr, P)
        assert s.fork(range(N)).all()
        return s

    def head(out, rows, hist, hist_len, tree=None):
        """logits of `rows` rows under the rules -> greedy tokens in `best`"""
        ops.quant_q8_1(out, H, rows, hq.ptr, bf16=True)
        ops.gemv(hq.ptr, H, rows, [ops.gemv_seg(table.ptr, V, logits.ptr)], order=1)
        mask_id = dev(np.tile(i32(0, -1, 1, -1), rows // N))
        more = dict(T=rows // N, draft=tree[0].ptr, path=tree[1], path_words=2) if tree else dict(T=1)
        ops.adjust_logits(ops.adjust_logits_args(
            logits=logits.ptr, V=V, B=N, history=hist.ptr, history_ld=history.shape[1], hist_len=hist_len.ptr, prompt_len=prompt_len.ptr, repetition=d_rules["rep"].ptr,
            presence=d_rules["pres"].ptr, frequency=d_rules["freq"].ptr, bias_token=bias_t.ptr, bias_value=bias_v.ptr, bias_n=bias_n.ptr, bias_ld=3, allowed=allowed.ptr,
            mask_id=mask_id.ptr, n_masks=2, allowed_words=V // 32, **more))
        ops.argmax(logits.ptr, V, rows, best.ptr, top.ptr, scratch.ptr)
        assert R.cuSync() == 0, R.last_error()      # (mask_id)

    # token by token
    s, said, clear = layer(), history.copy(), np.zeros((N, STEPS), bool)
    for step in range(STEPS):
        ids.upload(np.ascontiguousarray(said[:, P + step]))
        ops.embed(table.ptr, H, ids.ptr, N, x.ptr)
        h, n = dev(said), dev(np.full(N, P + step + 1, np.int32))           # (the token of this step among them: there is no path)
        head(s.step(x.ptr, adapters), N, h, n)
        y = np.sort(logits.download(np.float32, (N, V)), 1)
        # results of attention that are rounded the other way move a logit by a few 2^-8 of the hidden state's part in it
        clear[:, step] = y[:, -1] - y[:, -2] > 2.0 ** -4 * y[np.isfinite(y)].std()
        said[:, P + step + 1] = best.download(np.int32, (N,))
    assert clear.mean() > 0.5

    # with trees: a spine of the tokens that will come, the last of them wrong in some, branches of other tokens
    s, at, hist, hist_len = layer(), np.zeros(N, np.int64), dev(history), dev(np.full(N, P, np.int32))
    many = 0
    while at.min() < STEPS - T:
        parent, token = np.zeros((T, N), np.int32), np.zeros((T, N), np.int32)
        for i in range(N):
            line = said[i, P + at[i]:P + at[i] + T]
            parent[:, i] = [-1, 0, 0, 2, 3, 1, 4, 6, 2]                    # right: 0, 2, 3, 4, 6, 7
            token[:, i] = [line[0], line[1] + 1, line[1], line[2], line[3], line[2], line[4], line[5] + i % 2, line[2] + 1]
        token %= V
        flat = dev(token.reshape(-1))
        ops.embed(table.ptr, H, flat.ptr, T * N, x.ptr)
        out = s.draft(x.ptr, parent, adapters)
        head(out, T * N, hist, hist_len, (flat, s.b_mask.ptr))
        target = best.download(np.int32, (T, N))
        d = [dev(parent.reshape(-1)), s.lists["parent"]]
        assert np.array_equal(d[0].download(np.int32, (T * N,)), d[1].download(np.int32, (64,))[:T * N])
        kept, after = s.keep(token, best.ptr)
        lens = s.lens.download(np.int32, (N + 1,))
        h, n = hist.download(np.int32, history.shape), hist_len.download(np.int32, (N,))
        for i in range(N):
            assert 1 <= kept[i] <= 6 and lens[i + 1] == P + at[i] + kept[i]
            right = [0, 2, 3, 4, 6, 7][:6 if i % 2 == 0 else 5]
            for k, node in enumerate(right[:kept[i]]):
                if clear[i, at[i] + k]:
                    assert target[node, i] == said[i, P + at[i] + k + 1], (i, at[i], k)
            if clear[i, at[i]:at[i] + len(right)].all():
                assert kept[i] == len(right) and after[i] == said[i, P + at[i] + kept[i]]
                many += 1
            # go on along the tokens of the single steps
            h[i, n[i]:n[i] + kept[i]] = said[i, P + at[i]:P + at[i] + kept[i]]
        if (kept < [6, 5, 6, 5]).any() or any(said[i, P + at[i] + kept[i]] != after[i] for i in range(N)):
            break                                                          # (a near tie: the streams part)
        hist.upload(h)
        hist_len.upload((n + kept).astype(np.int32))
        at += kept
    assert many >= 4


def test_drafts_are_refused_where_they_do_not_fit(bk):
    from bunker_b200 import shared_prompt as S
    from bunker_b200.model import CONFIG_TINY as cfg
    w, lora = S.random_layer(cfg, seed=4)
    s = S.SharedPrompt(cfg, w, lora, 3, 64, 6)                              # six pages of 16 rows
    x = dev(rnd(np.random.default_rng(1), 64, cfg.hidden))
    s.prompt(x.ptr, 32)
    assert s.fork([0, 2]).tolist() == [True, True]
    chain = np.array([[-1] * 3] + [[t] * 3 for t in range(16)], np.int32)   # 17 nodes take two pages: four are free
    for bad in (np.zeros((22, 3), np.int32), np.zeros((3, 2), np.int32), np.zeros((0, 3), np.int32)):
        with pytest.raises(ValueError):
            s.draft(x.ptr, bad, [-1] * 3)
    for kw in (dict(adapters=[-1] * 2), dict(adapters=[-1] * 3, n_new=[1, 2]), dict(adapters=[-1] * 3, n_new=[18, 1, 1])):
        with pytest.raises(ValueError):
            s.draft(x.ptr, chain, **kw)
    with pytest.raises(RuntimeError):
        s.keep(chain, x.ptr)
    s.draft(x.ptr, chain, [-1] * 3)
    assert s.b_count.download(np.int32, (3,)).tolist() == [17, 0, 17]
    for call in (lambda: s.step(x.ptr, [-1] * 3), lambda: s.draft(x.ptr, chain, [-1] * 3), lambda: s.fork([1]), lambda: s.drop([0]), lambda: s.prompt(x.ptr, 1)):
        with pytest.raises(RuntimeError):
            call()
    with pytest.raises(ValueError):
        s.keep(chain[:3], x.ptr)
    token = np.arange(51, dtype=np.int32).reshape(17, 3)
    target = np.full((17, 3), 99, np.int32)
    target[:, 2] = np.append(token[1:, 2], 77)
    t = dev(target)
    kept, after = s.keep(token, t.ptr)
    assert kept.tolist() == [1, 0, 17] and after.tolist() == [99, -1, 77]
    assert s.lens.download(np.int32, (4,)).tolist() == [32, 33, 0, 49]
    # request 2 holds two pages, request 0 one, one is free: 16 more nodes fit for the first of the list alone
    s.draft(x.ptr, chain[:16], [-1] * 3, share=False)
    assert s.b_count.download(np.int32, (3,)).tolist() == [16, 0, 0]
    before, lens = s.data.download(np.uint16, (2, 6, 1, 16, cfg.head_dim)), s.lens.download(np.int32, (4,))
    assert lens.tolist() == [32, 49, 0, 49]
    kept, after = s.keep(token[:16], t.ptr)
    assert kept.tolist() == [1, 0, 0] and s.lens.download(np.int32, (4,)).tolist() == [32, 34, 0, 49]
    table = s.table.download(np.int32, (4, s.max_pages))
    mine = table[3, :4]
    assert np.array_equal(s.data.download(np.uint16, before.shape)[:, mine], before[:, mine])      # the refused one's rows are what they were
