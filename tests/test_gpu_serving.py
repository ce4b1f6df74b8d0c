"""Paged cache, attention over pages behind a shared prefix, and adapters, against plain implementations in 64 bits.

Tolerances.  bf16 has 8 significant bits: between 1 and 2 its values are 2^-7 apart, so rounding moves a value by at most 2^-8 of it, and f32 against
f64, which may turn a rounding, by at most 2^-7.
  attention  out is rounded once: 2^-8 |o|; probabilities carry 16 bits, scores and sums 24, exp2 about 21: below 2^-13 of the largest |v|.
             With the fused norm a value of q may be rounded the other way, which moves a score by 2^-7 |q_i k_i| scale < 2^-7 for nearly all values
             drawn here, and o by at most as much of the largest |v|.
  k rows     one rounding, which may be turned: 2^-7 of the value (and 2^-16 where a rotation cancels).
  adapters   f32 sums of K and rank terms: (K + rank) 2^-24 of the sum of magnitudes; bf16 outputs 2^-8 |y| more.
Tables, counts, lists and copied rows are equal bit for bit.
"""
import ctypes as C
import math

import numpy as np
import pytest

from bunker_b200 import ops
from bunker_b200 import pages as PG
from bunker_b200 import runtime as R
from tests.util import dev

pytestmark = pytest.mark.gpu


def bf16(x):
    """f64/f32 -> bf16 patterns, to nearest even (finite values)"""
    u = np.ascontiguousarray(np.asarray(x, np.float32)).view(np.uint32)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def val(h):
    return (np.asarray(h, np.uint16).astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def rnd(rng, *shape, std=1.0):
    return bf16(rng.normal(0, std, shape))


# ---- pages -------------------------------------------------------------------------

class Pool:
    """A pool on the device and the same in numpy."""

    def __init__(self, rng, planes=2, n_pages=24, heads=2, rows=16, row_vals=8, seqs=6, max_pages=6):
        self.shape = (planes, n_pages, heads, rows, row_vals)
        self.rows, self.n_pages, self.seqs, self.max_pages = rows, n_pages, seqs, max_pages
        self.data = rng.integers(0, 65536, self.shape).astype(np.uint16)
        self.ref = np.zeros(n_pages, np.int32)
        self.table = np.full((seqs, max_pages), -1, np.int32)
        self.lens = np.zeros(seqs, np.int32)

    def own(self, s, length, order):
        """sequence s gets `length` rows in the pages `order` takes"""
        n = -(-length // self.rows)
        self.table[s, :n] = [order.pop() for _ in range(n)]
        self.ref[self.table[s, :n]] += 1
        self.lens[s] = length

    def upload(self):
        self.d = {k: dev(getattr(self, k)) for k in ("data", "ref", "table", "lens")}
        nb = PG.scratch_bytes(self.n_pages, self.seqs)
        self.scratch = R.DeviceBuffer(nb)
        planes, n_pages, heads, rows, row_vals = self.shape
        self.pool = PG.PagePool(base=self.d["data"].ptr, n_planes=planes, n_pages=n_pages, heads=heads, page_rows=rows, row_bytes=2 * row_vals,
                                n_seqs=self.seqs, max_pages=self.max_pages, ref=self.d["ref"].ptr, table=self.d["table"].ptr, lens=self.d["lens"].ptr,
                                scratch=self.scratch.ptr, scratch_bytes=nb)
        return self.pool

    def check(self, what=""):
        assert R.cuSync() == 0, R.last_error()
        for k in ("lens", "table", "ref", "data"):
            want = getattr(self, k)
            got = self.d[k].download(want.dtype, want.shape)
            assert np.array_equal(got, want), (what, k, got, want)

    # the rules, one request after the other
    def free_pages(self):
        return list(np.nonzero(self.ref == 0)[0])

    def np_pages(self, rows):
        return -(-int(rows) // self.rows)

    def fork(self, src, dst):
        start, free, seen, need, ok = self.lens.copy(), self.free_pages(), set(), 0, []
        table0 = self.table.copy()
        for s, d in zip(src, dst):
            valid = 0 <= s < self.seqs and 0 <= d < self.seqs and s != d and start[d] == 0 and d not in seen and 0 <= start[s] <= self.max_pages * self.rows
            seen.add(d)
            if not valid:
                ok.append(0)
                continue
            part, whole = int(start[s]) % self.rows, int(start[s]) // self.rows
            need += part > 0
            if part and need > len(free):
                ok.append(0)
                continue
            ok.append(1)
            self.table[d, :whole] = table0[s, :whole]
            np.add.at(self.ref, table0[s, :whole], 1)
            if part:
                f = free[need - 1]
                self.table[d, whole], self.ref[f] = f, 1
                self.data[:, f, :, :part] = self.data[:, table0[s, whole], :, :part]
            self.lens[d] = start[s]
        return ok

    def grow(self, seqs, add):
        free, seen, need, ok = self.free_pages(), set(), 0, []
        for s, a in zip(seqs, add):
            valid = 0 <= s < self.seqs and s not in seen and a >= 0 and int(self.lens[s] if 0 <= s < self.seqs else 0) + int(a) <= self.max_pages * self.rows
            seen.add(s)
            if not valid:
                ok.append(0)
                continue
            n0, n1 = self.np_pages(self.lens[s]), self.np_pages(int(self.lens[s]) + int(a))
            need += n1 - n0
            if n1 > n0 and need > len(free):
                ok.append(0)
                continue
            ok.append(1)
            for i, f in enumerate(free[need - (n1 - n0):need]):
                self.table[s, n0 + i], self.ref[f] = f, 1
            self.lens[s] += a
        return ok

    def free(self, seqs):
        for s in seqs:
            if 0 <= s < self.seqs:
                n = self.np_pages(self.lens[s])
                np.add.at(self.ref, self.table[s, :n], -1)
                self.table[s, :n] = -1
                self.lens[s] = 0


def i32(*v):
    return np.array(v, np.int32)


@pytest.mark.parametrize("rows,row_vals,planes,heads", [(16, 8, 1, 1), (16, 128, 3, 2), (64, 256, 2, 4), (5, 24, 2, 3)])
def test_fork_shares_whole_pages_and_copies_the_partial_one(bk, rows, row_vals, planes, heads):
    rng = np.random.default_rng(rows)
    p = Pool(rng, planes, 24, heads, rows, row_vals, seqs=9)
    order = list(rng.permutation(24))
    for s, length in enumerate([3 * rows + 1, 2 * rows, 1, 0, rows - 1]):
        p.own(s, length, order)
    pool = p.upload()
    # shared, shared, partial twice from one parent, an empty parent, a full destination, itself, out of range, a repeated destination
    src, dst = i32(0, 1, 0, 3, 1, 5, -1, 9, 2, 0), i32(5, 6, 7, 3, 0, 5, 6, 7, 8, 8)
    ok = R.DeviceBuffer.from_numpy(np.full(10, 7, np.int32))
    ds, dd = dev(src), dev(dst)
    want = p.fork(src, dst)
    pool.fork(ds.ptr, dd.ptr, 10, ok.ptr)
    p.check("fork")
    assert ok.download(np.int32, (10,)).tolist() == want and want == [1, 1, 1, 0, 0, 0, 0, 0, 1, 0]


def test_fork_and_grow_when_pages_run_out(bk):
    rng = np.random.default_rng(3)
    p = Pool(rng, n_pages=8, seqs=8)
    p.own(0, 20, [5, 2])
    p.own(1, 32, [7, 1])
    pool = p.upload()          # four free pages: 0, 3, 4, 6
    src, dst, ok = dev(i32(0, 0, 1, 0, 0, 1)), dev(i32(2, 3, 4, 5, 6, 7)), R.DeviceBuffer(24)
    want = p.fork(i32(0, 0, 1, 0, 0, 1), i32(2, 3, 4, 5, 6, 7))
    pool.fork(src.ptr, dst.ptr, 6, ok.ptr)
    p.check("fork")
    assert want == [1] * 6 and ok.download(np.int32, (6,)).tolist() == want
    seqs, add = i32(2, 7, 3), i32(0, 1, 12)        # none is free: only what needs no page is served
    want = p.grow(seqs, add)
    a, b = dev(seqs), dev(add)
    pool.grow(a.ptr, b.ptr, 3, ok.ptr)
    p.check("grow")
    assert want == [1, 0, 1] and ok.download(np.int32, (3,)).tolist() == want
    gone = i32(3, 3, 99, -5, 2)
    g = dev(gone)
    p.free(gone)
    pool.free(g.ptr, 5)
    p.check("free")
    want = p.fork(i32(0, 0, 0), i32(2, 3, 0))      # two pages came back
    s2, d2 = dev(i32(0, 0, 0)), dev(i32(2, 3, 0))
    pool.fork(s2.ptr, d2.ptr, 3, ok.ptr)
    p.check("fork again")
    assert want == [1, 1, 0] and ok.download(np.int32, (3,)).tolist() == want


@pytest.mark.parametrize("n", [1, 33, 700, 1024])
def test_grow_gives_the_lowest_free_pages_in_list_order(bk, n):
    rng = np.random.default_rng(n)
    p = Pool(rng, planes=1, n_pages=9000, heads=1, rows=4, row_vals=8, seqs=1100, max_pages=12)
    p.ref[rng.random(9000) < 0.4] = 1     # pages that others hold
    pool = p.upload()
    seqs = rng.permutation(1100)[:n].astype(np.int32)
    if n > 2:
        seqs[2] = seqs[0]
    add = rng.integers(-1, 50, n).astype(np.int32)
    ok, a, b = R.DeviceBuffer(4 * n), dev(seqs), dev(add)
    for _ in range(2):
        want = p.grow(seqs, add)
        pool.grow(a.ptr, b.ptr, n, ok.ptr)
        p.check()
        assert ok.download(np.int32, (n,)).tolist() == want


@pytest.mark.parametrize("n_pages,used,in_place", [(1, 0, False), (1, 1, True), (24, 0, True), (24, 24, False), (24, 11, True), (1500, 700, False), (5000, 4990, True),
                                                   (2100, 3, True)])
def test_compact_moves_the_used_pages_to_the_front(bk, n_pages, used, in_place):
    rng = np.random.default_rng(n_pages + used)
    p = Pool(rng, planes=2, n_pages=n_pages, heads=1, rows=2, row_vals=8, seqs=7, max_pages=max(1, -(-used // 7)))
    held = rng.permutation(n_pages)[:used]
    p.table.reshape(-1)[rng.permutation(p.table.size)[:used]] = held
    p.ref[held] = rng.integers(1, 4, used)
    if used:
        p.table.reshape(-1)[np.nonzero(p.table.reshape(-1) < 0)[0][:1]] = n_pages + 5       # names no page
    pool = p.upload()
    to = {k: p.d[k] if in_place else R.DeviceBuffer.zeros(max(4, getattr(p, k).nbytes)) for k in ("table", "ref")}
    mp, un = R.DeviceBuffer(4 * n_pages), R.DeviceBuffer(4)
    pool.compact(to["table"].ptr, to["ref"].ptr, mp.ptr, un.ptr)
    assert R.cuSync() == 0
    place = np.full(n_pages, -1, np.int32)
    place[held] = held
    old, new = np.sort(held[held >= used]), np.array([q for q in range(used) if p.ref[q] == 0], np.int64)
    place[old] = new
    data, ref = p.data.copy(), np.zeros_like(p.ref)
    data[:, new] = p.data[:, old]
    ref[place[held]] = p.ref[held]
    inside = (p.table >= 0) & (p.table < n_pages)
    table = np.where(inside, place[np.where(inside, p.table, 0)], -1)
    assert un.download(np.int32, (1,))[0] == used
    assert np.array_equal(mp.download(np.int32, (n_pages,)), place)
    assert np.array_equal(to["ref"].download(np.int32, (n_pages,)), ref)
    assert np.array_equal(to["table"].download(np.int32, p.table.shape), table)
    assert np.array_equal(p.d["data"].download(np.uint16, p.shape), data)


@pytest.mark.parametrize("rows,row_vals", [(2, 8), (16, 256), (64, 128)])
def test_copy_between_pools_and_within_one(bk, rows, row_vals):
    rng = np.random.default_rng(rows)
    a, b = Pool(rng, 3, 20, 2, rows, row_vals), Pool(rng, 3, 31, 2, rows, row_vals)
    pa, pb = a.upload(), b.upload()
    src, dst = i32(19, 0, 7, 25, 3, -1), i32(30, 2, 0, 1, 31, 4)     # the last three name a page that is not there
    ds, dd = dev(src), dev(dst)
    pa.copy(pb, ds.ptr, dd.ptr, 6)
    b.data[:, [30, 2, 0]] = a.data[:, [19, 0, 7]]
    b.check("between")
    s2, d2 = dev(i32(1, 2)), dev(i32(3, 4))
    pa.copy(pa, s2.ptr, d2.ptr, 2)
    a.data[:, [3, 4]] = a.data[:, [1, 2]]
    a.check("within")
    pa.copy(pb, 0, 0, 0)           # an empty list does nothing
    b.check("nothing")


def test_copy_of_planes_apart_by_more_than_32_bits(bk):
    """Planes 5 GB apart in one allocation: offsets pass 32 bits."""
    rng = np.random.default_rng(8)
    planes, n_pages, page = 2, 4, 2 * 16 * 16
    gap = 5 << 30
    big = R.DeviceBuffer(gap + n_pages * page)
    host = rng.integers(0, 256, (planes, n_pages, page)).astype(np.uint8)
    for i in range(planes):
        R.cuHtoD(big.ptr + i * gap, host[i])
    meta = R.DeviceBuffer.zeros(1024)
    nb = PG.scratch_bytes(n_pages, 1)
    scratch = R.DeviceBuffer(nb)
    pool = PG.PagePool(base=big.ptr, plane_bytes=gap, n_planes=planes, n_pages=n_pages, heads=2, page_rows=16, row_bytes=16, n_seqs=1, max_pages=1,
                       ref=meta.ptr, table=meta.ptr + 256, lens=meta.ptr + 512, scratch=scratch.ptr, scratch_bytes=nb)
    s, d = dev(i32(1)), dev(i32(3))
    pool.copy(pool, s.ptr, d.ptr, 1)
    host[:, 3] = host[:, 1]
    got = np.empty((planes, n_pages, page), np.uint8)
    for i in range(planes):
        R.cuDtoH(got[i], big.ptr + i * gap)
    assert np.array_equal(got, host)
    big.free()


def test_pages_refusals(bk):
    p = Pool(np.random.default_rng(1))
    pool = p.upload()
    one = dev(i32(0, 1, 2, 3))
    lib = R.cu()

    def refused(call, **change):
        d = R.bkPages.from_buffer_copy(pool.desc)
        for k, v in change.items():
            setattr(d, k, v)
        assert call(d) == R.BK_ERR_ARG, (change, R.last_error())
        assert R.last_error()

    free = lambda d: lib.bkPagesFree(C.byref(d), one.ptr, 1)  # noqa: E731
    for change in ({"base": 0}, {"base": pool.desc.base + 8}, {"n_planes": 0}, {"n_pages": 0}, {"row_bytes": 8}, {"row_bytes": 0}, {"heads": -1}, {"page_rows": 0},
                   {"plane_bytes": pool.desc.plane_bytes - 16}, {"plane_bytes": pool.desc.plane_bytes + 8}, {"ref": 0}, {"table": 0}, {"lens": 0}, {"lens": pool.desc.lens + 2},
                   {"scratch": 0}, {"scratch_bytes": 16}, {"max_pages": 0}, {"n_seqs": 0}, {"max_pages": 1 << 30}, {"heads": 1 << 20, "page_rows": 1 << 20}):
        refused(free, **change)
    same = {}
    refused(lambda d: lib.bkPagesFree(C.byref(d), one.ptr, 1025), **same)
    refused(lambda d: lib.bkPagesFree(C.byref(d), 0, 1), **same)
    refused(lambda d: lib.bkPagesFork(C.byref(d), one.ptr, 0, 1, 0), **same)
    refused(lambda d: lib.bkPagesGrow(C.byref(d), one.ptr, one.ptr, -1, 0), **same)
    refused(lambda d: lib.bkPagesGrow(C.byref(d), one.ptr, one.ptr, 1, 3), **same)
    refused(lambda d: lib.bkPagesCompact(C.byref(d), one.ptr, one.ptr, 0, one.ptr), **same)
    refused(lambda d: lib.bkPagesCopy(C.byref(d), C.byref(pool.desc), one.ptr, one.ptr, 1), n_planes=1)
    assert lib.bkPagesFree(None, one.ptr, 1) == R.BK_ERR_ARG
    p.check("nothing changed")


# ---- attention over pages ---------------------------------------------------------------

class Case:
    """A pool of keys and values whose rows past every sequence's end are NaN, and the attention over it in 64 bits."""

    def __init__(self, seed, B, T, prefix, own_rows, new=None, Hq=4, Hkv=1, HD=128, rows=16, fused=True, gate=True, std=1.0, scale=None, max_len=None, rot=32):
        rng = np.random.default_rng(seed)
        self.B, self.T, self.P, self.Hq, self.Hkv, self.HD, self.rows, self.fused, self.rot = B, T, prefix, Hq, Hkv, HD, rows, fused, rot
        self.new = np.array([T] * B if new is None else new, np.int32)
        self.lens = np.array([prefix + n for n in own_rows], np.int32)
        shared = prefix // rows
        tail = [max(0, -(-int(n) // rows) - shared) for n in self.lens]
        self.n_pages = shared + sum(tail) + 3
        order = list(rng.permutation(self.n_pages))
        self.max_pages = max(1, shared + max(tail))
        self.max_len = self.max_pages * rows if max_len is None else max_len
        self.table = np.full((B, self.max_pages), -1, np.int32)
        common = [order.pop() for _ in range(shared)]
        self.kp = np.full((self.n_pages, Hkv, rows, HD), 0x7FC0, np.uint16)
        self.vp = self.kp.copy()
        self.kp[common], self.vp[common] = rnd(rng, shared, Hkv, rows, HD, std=std), rnd(rng, shared, Hkv, rows, HD)
        pre = rnd(rng, 2, Hkv, rows, HD, std=std)         # rows of the page that the prefix ends in
        for b in range(B):
            mine = [order.pop() for _ in range(tail[b])]
            self.table[b, :shared + tail[b]] = common + mine
            for j in range(shared * rows, int(self.lens[b])):
                at = self.table[b, j // rows], slice(None), j % rows
                self.kp[at] = pre[0][:, j % rows] if j < prefix else rnd(rng, Hkv, HD, std=std)
                self.vp[at] = pre[1][:, j % rows] if j < prefix else rnd(rng, Hkv, HD)
        n = T * B
        self.q, self.g = rnd(rng, n, Hq, HD), rnd(rng, n, Hq, HD) if gate else None
        self.k, self.v = rnd(rng, n, Hkv, HD), rnd(rng, n, Hkv, HD)
        self.qw, self.kw = rnd(rng, HD, std=0.1), rnd(rng, HD, std=0.1)
        ang = np.outer(np.arange(max(self.max_len, 1)), 1e4 ** (-np.arange(rot) / rot))
        self.cos, self.sin = np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)
        self.scale = np.float32(1 / math.sqrt(HD) if scale is None else scale)

    def positions(self):
        """row of (t, b), -1 where it is not there"""
        pos = np.full((self.T, self.B), -1)
        for b in range(self.B):
            n = min(int(self.new[b]), self.T)
            for t in range(max(n, 0)):
                at = int(self.lens[b]) - n + t
                pos[t, b] = at if 0 <= at < min(self.max_len, self.max_pages * self.rows) else -1
        return pos

    def turned(self, x, w, at):
        y = val(x)
        y = y / np.sqrt((y ** 2).mean(-1, keepdims=True) + 1e-6) * (1 + val(w))
        c, s, r = self.cos[at].astype(np.float64), self.sin[at].astype(np.float64), self.rot
        out = y.copy()
        out[..., :r], out[..., r:2 * r] = y[..., :r] * c - y[..., r:2 * r] * s, y[..., r:2 * r] * c + y[..., :r] * s
        return out

    def want(self):
        pos, kp, vp = self.positions(), self.kp.copy(), self.vp.copy()
        G, out = self.Hq // self.Hkv, np.zeros((self.T * self.B, self.Hq, self.HD))
        for b in range(self.B):
            for t in range(self.T):
                at, e = pos[t, b], t * self.B + b
                if at >= 0:
                    page = self.table[b, at // self.rows], slice(None), at % self.rows
                    kp[page] = bf16(self.turned(self.k[e], self.kw, at)) if self.fused else self.k[e]
                    vp[page] = self.v[e]
        for b in range(self.B):
            for t in range(self.T):
                at, e = pos[t, b], t * self.B + b
                if at < 0:
                    continue
                j = np.arange(at + 1)
                K, V = val(kp[self.table[b, j // self.rows], :, j % self.rows]), val(vp[self.table[b, j // self.rows], :, j % self.rows])
                q = val(bf16(self.turned(self.q[e], self.qw, at))) if self.fused else val(self.q[e])
                for h in range(self.Hq):
                    s = K[:, h // G] @ q[h] * float(self.scale)
                    w = np.exp(s - s.max())
                    out[e, h] = w @ V[:, h // G] / w.sum()
                if self.g is not None:
                    out[e] /= 1 + np.exp(-val(self.g[e]))
        return out, kp, vp

    def args(self, **change):
        n, self.keep = self.T * self.B, {}
        qg = np.concatenate([self.q, self.g], -1) if self.fused else self.q
        for name, a in (("qg", qg), ("k", self.k), ("v", self.v), ("qw", self.qw), ("kw", self.kw), ("cos", self.cos), ("sin", self.sin), ("kp", self.kp), ("vp", self.vp),
                        ("table", self.table), ("lens", self.lens), ("new", self.new), ("g", self.g)):
            if a is not None:
                self.keep[name] = dev(a)
        d = {k: b.ptr for k, b in self.keep.items()}
        nb = ops.paged_attn_scratch_bytes(self.B, self.T, self.Hq, self.Hkv, self.HD, self.P)
        self.scratch = R.DeviceBuffer.from_numpy(np.full(nb // 4 + 1, 0x7FC00000, np.uint32))      # (NaN: nothing of it is read before it is written)
        self.out = R.DeviceBuffer.from_numpy(np.full((n, self.Hq * self.HD), 0x7FC0, np.uint16))
        kw = dict(qg=d["qg"], k=d["k"], v=d["v"], k_pages=d["kp"], v_pages=d["vp"], table=d["table"], lens=d["lens"], n_new=d["new"], out=self.out.ptr,
                  scratch=self.scratch.ptr, scratch_bytes=nb, B=self.B, T=self.T, Hq=self.Hq, Hkv=self.Hkv, HD=self.HD, n_pages=self.n_pages,
                  page_rows=self.rows, max_pages=self.max_pages, prefix_rows=self.P, max_len=self.max_len, scale=self.scale, eps=1e-6, fused_norm_rope=int(self.fused))
        if self.fused:
            kw.update(q_norm_w=d["qw"], k_norm_w=d["kw"], cos_t=d["cos"], sin_t=d["sin"], rot_half=self.rot)
        elif self.g is not None:
            kw.update(gate=d["g"])
        kw.update(change)
        return ops.paged_attn_args(**kw)

    def check(self, times=2):
        a = self.args()
        want, kp, vp = self.want()
        vmax = np.nanmax(np.abs(np.where(np.isfinite(val(vp)), val(vp), 0)))
        first = None
        for _ in range(times):
            ops.paged_attn(a)
            assert R.cuSync() == 0, R.last_error()
            bits = self.out.download(np.uint16, (self.T * self.B, self.Hq, self.HD))
            got = val(bits)
            assert np.isfinite(got).all()
            tol = 2.0 ** -8 * np.abs(want) + (2.0 ** -7 if self.fused else 2.0 ** -13) * vmax
            bad = np.abs(got - want) > tol
            assert not bad.any(), (np.argwhere(bad)[:5], np.abs(got - want).max(), got[bad][:5], want[bad][:5])
            absent = (self.positions() < 0).reshape(-1)
            assert not bits[absent].any()
            assert first is None or np.array_equal(first, bits)       # the same call gives the same bits
            first = bits
        k, v = self.keep["kp"].download(np.uint16, self.kp.shape), self.keep["vp"].download(np.uint16, self.vp.shape)
        assert np.array_equal(v, vp)
        changed = kp != self.kp
        assert np.array_equal(k[~changed], kp[~changed])
        assert (np.abs(val(k[changed]) - val(kp[changed])) <= 2.0 ** -7 * np.abs(val(kp[changed])) + 2.0 ** -16).all()


@pytest.mark.parametrize("HD", [128, 256])
@pytest.mark.parametrize("own_rows", [[1], [2], [15], [16], [17], [63], [64], [65], [200]])
def test_attention_of_one_sequence(bk, HD, own_rows):
    Case(own_rows[0], 1, 1, 0, own_rows, HD=HD, Hq=8, Hkv=1).check()


@pytest.mark.parametrize("fused", [True, False])
@pytest.mark.parametrize("Hq,Hkv,HD,rows", [(16, 2, 256, 64), (24, 4, 256, 32), (4, 1, 256, 16), (3, 3, 128, 128), (16, 1, 128, 16), (14, 2, 128, 1024), (5, 1, 256, 256)])
def test_attention_behind_a_prefix_by_heads_and_page_sizes(bk, fused, Hq, Hkv, HD, rows):
    Case(Hq + rows, 5, 1, 150, [1, 40, 77, 3, 130], Hq=Hq, Hkv=Hkv, HD=HD, rows=rows, fused=fused).check()


@pytest.mark.parametrize("prefix", [1, 15, 16, 17, 48, 64, 80, 127, 128, 1000])
def test_attention_prefixes_that_end_anywhere(bk, prefix):
    Case(prefix, 3, 1, prefix, [1, 30, 70], Hq=8, Hkv=2, HD=128).check()


@pytest.mark.parametrize("T,new", [(2, [2, 1, 2]), (16, [16, 1, 7]), (33, [33, 0, 20]), (64, [64, 63, 1])])
@pytest.mark.parametrize("prefix", [0, 70])
def test_attention_of_several_new_tokens_is_causal(bk, T, new, prefix):
    Case(T, 3, T, prefix, [max(n, 1) + 9 * i for i, n in enumerate(new)], new=new, Hq=6, Hkv=1, HD=128).check()


def test_attention_of_many_rows_and_row_tiles(bk):
    Case(5, 40, 1, 200, [1 + 5 * (i % 9) for i in range(40)], Hq=8, Hkv=1, HD=256).check()            # 320 rows behind the prefix: three tiles, the last partial
    Case(6, 2, 40, 130, [40, 95], Hq=8, Hkv=1, HD=128).check()                                         # 320 rows of one sequence


def test_attention_of_more_jobs_than_shared_memory_plans(bk):
    Case(61, 300, 1, 70, [1 + 7 * i % 40 for i in range(300)], Hq=4, Hkv=4, HD=128).check()            # 1,204 jobs
    Case(62, 130, 1, 0, [i % 3 for i in range(130)], new=[min(1, i % 3) for i in range(130)], Hq=8, Hkv=8, HD=128).check()   # 1,040, a third of them empty


def test_attention_of_a_long_piece_of_prompt(bk):
    """One sequence, 150 new tokens of 8 heads: ten row tiles, with and without common rows, in one line and cut at the same keys."""
    Case(63, 1, 150, 0, [600], Hq=8, Hkv=1, HD=128).check()
    Case(64, 1, 150, 2000, [150], Hq=8, Hkv=1, HD=128, rows=64).check()
    Case(65, 2, 70, 1300, [70, 75], new=[70, 31], Hq=16, Hkv=2, HD=256, rows=128).check()


def test_attention_over_pages_beyond_32_bits(bk):
    """Pools of 5 GB of keys and of values: the pages in use lie at their end."""
    c = Case(66, 2, 1, 80, [40, 100], Hq=8, Hkv=2, HD=256, rows=64)
    page = 2 * 64 * 256 * 2
    far = (5 << 30) // page
    shift = far - c.n_pages
    want, kp, vp = c.want()
    big = [R.DeviceBuffer(5 << 30) for _ in range(2)]
    for b, host in zip(big, (c.kp, c.vp)):
        R.cuHtoD(b.ptr + shift * page, host)
    table = dev(np.where(c.table >= 0, c.table + shift, -1).astype(np.int32))
    ops.paged_attn(c.args(k_pages=big[0].ptr, v_pages=big[1].ptr, table=table.ptr, n_pages=far))
    assert R.cuSync() == 0, R.last_error()
    got = val(c.out.download(np.uint16, (2, c.Hq, 256)))
    vmax = np.abs(val(vp)[np.isfinite(val(vp))]).max()
    assert (np.abs(got - want) <= 2.0 ** -8 * np.abs(want) + 2.0 ** -7 * vmax).all()
    back = np.empty_like(c.vp)
    R.cuDtoH(back, big[1].ptr + shift * page)
    assert np.array_equal(back, vp)
    for b in big:
        b.free()


def test_attention_where_nothing_is_there(bk):
    Case(1, 3, 1, 0, [0, 5, 0], new=[0, 1, 0], HD=128).check()
    Case(2, 2, 1, 0, [0, 0], new=[0, 0], HD=256).check()                        # no work at all
    Case(3, 2, 4, 32, [4, 2], new=[9, -3], HD=128).check()                      # counts outside 0..T
    Case(4, 2, 1, 0, [40, 20], HD=128, max_len=30).check()                      # a sequence longer than the call allows: its token is not there
    c = Case(5, 3, 1, 64, [10, 0, 3], HD=128)                                   # sequences shorter than the prefix see only their own part of it
    c.lens = np.array([74, 20, 67], np.int32)
    c.check()


@pytest.mark.parametrize("HD,rows", [(128, 16), (256, 64)])
def test_attention_keeps_what_is_not_finite_to_the_tokens_that_see_it(bk, HD, rows):
    """Infinities and NaN in keys and values of later tokens, and of common rows behind a short sequence's end, do not reach a token; those it
    sees make its dims infinite or NaN."""
    T = 12
    c = Case(51, 2, T, 40, [30, 12], HD=HD, Hq=6, Hkv=1, rows=rows, fused=False, gate=False)
    c.v[7 * 2 + 0, 0, 3], c.v[7 * 2 + 0, 0, HD - 1], c.v[11 * 2 + 0, 0, 5], c.k[9 * 2 + 1, 0, 1] = 0x7F80, 0xFF80, 0x7FC0, 0x7FC0
    with np.errstate(invalid="ignore"):
        want, kp, vp = c.want()
    ops.paged_attn(c.args())
    assert R.cuSync() == 0, R.last_error()
    got = val(c.out.download(np.uint16, (T * 2, c.Hq, HD))).reshape(T, 2, c.Hq, HD)
    want = want.reshape(T, 2, c.Hq, HD)
    odd = np.zeros(want.shape, bool)
    odd[7:, 0, :, 3] = odd[7:, 0, :, HD - 1] = True
    odd[11:, 0, :, 5] = True
    odd[9:, 1] = True                                            # a NaN key: every later token of that sequence, all dims
    assert np.array_equal(~np.isfinite(want), odd)               # (the plain form says so too)
    assert np.array_equal(~np.isfinite(got), odd)
    assert np.array_equal(np.isnan(got[odd]), np.isnan(want[odd])) and (got[7:, 0, :, 3] == np.inf).all() and (got[7:, 0, :, HD - 1] == -np.inf).all()
    vmax = np.abs(val(vp)[np.isfinite(val(vp))]).max()
    assert (np.abs(got[~odd] - want[~odd]) <= 2.0 ** -8 * np.abs(want[~odd]) + 2.0 ** -13 * vmax).all()
    # common rows behind the end of a short sequence
    c = Case(52, 3, 1, 128, [10, 0, 3], HD=HD, fused=False, gate=False, rows=rows)
    c.lens = np.array([138, 50, 131], np.int32)
    page, row = c.table[0, 100 // rows], 100 % rows
    c.vp[page, 0, row, 2] = 0x7FC0
    with np.errstate(invalid="ignore"):
        want, kp, vp = c.want()
    ops.paged_attn(c.args())
    assert R.cuSync() == 0, R.last_error()
    got = val(c.out.download(np.uint16, (3, c.Hq, HD)))
    odd = np.zeros(want.shape, bool)
    odd[[0, 2], :, 2] = True
    assert np.array_equal(~np.isfinite(want), odd) and np.array_equal(~np.isfinite(got), odd)
    assert (np.abs(got[~odd] - want[~odd]) <= 2.0 ** -8 * np.abs(want[~odd]) + 2.0 ** -13 * np.abs(val(vp)[np.isfinite(val(vp))]).max()).all()


def test_attention_over_scores_of_all_sizes(bk):
    """Large scores (softmax of one row), a running maximum that rises from tile to tile, equal scores."""
    Case(11, 2, 1, 128, [100, 300], HD=128, std=6.0, fused=False).check()
    c = Case(12, 1, 1, 0, [400], HD=128, fused=False, gate=False)
    j = np.arange(400)
    c.kp[c.table[0, j // 16], :, j % 16] = bf16(np.broadcast_to((j * 0.05)[:, None, None], (400, 1, 128)))
    c.q[:] = bf16(np.ones(c.q.shape))
    c.check()
    c = Case(13, 1, 1, 0, [300], HD=256, fused=False, gate=False)
    c.q[:] = 0
    c.check()
    Case(14, 2, 1, 64, [70, 5], HD=128, scale=3e-3).check()


def test_attention_ready_queries_without_an_append(bk):
    c = Case(21, 2, 1, 64, [30, 9], HD=128, fused=False, gate=False)
    pos = c.positions()
    for b in range(2):
        at = pos[0, b]
        c.kp[c.table[b, at // 16], :, at % 16], c.vp[c.table[b, at // 16], :, at % 16] = c.k[b], c.v[b]
    want, kp, vp = c.want()
    ops.paged_attn(c.args(k=0, v=0, n_new=0))
    assert R.cuSync() == 0
    got = val(c.out.download(np.uint16, (2, c.Hq, c.HD)))
    assert (np.abs(got - want) <= 2.0 ** -8 * np.abs(want) + 2.0 ** -13 * np.nanmax(np.abs(np.where(np.isfinite(val(vp)), val(vp), 0)))).all()
    assert np.array_equal(c.keep["kp"].download(np.uint16, kp.shape), c.kp)


def test_attention_is_the_same_whatever_is_shared(bk):
    """Sharing is only a way of reading: without it the result is the same up to the order of sums."""
    a = Case(31, 6, 1, 500, [3, 50, 80, 1, 20, 64], Hq=16, Hkv=2, HD=256, rows=32)
    got = []
    for P in (500, 0, 33):
        ops.paged_attn(a.args(prefix_rows=P))
        assert R.cuSync() == 0
        got.append(val(a.out.download(np.uint16, (6, 16, 256))))
    for g in got[1:]:
        assert (np.abs(g - got[0]) <= 2.0 ** -7 * np.abs(got[0]) + 2.0 ** -12 * 5).all()


def test_attention_refusals(bk):
    c = Case(41, 2, 1, 32, [5, 9], HD=128)
    good = c.args()
    lib = R.cu()
    for change in ({"HD": 64}, {"Hq": 5, "Hkv": 2}, {"Hq": 17, "Hkv": 1}, {"B": 0}, {"T": 0}, {"page_rows": 24}, {"page_rows": 8}, {"page_rows": 2048}, {"n_pages": 0}, {"max_pages": 0},
                   {"n_pages": 1 << 28}, {"max_len": 0}, {"prefix_rows": -1}, {"prefix_rows": 10 ** 6}, {"qg": 0}, {"k": 0}, {"v": 0}, {"table": 0}, {"lens": 0}, {"out": 0}, {"scratch": 0},
                   {"scratch_bytes": 64}, {"qg": good.qg + 2}, {"out": good.out + 8}, {"lens": good.lens + 1}, {"q_norm_w": 0}, {"cos_t": 0}, {"rot_half": 0}, {"rot_half": 65},
                   {"gate": good.qg}, {"scale": 0.0}, {"scale": -1.0}, {"scale": float("inf")}, {"scale": float("nan")}, {"B": 1 << 23}):
        a = R.bkPagedAttnArgs.from_buffer_copy(good)
        for k, v in change.items():
            setattr(a, k, v)
        assert lib.bkPagedAttn(C.byref(a)) == R.BK_ERR_ARG and R.last_error(), change
    assert lib.bkPagedAttn(None) == R.BK_ERR_ARG
    with pytest.raises(TypeError):
        ops.paged_attn_args(heads=3)
    assert R.cuSync() == 0


# ---- adapters ----------------------------------------------------------------------

def lora_case(seed, B, K, rows, rank, n_adapters, ids, f32, with_base=True, with_scale=True, pad=0):
    rng = np.random.default_rng(seed)
    x, ids = rnd(rng, B, K), np.array(ids, np.int32)
    scale = rng.uniform(0.5, 2, n_adapters).astype(np.float32) if with_scale else None
    segs, keep, want = [], [], []
    for n in rows:
        A, M = rnd(rng, n_adapters, rank, K, std=0.1), rnd(rng, n_adapters, n, rank, std=0.3)
        ld = n + 2 * pad
        base = rng.normal(0, 1, (B, ld)).astype(np.float32)
        base = base if f32 else bf16(base)
        y = (base.astype(np.float64) if f32 else val(base)) if with_base else np.zeros((B, ld))
        mag = np.abs(y)
        for b in range(B):
            a = ids[b]
            if 0 <= a < n_adapters:
                sc = 1.0 if scale is None else float(scale[a])
                y[b, pad:pad + n] += sc * (val(M[a]) @ (val(A[a]) @ val(x[b])))
                mag[b, pad:pad + n] += sc * (np.abs(val(M[a])) @ (np.abs(val(A[a])) @ np.abs(val(x[b]))))
        fill = np.full((B, ld), np.nan, np.float32)
        out, d = dev(fill if f32 else bf16(np.full((B, ld), 1.5))), [dev(A), dev(M), dev(base)]
        keep.append((d, out, ld, n))
        want.append((y, mag))
        segs.append(ops.lora_seg(A=d[0].ptr, Bm=d[1].ptr, n_rows=n, base=d[2].ptr if with_base else 0, out=out.ptr, bf16=not f32, ld_out=ld, col_off=pad))
    nb = ops.lora_scratch_bytes(K, B, rank, len(rows))
    dx, di, ds, scratch = dev(x), dev(ids), dev(scale) if with_scale else None, R.DeviceBuffer(nb)
    args = ops.lora_args(x=dx.ptr, K=K, B=B, rank=rank, n_adapters=n_adapters, ids=di.ptr, segs=segs, scratch=scratch.ptr, scratch_bytes=nb, scale=ds.ptr if ds else 0)
    return args, keep, want, (dx, di, ds, scratch)


@pytest.mark.parametrize("B,K,rows,rank,n_adapters,ids", [
    (1, 8, [1], 8, 1, [0]),
    (1, 2048, [8192], 8, 3, [2]),
    (2, 264, [300, 7], 16, 2, [1, 1]),
    (5, 1000, [257, 64, 1], 24, 4, [3, -1, 0, 3, 9]),
    (9, 512, [130], 128, 2, [0] * 9),
    (33, 768, [96, 520], 40, 7, [i % 9 - 1 for i in range(33)]),
    (64, 256, [256, 255, 64, 65], 64, 64, list(range(64))),
    (64, 5120, [520], 16, 1, [0] * 64),
    (3, 256, [40], 8, 2, [-1, -7, 2]),
])
@pytest.mark.parametrize("f32", [True, False])
def test_adapters_of_many_requests(bk, B, K, rows, rank, n_adapters, ids, f32):
    args, keep, want, hold = lora_case(B + K, B, K, rows, rank, n_adapters, ids, f32)
    first = None
    for _ in range(2):
        ops.lora(args)
        assert R.cuSync() == 0, R.last_error()
        bits = []
        for (d, out, ld, n), (y, mag) in zip(keep, want):
            raw = out.download(np.uint32 if f32 else np.uint16, (B, ld))
            got = raw.view(np.float32).astype(np.float64) if f32 else val(raw)
            tol = (K + rank + 4) * 2.0 ** -24 * mag + (0 if f32 else 2.0 ** -8 * np.abs(y))
            assert (np.abs(got - y) <= tol).all(), np.abs(got - y).max()
            bits.append(raw)
        assert first is None or all(np.array_equal(a, b) for a, b in zip(first, bits))
        first = bits


@pytest.mark.parametrize("rank", [8, 16, 24, 32, 56, 64, 80, 96, 128])
@pytest.mark.parametrize("B,n_adapters,ids", [
    (5, 9, [7, 2, 7, -1, 7]),                    # more adapters than requests: three columns, one, none
    (4, 4, [3, 1, 3, 1]),                        # two columns each; two adapters without any
    (10, 2, [1, -1, 1, 1, 0, 1, 1, 2, 1, 1]),    # seven columns and one; two without
])
def test_adapters_of_every_rank(bk, rank, B, n_adapters, ids):
    for rows in ([2500], [31, 257]):             # tiles that end inside
        args, keep, want, hold = lora_case(rank + B, B, 1032, rows, rank, n_adapters, ids, True)
        ops.lora(args)
        assert R.cuSync() == 0, R.last_error()
        for (d, out, ld, n), (y, mag) in zip(keep, want):
            got = out.download(np.float32, (B, ld)).astype(np.float64)
            assert (np.abs(got - y) <= (1032 + rank + 4) * 2.0 ** -24 * mag).all()


@pytest.mark.parametrize("rank,shared", [(8, 1), (32, 1), (8, 4), (64, 2), (128, 3)])
def test_adapters_of_many_rows(bk, rank, shared):
    """So many rows and adapters that a CTA goes through several tiles; every adapter has `shared` columns."""
    B = 40
    args, keep, want, hold = lora_case(rank, B, 64, [9001 if rank > 32 else 17377], rank, B, [-1 if b == 7 else b // shared for b in range(B)], True)
    ops.lora(args)
    assert R.cuSync() == 0, R.last_error()
    for (d, out, ld, n), (y, mag) in zip(keep, want):
        got = out.download(np.float32, (B, ld)).astype(np.float64)
        assert (np.abs(got - y) <= (64 + rank + 4) * 2.0 ** -24 * mag).all()


def test_adapters_without_base_or_scale_in_place_and_in_columns(bk):
    for kw in ({"with_base": False}, {"with_scale": False}, {"pad": 5}):
        args, keep, want, hold = lora_case(7, 4, 320, [100, 30], 16, 3, [0, 2, -1, 0], True, **kw)
        pad = kw.get("pad", 0)
        ops.lora(args)
        assert R.cuSync() == 0
        for (d, out, ld, n), (y, mag) in zip(keep, want):
            got = out.download(np.float32, (4, ld)).astype(np.float64)
            cols = slice(pad, pad + n)
            assert (np.abs(got - y)[:, cols] <= (340 * 2.0 ** -24 * mag)[:, cols]).all()
            assert np.isnan(got[:, :pad]).all() and np.isnan(got[:, pad + n:]).all()      # nothing beside the segment's columns
    args, keep, want, hold = lora_case(8, 4, 320, [100], 16, 3, [0, 2, -1, 0], True)
    args.segs[0].out = args.segs[0].base
    ops.lora(args)
    assert R.cuSync() == 0
    got = keep[0][0][2].download(np.float32, (4, 100)).astype(np.float64)
    assert (np.abs(got - want[0][0]) <= 340 * 2.0 ** -24 * want[0][1]).all()


def test_adapters_of_segments_of_both_types(bk):
    a32, k32, w32, hold32 = lora_case(11, 7, 512, [70, 300], 24, 3, [0, 2, -1, 0, 1, 2, 2], True)
    a16, k16, w16, hold16 = lora_case(11, 7, 512, [70, 300], 24, 3, [0, 2, -1, 0, 1, 2, 2], False)
    args = R.bkLoraArgs.from_buffer_copy(a32)
    args.n_segs = 4
    for i, s in enumerate((a16.segs[0], a32.segs[0], a16.segs[1], a32.segs[1])):
        args.segs[i] = s
    args.x = a16.x                     # (the same draw)
    nb = ops.lora_scratch_bytes(512, 7, 24, 4)
    scratch = R.DeviceBuffer(nb)
    args.scratch, args.scratch_bytes = scratch.ptr, nb
    ops.lora(args)
    assert R.cuSync() == 0
    for keep, want, f32 in ((k16, w16, False), (k32, w32, True)):
        for (d, out, ld, n), (y, mag) in zip(keep, want):
            raw = out.download(np.uint32 if f32 else np.uint16, (7, ld))
            got = raw.view(np.float32).astype(np.float64) if f32 else val(raw)
            assert (np.abs(got - y) <= 540 * 2.0 ** -24 * mag + (0 if f32 else 2.0 ** -8 * np.abs(y))).all()


def test_adapters_keep_infinities_to_their_own_request(bk):
    """A request whose x holds inf or NaN does not reach the others, nor does an adapter that nobody has."""
    args, keep, want, (dx, di, ds, scratch) = lora_case(9, 4, 256, [64], 8, 3, [0, 0, 1, -1], True)
    x = dx.download(np.uint16, (4, 256))
    x[1, 5], x[3, 0] = 0x7F80, 0x7FC0
    dx.upload(x)
    A = keep[0][0][0].download(np.uint16, (3, 8, 256))
    A[2] = 0x7FC0
    keep[0][0][0].upload(A)
    ops.lora(args)
    assert R.cuSync() == 0
    got = keep[0][1].download(np.float32, (4, 64)).astype(np.float64)
    assert not np.isfinite(got[1]).all()
    for b in (0, 2, 3):
        assert (np.abs(got[b] - want[0][0][b]) <= 270 * 2.0 ** -24 * want[0][1][b]).all()


def test_adapters_refusals(bk):
    args, keep, want, hold = lora_case(10, 2, 256, [64], 8, 3, [0, 1], True)
    lib = R.cu()
    for change in ({"K": 0}, {"K": 12}, {"B": 0}, {"B": 65}, {"n_segs": 0}, {"n_segs": 5}, {"rank": 0}, {"rank": 12}, {"rank": 136}, {"n_adapters": 0}, {"x": 0}, {"x": args.x + 2}, {"ids": 0},
                   {"ids": args.ids + 1}, {"scratch": 0}, {"scratch_bytes": 8}):
        a = R.bkLoraArgs.from_buffer_copy(args)
        for k, v in change.items():
            setattr(a, k, v)
        assert lib.bkLora(C.byref(a)) == R.BK_ERR_ARG and R.last_error(), change
    for change in ({"A": 0}, {"Bm": 0}, {"out": 0}, {"A": args.segs[0].A + 8}, {"n_rows": 0}, {"dtype": 2}, {"ld_out": 63}, {"col_off": -1}, {"col_off": 1}, {"base": args.segs[0].base + 1}):
        a = R.bkLoraArgs.from_buffer_copy(args)
        for k, v in change.items():
            setattr(a.segs[0], k, v)
        assert lib.bkLora(C.byref(a)) == R.BK_ERR_ARG and R.last_error(), change
    assert lib.bkLora(None) == R.BK_ERR_ARG
    with pytest.raises(ValueError):
        ops.lora_args(x=1, K=8, B=1, rank=8, n_adapters=1, ids=1, segs=[], scratch=1, scratch_bytes=1)
    assert R.cuSync() == 0


# ---- all of it together ------------------------------------------------------------------

def test_requests_behind_one_prompt(bk):
    """The example layer: prompt, forks, steps with adapters, dropped requests, compaction.  Sharing changes only the order of sums; compaction
    changes nothing; and a request's attention is what bkAttnDecode gives over a contiguous cache of the same rows (it rounds q
    and k after the norm too: 2^-6 of the largest value)."""
    from bunker_b200 import shared_prompt as S
    from bunker_b200.model import CONFIG_TINY as cfg
    w, lora = S.random_layer(cfg, seed=3)
    n, rows, steps = 5, 75, 3
    rng = np.random.default_rng(4)
    x = dev(rnd(rng, rows, cfg.hidden))
    xs = [dev(rnd(rng, n, cfg.hidden)) for _ in range(steps)]
    adapters = [0, -1, 2, 1, 0]
    runs = []
    for share in (True, False):
        s = S.SharedPrompt(cfg, w, lora, n, rows + steps + 5, n_pages=30)
        s.prompt(x.ptr, rows)
        s.fork(range(n))
        outs = []
        for t in range(steps):
            if t == 2:
                s.drop([1, 3])
                if share:
                    s.compact()
            s.step(xs[t].ptr, adapters, share)
            assert R.cuSync() == 0, R.last_error()
            outs.append(val(s.out.download(np.uint16, (n, cfg.hidden))))
            att = val(s.att.download(np.uint16, (n, cfg.attn_q_heads * cfg.head_dim)))
            assert (s.ok.download(np.int32, (n,)) == 1).all()
        runs.append(outs)
        assert not att[[1, 3]].any() and att[[0, 2, 4]].any()      # dropped requests attend to nothing
        assert s.lens.download(np.int32, (n + 1,)).tolist() == [rows, rows + 3, 0, rows + 3, 0, rows + 3]
        if share:
            # 5 pages of the prompt; of three requests the copied page and, for one of 3 rows more than 75, nothing else
            assert s.used.download(np.int32, (1,))[0] == 5 + 3 and (np.sort(np.nonzero(s.ref.download(np.int32, (30,)))[0]) == np.arange(8)).all()
    for a, b in zip(*runs):
        assert (np.abs(a - b) <= 2.0 ** -6 * np.abs(b).max()).all()

    # request 2 over a contiguous cache: the rows that the pages hold, the last step's q, k, v
    hd, Hq, Hkv, last = cfg.head_dim, cfg.attn_q_heads, cfg.attn_kv_heads, rows + steps - 1
    table = s.table.download(np.int32, (n + 1, s.max_pages))[3]
    planes = [s.data.download(np.uint16, (2, 30, Hkv, 16, hd))[i][table[:-(-(last + 1) // 16)]].transpose(1, 0, 2, 3).reshape(Hkv, -1, hd) for i in range(2)]
    L = planes[0].shape[1]
    kc, vc = dev(planes[0]), dev(planes[1])
    row = lambda b, width: dev(b.download(np.uint16, (n, width))[2:3])  # noqa: E731
    qg, k, v = row(s.qg, Hq * 2 * hd), row(s.k, Hkv * hd), row(s.v, Hkv * hd)
    split, _ = ops.attn_plan(L, 1, Hkv)
    scratch = R.DeviceBuffer.zeros(ops.attn_scratch_bytes(1, Hq, hd, L, split))
    out, pos = R.DeviceBuffer(Hq * hd * 2), dev(i32(last))
    cos_t, sin_t = ops.rope_tables(L, cfg.rot_dim, cfg.rope_theta)
    dc, dsn = dev(cos_t), dev(sin_t)
    ops.attn_decode(qg=qg.ptr, k=k.ptr, v=v.ptr, q_norm_w=w["q_norm"].ptr, k_norm_w=w["k_norm"].ptr, cos_t=dc.ptr, sin_t=dsn.ptr, k_cache=kc.ptr, v_cache=vc.ptr,
                    pos=pos.ptr, out=out.ptr, scratch=scratch.ptr, B=1, Hq=Hq, Hkv=Hkv, HD=hd, rot_half=cfg.rot_dim // 2, max_len=L, split_len=split,
                    max_pos=L - 1, scale=1 / math.sqrt(hd), fused_norm_rope=1)
    assert R.cuSync() == 0, R.last_error()
    want = val(out.download(np.uint16, (Hq * hd,)))
    assert (np.abs(att[2] - want) <= 2.0 ** -6 * np.abs(val(planes[1])).max()).all()
