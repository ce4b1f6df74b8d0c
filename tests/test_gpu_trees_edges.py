"""Drafted trees where they can go wrong: grammars that allow nothing, results that lie over inputs, calls without counts or without new rows, trees and drafts of many nodes, and the
attention against bounds that a single hidden or extra node does not stay inside.  Expectations and helpers are those of test_gpu_trees.py.
"""
import ctypes as C
import math

import numpy as np
import pytest

from bunker_b200 import ops
from bunker_b200 import runtime as R
from tests.test_gpu_serving import bf16, i32, rnd, val
from tests.test_gpu_trees import Draft, Logits, TreeCase, words
from tests.util import dev

pytestmark = pytest.mark.gpu


# ---- grammars that allow nothing, or next to nothing ----------------------------------

@pytest.mark.parametrize("V", [37, 5000, 151936])
@pytest.mark.parametrize("how", ["argmax", "sample"])
def test_a_grammar_that_allows_nothing_ends_the_path(bk, V, how):
    """Rows of -inf: the selection says so by its val, and commit, which is given the vals, keeps no child of such a node although its token is the one that the selection named."""
    n, T = 4, 5
    rng = np.random.default_rng(V)
    c = Logits(V, n, T, V, history=20, n_masks=3)
    allowed = np.zeros((3, V), bool)
    allowed[1, rng.permutation(V)[:3]] = True
    allowed[2] = True
    c.allowed = words(allowed, c.W)
    c.allowed[:, -1] = 0xFFFFFFFF                      # (bits behind the vocabulary)
    c.mask_id = i32(*[(0, -1, 1, 2)[(t + i) % 4 if i else (1, 1, 0, 1, 1)[t]] for t in range(T) for i in range(n)])
    dead = (c.mask_id == 0).reshape(T, n)
    got = c.check()
    assert np.isneginf(got.reshape(T, n, V)[dead]).all() and dead.any(0).any()
    chosen, a = R.DeviceBuffer(8 * T * n), c.args()
    ops.adjust_logits(a)
    if how == "argmax":
        scratch = R.DeviceBuffer.zeros(ops.argmax_scratch_bytes(T * n))
        ops.argmax(a.logits, V, T * n, chosen.ptr, chosen.ptr + 4 * T * n, scratch.ptr)
    else:
        ops.sample(a.logits, V, T * n, chosen.ptr, chosen.ptr + 4 * T * n, temperature=1.3, top_k=40, seed=3)
    assert R.cuSync() == 0, R.last_error()
    idx, logit = chosen.download(np.int32, (2, T, n))[0], chosen.download(np.float32, (2, T, n))[1]
    assert np.array_equal(np.isneginf(logit), dead) and (idx >= 0).all() and (idx < V).all()
    p = Draft(rng, n_pages=24, seqs=n)
    order = list(rng.permutation(24))
    for s in range(n):
        p.own(s, 20 + 3 * s, order)
    p.grown(rng, T, [T] * n)
    p.parent[:] = np.arange(-1, T - 1)[:, None]
    p.token[1:] = idx[:-1]                             # every node is what the selection named after its parent
    pool = p.upload()
    d = {k: dev(x) for k, x in (("seqs", np.arange(n, dtype=np.int32)), ("parent", p.parent), ("token", p.token))}
    o = {k: R.DeviceBuffer.from_numpy(np.full(size, 77, np.int32)) for k, size in (("path", T * n), ("n_path", n), ("next", n), ("ok", n))}
    pool.commit(n=n, T=T, target=chosen.ptr, values=True, **{k: b.ptr for k, b in {**d, **o}.items()})
    p.target = np.where(dead, -1, idx)
    want = p.commit(np.arange(n))
    p.check()
    for (name, b), w in zip(o.items(), want):
        assert np.array_equal(b.download(np.int32, w.shape), w), name
    first = np.where(dead.any(0), dead.argmax(0), T - 1)
    assert np.array_equal(want[1], first + 1) and np.array_equal(want[2] == -1, dead.any(0))


def test_a_target_below_zero_is_no_token(bk):
    """Also where a node's own token is below zero."""
    rng = np.random.default_rng(1)
    p = Draft(rng, seqs=2)
    p.own(0, 20, [3, 4])
    p.grown(rng, 4, [4])
    p.parent[:, 0], p.token[:, 0], p.target[:, 0] = [-1, 0, 0, 1], [5, -1, 8, 9], [-1, 9, 3, 2]
    pool = p.upload()
    d = {k: dev(x) for k, x in (("seqs", i32(0)), ("parent", p.parent), ("token", p.token), ("target", p.target))}
    o = {k: R.DeviceBuffer.from_numpy(np.full(4, 77, np.int32)) for k in ("path", "n_path", "next", "ok")}
    pool.commit(n=1, T=4, **{k: b.ptr for k, b in {**d, **o}.items()})
    assert R.cuSync() == 0, R.last_error()
    got = {k: b.download(np.int32, (4,)).tolist() for k, b in o.items()}
    assert got == {"path": [0, -1, -1, -1], "n_path": [1, 77, 77, 77], "next": [-1, 77, 77, 77], "ok": [1, 77, 77, 77]}
    assert p.d["lens"].download(np.int32, (2,)).tolist() == [17, 0]
    a = R.bkPagesCommitArgs(seqs=d["seqs"].ptr, parent=d["parent"].ptr, token=d["token"].ptr, target=d["target"].ptr, n=1, T=4, values=2)
    assert R.cu().bkPagesCommit(C.byref(pool.desc), C.byref(a)) == R.BK_ERR_ARG and "values" in R.last_error()


@pytest.mark.parametrize("V,few", [(33, 1), (33, 7), (9000, 1), (9000, 5), (151936, 3), (151936, 39)])
@pytest.mark.parametrize("top_k", [1, 2, 40, 64])
def test_a_sample_of_fewer_tokens_than_it_may_look_at(bk, V, few, top_k):
    """A mask that leaves fewer tokens than top_k: only those are ever chosen, whatever the temperature and nucleus."""
    B, rng = 3, np.random.default_rng(V + few)
    c = Logits(few, B, 1, V, n_masks=1, history=9)
    allowed = np.zeros((1, V), bool)
    allowed[0, rng.permutation(V)[:few]] = True
    c.allowed, c.mask_id = words(allowed, c.W), i32(0, 0, 0)
    a = c.args()
    ops.adjust_logits(a)
    idx, v = R.DeviceBuffer(4 * B), R.DeviceBuffer(4 * B)
    seen = set()
    for step in range(40):
        ops.sample(a.logits, V, B, idx.ptr, v.ptr, temperature=(0.0, 0.3, 1.0, 50.0)[step % 4], top_k=top_k, top_p=(1.0, 0.9)[step % 2], seed=11, step_add=step)
        got = idx.download(np.int32, (B,))
        assert allowed[0, got].all() and np.isfinite(v.download(np.float32, (B,))).all()
        seen |= set(got.tolist())
    assert few == 1 or top_k == 1 or len(seen) > 1


def test_the_layer_ends_a_path_where_nothing_is_allowed(bk):
    from bunker_b200 import shared_prompt as S
    from bunker_b200.model import CONFIG_TINY as cfg
    w, lora = S.random_layer(cfg, seed=5)
    s = S.SharedPrompt(cfg, w, lora, 2, 64, 8)
    x = dev(rnd(np.random.default_rng(1), 64, cfg.hidden))
    s.prompt(x.ptr, 20)
    assert s.fork([0, 1]).all()
    chain = np.array([[-1, -1], [0, 0], [1, 1]], np.int32)
    token = np.array([[4, 4], [0, 0], [6, 6]], np.int32)
    target, logit = np.array([[0, 0], [6, 6], [2, 3]], np.int32), np.array([[1.5, -np.inf], [0.0, 1.0], [-2.0, 1.0]], np.float32)
    for values, kept_want, next_want in ((False, [3, 3], [2, 3]), (True, [3, 1], [2, -1])):
        s.draft(x.ptr, chain, [-1, -1])
        d = dev(np.concatenate([target.view(np.uint32), logit.view(np.uint32)]))
        kept, after = s.keep(token, d.ptr, values=values)
        assert kept.tolist() == kept_want and after.tolist() == next_want


# ---- results that lie over what a call reads --------------------------------------------

def test_commit_refuses_results_over_its_inputs(bk):
    """Ranges, not addresses alone: lists, trees, histories, and the pool's own tables, counts, lengths and pages."""
    rng = np.random.default_rng(5)
    p = Draft(rng, planes=2, seqs=3)
    p.own(0, 20, [3, 4])
    p.own(1, 30, [5, 6])
    n, T = 2, 4
    p.grown(rng, T, [T] * n)
    pool = p.upload()
    every = R.DeviceBuffer.from_numpy(np.full(512, 1, np.int32))
    size = dict(seqs=n, n_new=n, parent=n * T, token=n * T, target=2 * n * T, path=n * T, n_path=n, next=n, ok=n, history=3 * 9, hist_len=3)
    at, place = {}, every.ptr
    for k, m in size.items():
        at[k], place = place, place + 4 * m
    lib = R.cu()

    def call(**change):
        a = R.bkPagesCommitArgs(**{**at, **dict(n=n, T=T, history_ld=9, values=1), **change})
        return lib.bkPagesCommit(C.byref(pool.desc), C.byref(a))

    data = p.d["data"].ptr
    pools = [(p.d["lens"].ptr, 12), (p.d["table"].ptr, p.table.nbytes), (p.d["ref"].ptr, p.ref.nbytes), (data, p.data.nbytes // 2), (data + p.data.nbytes // 2, p.data.nbytes // 2)]
    for w in ("path", "n_path", "next", "ok", "history", "hist_len"):
        reads = [k for k in ("seqs", "n_new", "parent", "token", "target", "history", "hist_len") if k != w and not (w == "hist_len" and k == "history")]
        for lo, length in [(at[k], 4 * size[k]) for k in reads] + pools:
            for place in (lo, lo + length - 4, lo - 4 * size[w] + 4):
                assert call(**{w: place}) == R.BK_ERR_ARG and "apart" in R.last_error(), (w, R.last_error())
    p.check("nothing changed")
    assert np.array_equal(every.download(np.int32, (512,)), np.full(512, 1, np.int32))
    # side by side, as they lie here, they are apart
    R.cuHtoD(at["seqs"], i32(0, 1))
    R.cuHtoD(at["n_new"], i32(T, T))
    for k, x in (("parent", p.parent), ("token", p.token), ("target", p.target)):
        R.cuHtoD(at[k], x)
    R.cuHtoD(at["hist_len"], i32(0, 2, 0))
    history, hist_len = np.full((3, 9), 1, np.int32), i32(0, 2, 0)
    assert call() == 0
    want = p.commit(i32(0, 1), history, hist_len)
    p.check()
    got = every.download(np.int32, (512,))
    for k, w in (("path", want[0]), ("n_path", want[1]), ("next", want[2]), ("ok", want[3]), ("history", history), ("hist_len", hist_len)):
        first = (at[k] - every.ptr) // 4
        assert np.array_equal(got[first:first + w.size], w.reshape(-1)), k


def test_batch_refuses_results_over_its_inputs(bk):
    """lens in the place of the pool's own lens, for one, would be written by a sequence's first CTA while the others read it."""
    rng = np.random.default_rng(6)
    p = Draft(rng, planes=2, seqs=3)
    p.own(0, 20, [3, 4])
    p.own(1, 30, [5, 6])
    n, T, W = 3, 4, 2
    pool = p.upload()
    every = R.DeviceBuffer.from_numpy(np.full(512, 1, np.int32))
    size = dict(seqs=n, n_new=n, parent=n * T, ok=n, table=n * p.max_pages, lens=n, pos=n * T, slot=n * T, mask=n * T * W, count=n)
    at, place = {}, every.ptr
    for k, m in size.items():
        at[k], place = place, place + 4 * m
    lib = R.cu()

    def call(**change):
        a = R.bkPagesBatchArgs(**{**at, **dict(n=n, T=T, mask_words=W), **change})
        return lib.bkPagesBatch(C.byref(pool.desc), C.byref(a))

    pools = [(p.d["lens"].ptr, 12), (p.d["table"].ptr, p.table.nbytes), (p.d["ref"].ptr, p.ref.nbytes), (p.d["data"].ptr, p.data.nbytes)]
    for w in ("table", "lens", "pos", "slot", "mask", "count"):
        for k, lo, length in [(k, at[k], 4 * size[k]) for k in ("seqs", "n_new", "parent", "ok")] + [("pool", *x) for x in pools]:
            for place in (lo, lo + length - 4, lo - 4 * size[w] + 4):
                if w == "count" and k in ("n_new", "ok") and place == lo:
                    continue                                    # (these may be the same)
                assert call(**{w: place}) == R.BK_ERR_ARG and "apart" in R.last_error(), (w, k, R.last_error())
    p.check("nothing changed")
    assert np.array_equal(every.download(np.int32, (512,)), np.full(512, 1, np.int32))
    assert call(count=at["n_new"], lens=at["n_new"]) == R.BK_ERR_ARG and "apart" in R.last_error()
    # side by side, as they lie here, they are apart; so are count and what it comes from where they are one array
    for one in ("count", "n_new", "ok"):
        R.cuHtoD(every.ptr, np.full(512, 1, np.int32))
        R.cuHtoD(at["seqs"], i32(0, 2, 1))
        R.cuHtoD(at["n_new"], i32(T, T, 2))
        assert call(count=at[one], parent=0) == 0
        assert R.cuSync() == 0
        got = every.download(np.int32, (512,))
        part = {k: got[(at[k] - every.ptr) // 4:][:m] for k, m in size.items()}
        assert part[one].tolist() == [T, 0, 2] and part["lens"].tolist() == [20, 0, 30]
        assert part["pos"].reshape(T, n).T.tolist() == [[16, 17, 18, 19], [-1] * 4, [28, 29, -1, -1]]
    p.check("unchanged")
    b = R.bkPagesBatchArgs(seqs=at["seqs"], n=n, T=T, n_new=at["n_new"], ok=at["n_new"], count=at["n_new"])      # all three
    assert lib.bkPagesBatch(C.byref(pool.desc), C.byref(b)) == 0 and R.cuSync() == 0


# ---- attention: what a single hidden or extra node moves ---------------------------------

def row_bound(w, v, o, d, gate=1.0):
    """What a row's result o gate [HD], o = w v, may be off by: 16 bits of probabilities (2^-13 of the largest |v|, see test_gpu_trees.py), scores that are off by up to d, 2^-20 of it
    for the sigmoid and its product, and one rounding of what all that gives (2^-8 of it).  Weights w_j f_j with 1 / e^d <= f_j <= e^d give
    o + sum w_j (f_j - 1) (v_j - o) / sum w_j f_j, for sum w_j (v_j - o) is 0: at most (e^d - 1) e^d sum w_j |v_j - o| from o."""
    before = gate * (2.0 ** -13 * np.abs(v).max() + math.expm1(d) * math.exp(d) * (w @ np.abs(v - o))) + 2.0 ** -20 * np.abs(o * gate)
    return 2.0 ** -8 * np.abs(o * gate) + (1 + 2.0 ** -8) * before


def check_rows(c, **change):
    """As TreeCase.check, but with the keys that the call left in the pages, and with values of a query that lie so near the border of two bf16 values that the call may have taken either:
    a score is off by what those make of it, and no more.  A value of q is x / sqrt(mean x^2 + eps) (1 + w), in f32: the sum of squares is off by 14 roundings of 2^-24, half of it after the
    root, which has 4 more, and 3 products; then the rotation's products and sum, 3 of its terms' size, which the pair's length bounds: 2^-19 of the length in all."""
    bits = c.run(c.tree_args(**change))
    got = val(bits)
    want, kp, vp = c.want()
    k = c.keep["kp"].download(np.uint16, c.kp.shape)
    assert np.array_equal(c.keep["vp"].download(np.uint16, c.vp.shape), vp)
    changed = kp != c.kp
    assert np.array_equal(k[~changed], kp[~changed])
    assert (np.abs(val(k[changed]) - val(kp[changed])) <= 2.0 ** -7 * np.abs(val(kp[changed])) + 2.0 ** -16).all()
    assert not bits[c.nothing_seen()].any()
    at, G, r = c.positions(), c.Hq // c.Hkv, c.rot
    for b in range(c.B):
        n, base = c.n_base(b)
        for t in range(n):
            e, j = t * c.B + b, np.concatenate([np.arange(base), base + np.nonzero(c.sees[t, b, :n])[0]])
            if at[t, b] < 0 or not len(j):
                continue
            K, V = (val(x[c.table[b, j // c.rows], :, j % c.rows]) for x in (k, vp))
            q, off = val(c.q[e]), np.zeros((c.Hq, c.HD))
            if c.fused:
                y = c.turned(c.q[e], c.qw, c.pos[t, b])
                size = np.abs(y)
                size[:, :r] = size[:, r:2 * r] = np.hypot(y[:, :r], y[:, r:2 * r])
                q = val(bf16(y))
                off = np.abs(val(bf16(y + 2.0 ** -19 * size)) - val(bf16(y - 2.0 ** -19 * size)))
            gate = 1 / (1 + np.exp(-val(c.g[e]))) if c.g is not None else np.ones((c.Hq, c.HD))
            for h in range(c.Hq):
                Kh, Vh = K[:, h // G], V[:, h // G]
                s = Kh @ q[h] * float(c.scale)
                w = np.exp(s - s.max())
                w /= w.sum()
                o = w @ Vh
                d = float(c.scale) * (np.abs(Kh) @ off[h]).max()
                tol = row_bound(w, Vh, o, d, gate[h])
                bad = np.abs(got[e, h] - o * gate[h]) > tol
                assert not bad.any(), (b, t, h, np.abs(got[e, h] - o * gate[h])[bad][:4], tol[bad][:4], d)


@pytest.mark.parametrize("fused", [True, False])
@pytest.mark.parametrize("B,T,prefix,own,new,Hq,Hkv,HD,rows", [
    (1, 8, 0, [8], None, 4, 1, 128, 16), (1, 32, 0, [65], None, 4, 1, 128, 16), (1, 32, 0, [33], None, 8, 1, 256, 32), (4, 12, 150, [12, 40, 77, 13], [12, 5, 1, 12], 16, 2, 256, 64),
    (2, 40, 0, [140, 41], [40, 33], 8, 2, 256, 16), (1, 64, 0, [128], None, 6, 1, 128, 16), (3, 9, 70, [9, 50, 20], [9, 4, 9], 4, 1, 128, 16), (2, 33, 64, [70, 34], [33, 20], 24, 4, 128, 32),
    (20, 5, 40, [5 + i for i in range(20)], [5 - i % 3 for i in range(20)], 8, 1, 256, 16)])
@pytest.mark.parametrize("tree", ["tree", "any"])
def test_no_node_is_hidden_or_shown_that_is_not(bk, fused, B, T, prefix, own, new, Hq, Hkv, HD, rows, tree):
    """Up to 230 keys a row: a bit that is wrong in one row is outside these bounds (the CPU's tests say how surely), with ready queries and with the fused norm."""
    check_rows(TreeCase(T + Hq + HD, B, T, prefix, own, tree=tree, new=new, Hq=Hq, Hkv=Hkv, HD=HD, rows=rows, fused=fused))


# ---- attention: forms of the call ---------------------------------------------------------

@pytest.mark.parametrize("HD,prefix", [(128, 0), (128, 70), (256, 48)])
def test_trees_whose_rows_are_in_the_pages_already(bk, HD, prefix):
    """k, v and slot 0: nothing is stored, the same results to the bit."""
    c = TreeCase(HD + prefix, 3, 9, prefix, [9, 50, 20], new=[9, 4, 9], Hq=8, Hkv=2, HD=HD, fused=False)
    first = c.run(c.tree_args())
    _, c.kp, c.vp = c.want()
    a = c.tree_args(pos=0, slot=0)
    a.attn.k = a.attn.v = 0
    assert np.array_equal(c.run(a), first)
    assert np.array_equal(c.keep["kp"].download(np.uint16, c.kp.shape), c.kp) and np.array_equal(c.keep["vp"].download(np.uint16, c.vp.shape), c.vp)


@pytest.mark.parametrize("fused", [True, False])
@pytest.mark.parametrize("B,T,own", [(1, 1, [1]), (3, 7, [7, 60, 8]), (5, 33, [40, 33, 32, 90, 34])])
def test_trees_of_all_nodes_without_counts(bk, fused, B, T, own):
    """n_new 0: T of each; a sequence with fewer rows has none."""
    c = TreeCase(T, B, T, 0, own, new=[T] * B, Hq=4, Hkv=2, HD=128, fused=fused)
    first = c.run(c.tree_args())
    c = TreeCase(T, B, T, 0, own, new=[T] * B, Hq=4, Hkv=2, HD=128, fused=fused)
    a = c.tree_args()
    a.attn.n_new = 0
    assert np.array_equal(c.run(a), first)
    c.check()


@pytest.mark.parametrize("B,T,prefix,own,new,Hq,Hkv,HD,tree", [
    (1, 300, 0, [300], None, 2, 1, 128, "any"), (2, 600, 100, [611, 320], [600, 311], 2, 2, 128, "tree"), (1, 1024, 0, [1200], None, 4, 1, 128, "tree"), (1, 513, 40, [513], None, 16, 1, 256, "tree"),
    (3, 257, 0, [257, 300, 200], [257, 256, 129], 3, 1, 256, "any")])
def test_trees_of_many_nodes(bk, B, T, prefix, own, new, Hq, Hkv, HD, tree):
    TreeCase(T, B, T, prefix, own, tree=tree, new=new, Hq=Hq, Hkv=Hkv, HD=HD, fused=T % 2 == 0).check(1)


# ---- logits of many nodes -------------------------------------------------------------------

@pytest.mark.parametrize("B,T,V,history,n_bias,n_masks", [(1, 513, 300, 0, 0, 0), (1, 1024, 700, 50, 9, 3), (2, 600, 1500, 300, 0, 2), (1, 1000, 9000, 4000, 1024, 0), (3, 512, 33, 7, 2, 2)])
def test_logits_of_trees_of_many_nodes(bk, B, T, V, history, n_bias, n_masks):
    """Above 512 nodes a thread has more than one drafted token; tokens of the whole vocabulary, and of a few."""
    c = Logits(T + V, B, T, V, history=history, n_bias=n_bias, n_masks=n_masks, tree=True)
    c.check()
    c.draft = np.random.default_rng(T).integers(-1, V + 1, T * B).astype(np.int32)
    c.check()
