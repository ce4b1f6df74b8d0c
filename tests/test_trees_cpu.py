"""Host side of drafted trees on the paged cache: struct layouts, argument packing, and the bounds that the GPU tests allow, without a GPU."""
import ctypes as C

import numpy as np
import pytest

from bunker_b200 import ops
from bunker_b200 import runtime as R


def test_struct_layouts_match_the_header():
    assert C.sizeof(R.bkPagesBatchArgs) == 10 * 8 + 4 * 4 and R.bkPagesBatchArgs.n.offset == 80
    assert C.sizeof(R.bkTreeAttnArgs) == C.sizeof(R.bkPagedAttnArgs) + 3 * 8 + 8 and R.bkTreeAttnArgs.pos.offset == 184 and R.bkTreeAttnArgs.mask_words.offset == 208
    assert C.sizeof(R.bkLogitsArgs) == 15 * 8 + 10 * 4 and R.bkLogitsArgs.B.offset == 120
    assert C.sizeof(R.bkPagesCommitArgs) == 11 * 8 + 4 * 4 and R.bkPagesCommitArgs.T.offset == 92


def test_arguments_are_packed_and_checked():
    a = ops.tree_attn_args(qg=16, lens=32, B=3, T=5, scale=0.5, mask=64, mask_words=1, pos=48)
    assert (a.attn.qg, a.attn.lens, a.attn.B, a.attn.T, a.attn.scale, a.mask, a.mask_words, a.pos, a.slot) == (16, 32, 3, 5, 0.5, 64, 1, 48, 0)
    with pytest.raises(TypeError):
        ops.tree_attn_args(mask=64, mask_words=1, tree=3)
    with pytest.raises(TypeError):
        ops.tree_attn_args(B=3)
    b = ops.adjust_logits_args(logits=16, V=100, B=2, T=1, history=32, history_ld=7)
    assert (b.logits, b.V, b.B, b.T, b.history, b.history_ld, b.ld, b.mask_id) == (16, 100, 2, 1, 32, 7, 0, 0)
    with pytest.raises(TypeError):
        ops.adjust_logits_args(logit=16)


@pytest.mark.parametrize("keys,T,HD", [(40, 9, 128), (300, 40, 128), (900, 64, 256)])
def test_the_bound_of_ready_queries_sees_a_node(keys, T, HD):
    """What the tests of the attention of trees with ready queries allow (2^-8 |o| + 2^-13 of the largest |v|), against an oracle that hides a node which a row
    sees, or shows one which it does not, in the same way for all rows: some row has values outside."""
    rng = np.random.default_rng(keys)
    k, v, q = (rng.normal(0, 1, (n, HD)) for n in (keys + T, keys + T, T))
    s = q @ k.T / np.sqrt(HD)
    seen = np.ones((T, keys + T), bool)
    seen[:, keys:] = np.tril(rng.random((T, T)) < 0.5) | np.eye(T, dtype=bool)
    w = np.exp(s - s.max(1, keepdims=True))

    def attend(m):
        return (w * m) @ v / (w * m).sum(1, keepdims=True)

    o = attend(seen)
    tol = 2.0 ** -8 * np.abs(o) + 2.0 ** -13 * np.abs(v).max()
    for u in range(T):
        other = seen.copy()
        other[:, keys + u] ^= True
        assert (np.abs(attend(other) - o) > tol).any(), u
