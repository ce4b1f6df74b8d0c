"""Host side of drafted trees, without a GPU: the layout of what commit takes, and what the command refuses, and what the bounds of the attention's
tests see."""
import ctypes as C
import sys

import numpy as np
import pytest

from bunker_b200 import runtime as R
from tests.test_gpu_trees_edges import row_bound


def test_commit_takes_the_logits_of_its_targets():
    assert C.sizeof(R.bkPagesCommitArgs) == 104 and R.bkPagesCommitArgs.history_ld.offset == 96 and R.bkPagesCommitArgs.values.offset == 100


@pytest.mark.parametrize("requests", ["-1", "0", "65"])
def test_the_command_refuses_counts_of_requests_by_name(monkeypatch, requests):
    from bunker_b200 import shared_prompt as S
    monkeypatch.setattr(S, "random_layer", lambda cfg: ({}, {"rank": 8, "n_adapters": 3}))
    monkeypatch.setattr(sys, "argv", ["shared_prompt", "--requests", requests])
    with pytest.raises(ValueError, match=f"{requests} requests"):
        S.main()


@pytest.mark.parametrize("gated", [True, False])
@pytest.mark.parametrize("keys,T,HD,G,missed", [(0, 8, 128, 4, 0), (33, 32, 128, 4, 0), (1, 32, 256, 8, 0), (190, 12, 256, 8, 0), (64, 64, 128, 6, 0), (100, 40, 256, 4, 0.004)])
def test_the_bound_of_a_row_sees_one_bit(keys, T, HD, G, missed, gated):
    """A node that one row sees and should not, or the other way, among keys + T keys: some of its G heads has a value outside what the row is allowed, with a value of its query that may
    be rounded either way.  All bits of all rows, but for `missed` of them (a node of little weight in every head)."""
    rng = np.random.default_rng(keys + T)
    k, v = (rng.normal(0, 1, (keys + T, HD)) for _ in range(2))
    q, gate = rng.normal(0, 1, (T, G, HD)), 1 / (1 + np.exp(-rng.normal(0, 1, (T, G, HD)))) if gated else np.ones((T, G, HD))
    s = np.einsum("tgd,jd->tgj", q, k) / np.sqrt(HD)
    weight = np.exp(s - s.max(2, keepdims=True))
    seen = np.ones((T, keys + T), bool)
    seen[:, keys:] = np.tril(rng.random((T, T)) < 0.5) | np.eye(T, dtype=bool)
    inside = 0
    for t in range(T):
        w = weight[t] * seen[t]
        z = w.sum(1)
        o = w @ v / z[:, None]
        d = 2.0 ** -7 * np.abs(q[t]).max() * np.abs(k).max() / np.sqrt(HD)
        tol = np.stack([row_bound(w[h] / z[h], v, o[h], d, gate[t, h]) for h in range(G)])
        for u in range(T):
            flip = weight[t, :, keys + u] * (-1 if seen[t, keys + u] else 1)
            if (z + flip).min() <= 1e-9:
                continue                       # (its only key: then the row is zeros)
            other = (w @ v + flip[:, None] * v[keys + u]) / (z + flip)[:, None]
            inside += not (np.abs(other - o) * gate[t] > tol).any()
    assert inside <= missed * T * T
