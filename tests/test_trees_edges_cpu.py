"""Host side of drafted trees, without a GPU: the layout of what commit takes, and what the command refuses."""
import ctypes as C
import sys

import pytest

from bunker_b200 import runtime as R


def test_commit_takes_the_logits_of_its_targets():
    assert C.sizeof(R.bkPagesCommitArgs) == 104 and R.bkPagesCommitArgs.history_ld.offset == 96 and R.bkPagesCommitArgs.values.offset == 100


@pytest.mark.parametrize("requests", ["-1", "0", "65"])
def test_the_command_refuses_counts_of_requests_by_name(monkeypatch, requests):
    from bunker_b200 import shared_prompt as S
    monkeypatch.setattr(S, "random_layer", lambda cfg: ({}, {"rank": 8, "n_adapters": 3}))
    monkeypatch.setattr(sys, "argv", ["shared_prompt", "--requests", requests])
    with pytest.raises(ValueError, match=f"{requests} requests"):
        S.main()
