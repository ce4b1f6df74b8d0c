"""Host side of drafted trees, without a GPU: the layout of what commit takes."""
import ctypes as C

from bunker_b200 import runtime as R


def test_commit_takes_the_logits_of_its_targets():
    assert C.sizeof(R.bkPagesCommitArgs) == 104 and R.bkPagesCommitArgs.history_ld.offset == 96 and R.bkPagesCommitArgs.values.offset == 100
