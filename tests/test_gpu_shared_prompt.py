"""The example layer where the pool cannot serve a request: nothing that was there may change, and nobody may read what is not there.

Everything that is compared is equal bit for bit: pages, tables and lengths of the same inputs, or of a run that had room.
"""
import numpy as np
import pytest

from bunker_b200 import runtime as R
from bunker_b200 import shared_prompt as S
from bunker_b200.model import CONFIG_TINY as cfg
from tests.test_gpu_serving import rnd
from tests.util import dev

pytestmark = pytest.mark.gpu

ADAPTERS = [0, -1, 2]


@pytest.fixture(scope="module")
def layer(bk):
    return S.random_layer(cfg, seed=5)


@pytest.fixture(scope="module")
def x(bk):
    return dev(rnd(np.random.default_rng(6), 128, cfg.hidden))


def make(layer, max_rows, n_pages, n=3):
    return S.SharedPrompt(cfg, *layer, n, max_rows, n_pages)


def held(s):
    """(keys and values of each sequence's rows, lens)"""
    d = s.pool.desc
    data = s.data.download(np.uint16, (2, d.n_pages, d.heads, d.page_rows, d.row_bytes // 2))
    lens = s.lens.download(np.int32, (d.n_seqs,))
    table = s.table.download(np.int32, (d.n_seqs, d.max_pages))
    out = []
    for i, n in enumerate(lens):
        j = np.arange(n)
        out.append(data[:, table[i, j // d.page_rows], :, j % d.page_rows].copy())
    return out, lens.tolist()


def attended(s):
    return s.att.download(np.uint16, (s.n, cfg.attn_q_heads * cfg.head_dim))


def test_a_step_without_a_page_for_all_leaves_the_prompt_as_it_was(layer, x):
    """48 rows fill three pages, which all requests share; one page is left for three of them.  Who is served gets what it gets alone."""
    def alone(i):
        r = make(layer, 80, 12)
        r.prompt(x.ptr, 48)
        r.fork([i])
        r.step(x.ptr, ADAPTERS)
        assert R.cuSync() == 0, R.last_error()
        return attended(r)

    s = make(layer, 80, 4)
    s.prompt(x.ptr, 48)
    s.fork(range(3))
    before, _ = held(s)
    s.step(x.ptr, ADAPTERS)
    assert R.cuSync() == 0, R.last_error()
    rows, lens = held(s)
    assert s.ok.download(np.int32, (3,)).tolist() == [1, 0, 0] and lens == [48, 49, 48, 48]
    for i in range(4):
        assert np.array_equal(rows[i][:48], before[i])
    got = attended(s)
    assert not got[1:].any() and np.array_equal(got[0], alone(0)[0])      # refused: not there
    # a page comes back: the next step serves who has room
    s.drop([0])
    s.step(x.ptr, ADAPTERS)
    assert s.ok.download(np.int32, (3,)).tolist() == [1, 1, 0]            # (no row is asked for request 0)
    rows, lens = held(s)
    assert lens == [48, 0, 49, 48]
    for i in (0, 2, 3):
        assert np.array_equal(rows[i][:48], before[i])
    got = attended(s)
    assert not got[[0, 2]].any() and np.array_equal(got[1], alone(1)[1])


def test_a_step_past_the_longest_sequence_changes_nothing(layer, x):
    s = make(layer, 64, 20)
    s.prompt(x.ptr, 62)
    s.fork([0, 2])
    for _ in range(2):
        s.step(x.ptr, ADAPTERS)
    before, lens = held(s)
    assert lens == [62, 64, 0, 64]
    s.step(x.ptr + 2 * cfg.hidden, ADAPTERS)
    after, lens = held(s)
    assert lens == [62, 64, 0, 64] and not attended(s).any()
    assert all(np.array_equal(a, b) for a, b in zip(before, after))


@pytest.mark.parametrize("max_rows,n_pages", [(112, 4), (64, 20)])    # the pages run out, or the table's row
def test_a_prompt_that_does_not_fit_says_so_and_keeps_what_did(layer, x, max_rows, n_pages):
    s, fits = make(layer, max_rows, n_pages), make(layer, 112, 20)
    fits.prompt(x.ptr, 64)
    with pytest.raises(RuntimeError, match="64 of 100"):
        s.prompt(x.ptr, 100)
    assert R.cuSync() == 0 and s.prompt_rows == 64
    rows, lens = held(s)
    assert lens[0] == 64 and np.array_equal(rows[0], held(fits)[0][0])


def test_a_request_whose_fork_found_no_page_is_not_active(layer, x):
    s = make(layer, 64, 4)
    s.prompt(x.ptr, 40)                      # three pages, the last one partial: every fork needs one
    assert s.fork([1, 0, 2]).tolist() == [True, False, False]
    assert s.active.tolist() == [False, True, False]
    assert s.fork([1]).tolist() == [False] and s.active.tolist() == [False, True, False]     # (it is not empty)
    s.step(x.ptr, ADAPTERS)
    rows, lens = held(s)
    assert lens == [40, 0, 41, 0] and not attended(s)[[0, 2]].any() and attended(s)[1].any()


def test_a_prompt_cannot_grow_under_its_requests(layer, x):
    """Rows added then would be read as common rows by requests that do not have them."""
    s = make(layer, 96, 20)
    s.prompt(x.ptr, 32)
    s.fork([0, 1])
    before, lens = held(s)
    with pytest.raises(RuntimeError, match="request"):
        s.prompt(x.ptr, 16)
    after, now = held(s)
    assert s.prompt_rows == 32 and now == lens and all(np.array_equal(a, b) for a, b in zip(before, after))
    s.drop([0, 1])
    s.prompt(x.ptr, 16)
    assert s.prompt_rows == 48 and s.fork([2]).all() and held(s)[1] == [48, 0, 0, 48]


def test_requests_that_are_none_are_refused(layer, x):
    """Request -1 would be the prompt's own sequence."""
    s = make(layer, 64, 20)
    s.prompt(x.ptr, 32)
    s.fork([0])
    before, lens = held(s)
    for bad in ([-1], [0, 3]):
        with pytest.raises(IndexError):
            s.drop(bad)
        with pytest.raises(IndexError):
            s.fork(bad)
    with pytest.raises(ValueError):
        s.step(x.ptr, ADAPTERS[:2])
    after, now = held(s)
    assert now == lens and all(np.array_equal(a, b) for a, b in zip(before, after)) and s.active.tolist() == [True, False, False]


@pytest.mark.parametrize("steps", [1, 2, 3, 20])
def test_the_command_has_room_for_its_steps(bk, monkeypatch, steps):
    """Every step that the command takes is served."""
    seen = []
    step = S.SharedPrompt.step

    def watched(self, *a, **kw):
        out = step(self, *a, **kw)
        seen.append(bool(self.ok.download(np.int32, (self.n,)).all()))
        return out

    monkeypatch.setattr(S.SharedPrompt, "step", watched)
    monkeypatch.setattr("sys.argv", ["shared_prompt", "--requests", "4", "--prompt", "46", "--steps", str(steps)])
    S.main()
    assert seen and all(seen)
