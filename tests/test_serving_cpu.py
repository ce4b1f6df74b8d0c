"""Host side of the paged cache, the attention over it and the adapters: struct layouts and argument packing, without a GPU."""
import ctypes as C

import numpy as np
import pytest

from bunker_b200 import ops, pages
from bunker_b200 import runtime as R


def test_struct_layouts_match_the_header():
    assert C.sizeof(R.bkPages) == 7 * 8 + 8 * 4 and R.bkPages.n_planes.offset == 56
    assert C.sizeof(R.bkPagedAttnArgs) == 16 * 8 + 12 * 4 + 8 and R.bkPagedAttnArgs.B.offset == 128 and R.bkPagedAttnArgs.scale.offset == 176
    assert C.sizeof(R.bkLoraSeg) == 48 and C.sizeof(R.bkLoraArgs) == 24 + 5 * 8 + 4 * 48 and R.bkLoraArgs.segs.offset == 64


def test_scratch_sizes_without_a_gpu():
    assert pages.scratch_bytes(0, 1) == 0 and pages.scratch_bytes(1000, 4) >= 8000 and pages.scratch_bytes(1000, 4) % 16 == 0
    assert ops.lora_scratch_bytes(5120, 64, 32, 2) >= 64 * 32 * 2 * 4 and ops.lora_scratch_bytes(0, 1, 8, 1) == 0


def test_a_pool_is_described_as_given():
    p = pages.PagePool(base=256, n_planes=3, n_pages=7, heads=2, page_rows=16, row_bytes=512, n_seqs=4, max_pages=5, ref=1024, table=2048, lens=4096,
                       scratch=8192, scratch_bytes=999)
    d = p.desc
    assert d.plane_bytes == 7 * 2 * 16 * 512 and (d.n_planes, d.n_pages, d.heads, d.page_rows, d.row_bytes, d.n_seqs, d.max_pages) == (3, 7, 2, 16, 512, 4, 5)
    assert p.plane(2) == 256 + 2 * d.plane_bytes
    with pytest.raises(IndexError):
        p.plane(3)


def test_arguments_are_packed_and_checked():
    a = ops.paged_attn_args(qg=16, len=32, B=3, scale=0.5)
    assert (a.qg, a.lens, a.B, a.scale, a.k) == (16, 32, 3, 0.5, 0)
    with pytest.raises(TypeError):
        ops.paged_attn_args(batch=3)
    seg = ops.lora_seg(A=16, Bm=32, n_rows=10, out=48, col_off=6)
    assert (seg.ld_out, seg.dtype, seg.base) == (16, R.BK_DTYPE_F32, 0)
    l = ops.lora_args(x=16, K=64, B=2, rank=8, n_adapters=1, ids=32, segs=[seg, seg], scratch=64, scratch_bytes=128)
    assert l.n_segs == 2 and l.segs[1].A == 16 and l.scale == 0
    for n in (0, 5):
        with pytest.raises(ValueError):
            ops.lora_args(x=16, K=64, B=2, rank=8, n_adapters=1, ids=32, segs=[seg] * n, scratch=64, scratch_bytes=128)


def test_the_plan_of_the_example_is_refused_for_too_many_requests():
    from bunker_b200.model import CONFIG_TINY
    from bunker_b200.shared_prompt import SharedPrompt
    for n in (0, 65):
        with pytest.raises(ValueError):
            SharedPrompt(CONFIG_TINY, {}, {"rank": 8, "n_adapters": 1}, n, 100, 10)


@pytest.mark.parametrize("keys,HD", [(2150, 128), (1375, 256), (2577, 256)])
def test_the_bound_of_ready_queries_sees_a_tile_of_keys(keys, HD):
    """What the tests of attention over pages with ready queries allow (2^-8 |o| + 2^-13 of the largest |v|), against an oracle that leaves out a tile of
    64 keys, or 16 keys, or takes them twice: every row of queries has values outside."""
    rng = np.random.default_rng(keys)
    k, v, q = (rng.normal(0, 1, (n, HD)) for n in (keys, keys, 48))
    s = q @ k.T / np.sqrt(HD)
    w = np.exp(s - s.max(1, keepdims=True))
    o = w @ v / w.sum(1, keepdims=True)
    tol = 2.0 ** -8 * np.abs(o) + 2.0 ** -13 * np.abs(v).max()
    for first, n in [(64 * i, 64) for i in range(keys // 64)] + [(64 * i + 48, 16) for i in range(keys // 64)]:
        for times in (0, 2):
            z = w.copy()
            z[:, first:first + n] *= times
            wrong = z @ v / z.sum(1, keepdims=True)
            assert (np.abs(wrong - o) > tol).any(1).all(), (first, n, times)
