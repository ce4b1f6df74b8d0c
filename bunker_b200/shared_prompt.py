"""Many requests behind one prompt: an attention layer served from a cache in pages, with an adapter per request.

    python -m bunker_b200.shared_prompt [--requests N] [--prompt N] [--steps N] [--draft N]

The prompt is written once, in chunks of up to 64 tokens; every request is a fork of it (whole pages shared, a partial last page
copied); a step of all requests is RMSNorm, the shared Q4_K projections with the requests' adapters beside them, the attention
that computes the prompt's rows once for all, and the output projection with the residual.  Instead of one token a request may bring
a tree of drafted ones (``draft``), of which ``keep`` leaves the path that the model agrees with.  Finished requests give their pages
back, and the pool can be compacted at any time.  All of it is enqueued on the library stream.  The host waits for the GPU where it
uploads a list (three times a step; a server would keep lists that stay in their place) and where it asks the pool what was served
(``prompt``, ``fork``; not ``step``, whose answer is ``ok``).
"""
from __future__ import annotations

import math
from typing import Sequence

import numpy as np

from . import ops, pages, synth
from . import runtime as R
from .model import CONFIG_TINY, ModelConfig


class SharedPrompt:
    """One attention layer of ``cfg`` for up to ``requests`` requests.  ``w``: device buffers, Q4_K rows "q", "k", "v", "o" and bf16
    "ln", "q_norm", "k_norm"; ``lora``: bf16 "A_q", "B_q", "A_k", "B_k", "A_v", "B_v" of all adapters, ``rank``, ``n_adapters``."""

    CHUNK = 64      # columns of a projection

    def __init__(self, cfg: ModelConfig, w: dict, lora: dict, requests: int, max_rows: int, n_pages: int, page_rows: int = 16):
        if not 1 <= requests <= self.CHUNK:
            raise ValueError(f"{requests} requests (1 to {self.CHUNK})")
        self.cfg, self.w, self.lora, self.n = cfg, w, lora, requests
        self.heads, self.kv_heads, self.hd = cfg.attn_q_heads, cfg.attn_kv_heads, cfg.head_dim
        self.max_pages = -(-max_rows // page_rows)
        self.max_rows = self.max_pages * page_rows
        n_seqs = requests + 1                                   # sequence 0 is the prompt, request i is sequence i + 1
        z = R.DeviceBuffer.zeros
        page = self.kv_heads * page_rows * self.hd * 2
        self.table, self.lens, self.ref = z(4 * n_seqs * self.max_pages), z(4 * n_seqs), z(4 * n_pages)
        self.data = z(2 * n_pages * page)
        nb = pages.scratch_bytes(n_pages, n_seqs)
        self.pool_scratch = R.DeviceBuffer(nb)
        self.pool = pages.PagePool(base=self.data.ptr, n_planes=2, n_pages=n_pages, heads=self.kv_heads, page_rows=page_rows, row_bytes=2 * self.hd,
                                   n_seqs=n_seqs, max_pages=self.max_pages, ref=self.ref.ptr, table=self.table.ptr, lens=self.lens.ptr,
                                   scratch=self.pool_scratch.ptr, scratch_bytes=nb)
        cos_t, sin_t = ops.rope_tables(self.max_rows, cfg.rot_dim, cfg.rope_theta)
        self.cos, self.sin = R.DeviceBuffer.from_numpy(cos_t), R.DeviceBuffer.from_numpy(sin_t)
        H, c, q = cfg.hidden, self.CHUNK, self.heads * self.hd
        self.xn, self.xq = R.DeviceBuffer(c * H * 2), R.DeviceBuffer(c * H // 32 * 36)
        self.qg, self.k, self.v = R.DeviceBuffer(c * 2 * q * 2), R.DeviceBuffer(c * self.kv_heads * self.hd * 2), R.DeviceBuffer(c * self.kv_heads * self.hd * 2)
        self.att, self.attq, self.out = R.DeviceBuffer(c * q * 2), R.DeviceBuffer(c * q // 32 * 36), R.DeviceBuffer(c * H * 2)
        self.ok, self.map, self.used = z(4 * n_seqs), R.DeviceBuffer(4 * n_pages), R.DeviceBuffer(4)
        nb = ops.lora_scratch_bytes(H, c, lora["rank"], 3)
        self.lora_scratch, self.lora_bytes = R.DeviceBuffer(nb), nb
        self.att_scratch, self.att_bytes = R.DeviceBuffer(16), 16
        self.lists = {k: R.DeviceBuffer(4 * c) for k in ("seqs", "src", "add", "ids", "new", "parent", "token", "target")}
        # a step of drafted trees: its maps, and what stays
        self.b_table, self.b_lens, self.b_count = R.DeviceBuffer(4 * requests * self.max_pages), R.DeviceBuffer(4 * requests), R.DeviceBuffer(4 * requests)
        self.b_pos, self.b_slot, self.b_mask = R.DeviceBuffer(4 * c), R.DeviceBuffer(4 * c), R.DeviceBuffer(8 * c)
        self.path, self.n_path, self.next = R.DeviceBuffer(4 * c), R.DeviceBuffer(4 * requests), R.DeviceBuffer(4 * requests)
        self.nodes = 0      # of the last step's trees
        self.prompt_rows = 0
        self.active = np.zeros(requests, bool)

    def _list(self, name: str, values: Sequence[int]) -> int:
        self.lists[name].upload(np.asarray(values, np.int32))
        return self.lists[name].ptr

    def _check_requests(self, requests: Sequence[int]) -> None:
        for r in requests:
            if not 0 <= r < self.n:
                raise IndexError(f"request {r} of {self.n}")

    def _no_trees(self) -> None:
        if self.nodes:
            raise RuntimeError("the rows of drafted trees are in the cache: keep() comes first")

    def _layer(self, x: int, cols: int, B: int, T: int, first_seq: int, n_new: int, ids: Sequence[int], prefix: int,
               tree: bool = False) -> int:
        """x bf16 [cols][H] of B sequences from first_seq on, T columns each -> out bf16 [cols][H] (device pointer).  tree: of the requests, by the maps of the
        step's trees"""
        cfg, w, lo, H, hd = self.cfg, self.w, self.lora, self.cfg.hidden, self.hd
        q_rows, kv_rows = self.heads * 2 * hd, self.kv_heads * hd
        ops.rmsnorm(x, w["ln"].ptr, H, cols, self.xn.ptr, cfg.eps)
        ops.quant_q8_1(self.xn.ptr, H, cols, self.xq.ptr, bf16=True)
        ops.gemv(self.xq.ptr, H, cols, [ops.gemv_seg(w[n].ptr, rows, o.ptr, R.BK_EPI_BF16) for n, rows, o in
                                        (("q", q_rows, self.qg), ("k", kv_rows, self.k), ("v", kv_rows, self.v))])
        ops.lora(ops.lora_args(x=self.xn.ptr, K=H, B=cols, rank=lo["rank"], n_adapters=lo["n_adapters"], ids=self._list("ids", ids),
                               scratch=self.lora_scratch.ptr, scratch_bytes=self.lora_bytes,
                               segs=[ops.lora_seg(A=lo["A_" + n].ptr, Bm=lo["B_" + n].ptr, n_rows=rows, base=o.ptr, out=o.ptr, bf16=True) for n, rows, o in
                                     (("q", q_rows, self.qg), ("k", kv_rows, self.k), ("v", kv_rows, self.v))]))
        need = (ops.tree_attn_scratch_bytes if tree else ops.paged_attn_scratch_bytes)(B, T, self.heads, self.kv_heads, hd, prefix)
        if need > self.att_bytes:
            R._check(R.cu().bkSync())       # (the smaller one may still be in use)
            self.att_scratch.free()
            self.att_scratch, self.att_bytes = R.DeviceBuffer(need), need
        d = self.pool.desc
        fields = dict(
            qg=self.qg.ptr, k=self.k.ptr, v=self.v.ptr, q_norm_w=w["q_norm"].ptr, k_norm_w=w["k_norm"].ptr, cos_t=self.cos.ptr, sin_t=self.sin.ptr,
            k_pages=self.pool.plane(0), v_pages=self.pool.plane(1), table=self.table.ptr + 4 * first_seq * self.max_pages, lens=self.lens.ptr + 4 * first_seq,
            n_new=n_new, out=self.att.ptr, scratch=self.att_scratch.ptr, scratch_bytes=self.att_bytes, B=B, T=T, Hq=self.heads, Hkv=self.kv_heads, HD=hd,
            rot_half=cfg.rot_dim // 2, n_pages=d.n_pages, page_rows=d.page_rows, max_pages=self.max_pages, prefix_rows=prefix, max_len=self.max_rows,
            scale=1.0 / math.sqrt(hd), eps=cfg.eps, fused_norm_rope=1)
        if tree:
            fields.update(table=self.b_table.ptr, lens=self.b_lens.ptr, pos=self.b_pos.ptr, slot=self.b_slot.ptr, mask=self.b_mask.ptr, mask_words=2)
            ops.tree_attn(ops.tree_attn_args(**fields))
        else:
            ops.paged_attn(ops.paged_attn_args(**fields))
        ops.quant_q8_1(self.att.ptr, self.heads * hd, cols, self.attq.ptr, bf16=True)
        ops.gemv(self.attq.ptr, self.heads * hd, cols, [ops.gemv_seg(w["o"].ptr, H, self.out.ptr, R.BK_EPI_ADD_BF16, residual=x)])
        return self.out.ptr

    def prompt(self, x: int, rows: int, adapter: int = -1) -> None:
        """The prompt's rows x bf16 [rows][H] into sequence 0.  Waits for each chunk's room; where the pool has none left, the chunks before are
        the prompt and RuntimeError says how many rows that is.  Only while no request is active: the requests' steps read the prompt's rows as
        common ones, and those that have begun would not have the new ones."""
        self._no_trees()
        if self.active.any():
            raise RuntimeError(f"the prompt cannot grow behind {int(self.active.sum())} active requests")
        for at in range(0, rows, self.CHUNK):
            n = min(self.CHUNK, rows - at)
            self.pool.grow(self._list("seqs", [0]), self._list("add", [n]), 1, self.ok.ptr)
            if not self.ok.download(np.int32, (1,))[0]:
                raise RuntimeError(f"no room for the prompt: {at} of {rows} rows are in")
            self._layer(x + at * self.cfg.hidden * 2, n, 1, n, 0, 0, [adapter] * n, 0)
            self.prompt_rows += n

    def fork(self, requests: Sequence[int]) -> np.ndarray:
        """These requests begin behind the prompt.  Waits for the pool's answer: which of them were served (a prompt that ends inside a page takes
        a page for each); the others stay as they were."""
        self._no_trees()
        self._check_requests(requests)
        n = len(requests)
        self.pool.fork(self._list("src", [0] * n), self._list("seqs", [r + 1 for r in requests]), n, self.ok.ptr)
        served = self.ok.download(np.int32, (n,)) != 0
        self.active[np.asarray(requests, np.int64)[served]] = True
        return served

    def step(self, x: int, adapters: Sequence[int], share: bool = True) -> int:
        """One token of every active request: x bf16 [requests][H] -> out bf16 [requests][H] (rows of others: what the residual gives).
        ``ok`` (int32 [requests], on the device) says who had room.  A request without room has no token in this step: its ok is its number of new
        tokens, so nothing is stored for it (the row before its next one may be the prompt's, which all share).  An inactive one has no rows."""
        if len(adapters) != self.n:
            raise ValueError(f"{len(adapters)} adapters for {self.n} requests")
        self._no_trees()
        new = self.active.astype(np.int32)
        self.pool.grow(self._list("seqs", np.arange(1, self.n + 1)), self._list("add", new), self.n, self.ok.ptr)
        return self._layer(x, self.n, self.n, 1, 1, self.ok.ptr, adapters, self.prompt_rows if share and new[0] else 0)

    def draft(self, x: int, parent: np.ndarray, adapters: Sequence[int], n_new: Sequence[int] | None = None, share: bool = True) -> int:
        """A tree of up to T drafted tokens of every active request: x bf16 [T * requests][H], row t * requests + i is node t of request i, as parent int
        [T][requests] (node 0 is the last certain token, its parent -1) -> out bf16 of the same rows.  n_new: nodes of each request (all T).  A
        request without room has no nodes in this step; ``b_count`` (int32 [requests], on the device) says how many each has.  ``keep`` comes next."""
        parent = np.ascontiguousarray(parent, np.int32)
        T = len(parent)
        if parent.shape != (T, self.n) or not 1 <= T * self.n <= self.CHUNK or len(adapters) != self.n or (n_new is not None and len(n_new) != self.n):
            raise ValueError(f"trees {parent.shape} and {len(adapters)} adapters for {self.n} requests ({self.CHUNK} nodes in all)")
        new = np.where(self.active, T if n_new is None else np.asarray(n_new), 0).astype(np.int32)
        if (new < 0).any() or (new > T).any():
            raise ValueError(f"{new.tolist()} nodes of trees of up to {T}")
        self._no_trees()
        seqs = self._list("seqs", np.arange(1, self.n + 1))
        self.pool.grow(seqs, self._list("new", new), self.n, self.ok.ptr)
        self.pool.batch(seqs, self.n, T=T, n_new=self.lists["new"].ptr, parent=self._list("parent", parent.reshape(-1)), table=self.b_table.ptr, lens=self.b_lens.ptr,
                        pos=self.b_pos.ptr, slot=self.b_slot.ptr, mask=self.b_mask.ptr, mask_words=2, ok=self.ok.ptr, count=self.b_count.ptr)
        self.nodes = T
        return self._layer(x, T * self.n, self.n, T, 1, self.b_count.ptr, [a for _ in range(T) for a in adapters], self.prompt_rows if share and new[0] else 0, tree=True)

    def keep(self, token: np.ndarray, target: int, values: bool = False) -> tuple[np.ndarray, np.ndarray]:
        """Of the trees of ``draft``, whose tokens are token int [T][requests], the paths that agree with target (device int32 [T * requests], the model's token after each
        node) stay.  values: the logits of those tokens lie behind them (f32 [T * requests]), and one of -inf is no token.  Waits for the answer: (how many nodes of each request stayed, the
        token that follows them, -1 where there is none); 0 and -1 for requests without nodes."""
        if not self.nodes:
            raise RuntimeError("no drafted trees")
        token = np.ascontiguousarray(token, np.int32)
        if token.shape != (self.nodes, self.n):
            raise ValueError(f"tokens {token.shape} of {self.nodes} nodes for {self.n} requests")
        self.pool.commit(self._list("seqs", np.arange(1, self.n + 1)), self.n, T=self.nodes, n_new=self.b_count.ptr, parent=self.lists["parent"].ptr,
                         token=self._list("token", token.reshape(-1)), target=target, path=self.path.ptr, n_path=self.n_path.ptr, next=self.next.ptr, values=values)
        self.nodes = 0
        return self.n_path.download(np.int32, (self.n,)), self.next.download(np.int32, (self.n,))

    def drop(self, requests: Sequence[int]) -> None:
        self._no_trees()
        self._check_requests(requests)
        self.pool.free(self._list("seqs", [r + 1 for r in requests]), len(requests))
        self.active[list(requests)] = False

    def compact(self) -> None:
        self.pool.compact(self.table.ptr, self.ref.ptr, self.map.ptr, self.used.ptr)


def random_layer(cfg: ModelConfig, rank: int = 8, n_adapters: int = 3, seed: int = 0) -> tuple[dict, dict]:
    """Device buffers of a layer with random weights, and of adapters."""
    rng = synth.rng_for(seed, 71)
    H, hd = cfg.hidden, cfg.head_dim
    q, kv = cfg.attn_q_heads * hd, cfg.attn_kv_heads * hd
    w = {}
    for name, rows, K in (("q", 2 * q, H), ("k", kv, H), ("v", kv, H), ("o", H, q)):
        x = R.DeviceBuffer.from_numpy(rng.normal(0, 1 / math.sqrt(K), (rows, K)).astype(np.float32))
        w[name] = R.DeviceBuffer(rows * K // 256 * 144)
        ops.quantize_q4k(x.ptr, rows, K, w[name].ptr)
        R._check(R.cu().bkSync())
        x.free()
    for name, n in (("ln", H), ("q_norm", hd), ("k_norm", hd)):
        w[name] = R.DeviceBuffer.from_numpy(synth.normal_bf16(rng, (n,), 0.02))
    lora = {"rank": rank, "n_adapters": n_adapters}
    for name, rows in (("q", 2 * q), ("k", kv), ("v", kv)):
        lora["A_" + name] = R.DeviceBuffer.from_numpy(synth.normal_bf16(rng, (n_adapters, rank, H), 1 / math.sqrt(H)))
        lora["B_" + name] = R.DeviceBuffer.from_numpy(synth.normal_bf16(rng, (n_adapters, rows, rank), 0.3 / math.sqrt(rank)))
    return w, lora


def main() -> None:
    import argparse
    ap = argparse.ArgumentParser(description="an attention layer served to many requests behind one prompt")
    ap.add_argument("--requests", type=int, default=16)
    ap.add_argument("--prompt", type=int, default=500)
    ap.add_argument("--steps", type=int, default=20)
    ap.add_argument("--draft", type=int, default=4, help="nodes of a request's drafted tree")
    a = ap.parse_args()
    cfg = CONFIG_TINY
    w, lora = random_layer(cfg)
    half = max(1, (a.steps - 2) // 2)
    nodes = max(1, min(a.draft, SharedPrompt.CHUNK // max(1, a.requests)))
    rows = a.prompt + 2 * (1 + half) + nodes * (1 + half) + 1    # (both ways of reading the prompt and trees, each with a step ahead of the timed ones, and one at the end)
    layer = SharedPrompt(cfg, w, lora, a.requests, rows, n_pages=-(-a.prompt // 16) + a.requests * (-(-rows // 16) - a.prompt // 16))
    rng = synth.rng_for(1, 72)
    x = R.DeviceBuffer.from_numpy(synth.normal_bf16(rng, (max(a.prompt, a.requests * nodes), cfg.hidden)))
    layer.prompt(x.ptr, a.prompt)
    layer.fork(range(a.requests))
    adapters = [i % (lora["n_adapters"] + 1) - 1 for i in range(a.requests)]
    for share in (False, True):
        layer.step(x.ptr, adapters, share)      # warm
        e0, e1 = R.Event().record(), R.Event()
        for _ in range(half):
            layer.step(x.ptr, adapters, share)
        e1.record().synchronize()
        print(f"{a.requests} requests behind {a.prompt} rows, prompt {'once for all' if share else 'by every request'}: {e0.elapsed_ms(e1) * 1e3 / half:.1f} us a step, the waits for its lists among them")
    # trees: a chain that the model agrees with half way, then one branch
    parent = np.tile(np.array([max(t - 1, -1) for t in range(nodes)], np.int32)[:, None], (1, a.requests))
    parent[nodes - 1] = 0 if nodes > 1 else -1
    token = np.arange(nodes * a.requests, dtype=np.int32).reshape(nodes, a.requests)
    agreed = np.full_like(token, -1)
    agreed[:nodes // 2] = token[1:nodes // 2 + 1]
    target = R.DeviceBuffer.from_numpy(agreed)
    kept = 0
    for i in range(1 + half):
        if i == 1:
            e0, e1 = R.Event().record(), R.Event()
        layer.draft(x.ptr, parent, adapters)
        kept += int(layer.keep(token, target.ptr)[0].sum())
    if half:
        e1.record().synchronize()
        print(f"trees of {nodes} drafted tokens: {e0.elapsed_ms(e1) * 1e3 / half:.1f} us a step, {kept / (1 + half) / a.requests:.1f} rows of a request stay")
    layer.drop(range(0, a.requests, 2))
    layer.compact()
    layer.step(x.ptr, adapters, False)
    R._check(R.cu().bkSync())
    print("half of the requests dropped, pool compacted:", int(layer.used.download(np.int32, (1,))[0]), "pages in use")


if __name__ == "__main__":
    main()
