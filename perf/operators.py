"""Serving many requests from one paged key/value cache, as measurable cases.

``kind`` names the operator that one pass goes through:

  attn     append the new rows and attend over pages; the rows that all sequences share are computed once   (bkPagedAttn)
  beam     drop the old beams, fork the kept ones, make room for their next rows               (bkPagesFree / Fork / Grow)
  compact  move the used pages of a fragmented pool to its front and rewrite the tables                   (bkPagesCompact)
  copy     pages of one pool into another                                                                    (bkPagesCopy)
  lora     low-rank adapters, one per request, added to a shared projection's output                              (bkLora)

With ``own`` false ``run`` computes the same with elementary torch operations in 32 bits.  Head counts, widths and layer counts are
those of the two benchmark models and of the small test model, or log-uniform between them.
"""
import math
import random

import torch

own = False

ROT = 32   # rotary pairs of a head: the first 2 * ROT values
EPS = 1e-6


def listed():
    return [
        # one sequence of a chat on pages, nothing shared: the smallest attention call, latency counts
        {"name": "attn_b1_300", "kind": "attn", "B": 1, "T": 1, "prefix": 0, "suffix": 300, "Hq": 16, "Hkv": 2, "HD": 256, "page": 16},
        # a server batch behind one long system prompt, the 24-layer model's heads
        {"name": "attn_b32_p8192", "kind": "attn", "B": 32, "T": 1, "prefix": 8192, "suffix": 512, "Hq": 16, "Hkv": 2, "HD": 256, "page": 64},
        # the largest: 64 requests about one long document, the 64-layer model's heads
        {"name": "attn_b64_p32768", "kind": "attn", "B": 64, "T": 1, "prefix": 32768, "suffix": 1024, "Hq": 24, "Hkv": 4, "HD": 256, "page": 64},
        # pieces of prompts (up to 16 tokens, ragged) after a common preamble that ends inside a page, narrow heads
        {"name": "attn_b4_t16", "kind": "attn", "B": 4, "T": 16, "prefix": 1000, "suffix": 333, "Hq": 24, "Hkv": 4, "HD": 128, "page": 32},
        # four beams of one short answer: metadata and a few rows
        {"name": "beam_1x4", "kind": "beam", "parents": 1, "children": 4, "len": 100, "page": 16, "planes": 12, "heads": 2, "HD": 256},
        # eight beams of each of eight requests, sixteen planes of four heads
        {"name": "beam_8x8", "kind": "beam", "parents": 8, "children": 64, "len": 4096, "page": 64, "planes": 16, "heads": 4, "HD": 256},
        # a small fragmented pool
        {"name": "compact_64", "kind": "compact", "pages": 64, "used": 0.5, "seqs": 5, "planes": 2, "page": 16, "heads": 1, "HD": 256},
        # the pool of the 24-layer model (six attention layers) after many requests have come and gone
        {"name": "compact_2048", "kind": "compact", "pages": 2048, "used": 0.6, "seqs": 40, "planes": 12, "page": 64, "heads": 2, "HD": 256},
        # one page of every layer
        {"name": "copy_1", "kind": "copy", "n": 1, "from": 40, "to": 50, "planes": 12, "page": 16, "heads": 2, "HD": 256},
        # the cache moves into a larger pool
        {"name": "copy_500", "kind": "copy", "n": 500, "from": 512, "to": 700, "planes": 12, "page": 64, "heads": 2, "HD": 256},
        # one request's adapter on the query projection of the 24-layer model
        {"name": "lora_b1", "kind": "lora", "B": 1, "K": 2048, "rows": "8192", "rank": 8, "adapters": 4, "f32": False},
        # a full batch of tenants on gate and up of the 64-layer model
        {"name": "lora_b64", "kind": "lora", "B": 64, "K": 5120, "rows": "17408,17408", "rank": 32, "adapters": 48, "f32": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    kind = rng.choice(["attn", "attn", "attn", "beam", "compact", "copy", "lora", "lora"])
    if kind == "attn":
        hq, hkv = rng.choice([(16, 2), (24, 4), (4, 1)])
        b = _log(rng, 1, 64)
        t = _log(rng, 1, 64 // b) if rng.random() < 0.5 else 1
        return {"kind": kind, "B": b, "T": t, "prefix": _log(rng, 16, 16384) if rng.random() < 0.8 else 0, "suffix": t + _log(rng, 1, 1000), "Hq": hq,
                "Hkv": hkv, "HD": rng.choice([256, 256, 128]), "page": rng.choice([16, 32, 64, 128])}
    planes, heads = rng.choice([(12, 2), (16, 4), (2, 1)])
    page = rng.choice([16, 32, 64])
    if kind == "beam":
        parents = _log(rng, 1, 8)
        return {"kind": kind, "parents": parents, "children": _log(rng, 1, 64), "len": _log(rng, 1, 4096), "page": page, "planes": planes, "heads": heads,
                "HD": 256}
    if kind == "compact":
        return {"kind": kind, "pages": _log(rng, 16, 600), "used": round(rng.uniform(0.1, 0.95), 2), "seqs": _log(rng, 1, 40), "planes": planes,
                "page": page, "heads": heads, "HD": 256}
    if kind == "copy":
        n = _log(rng, 1, 180)
        return {"kind": kind, "n": n, "from": n + rng.randint(0, 50), "to": n + rng.randint(0, 100), "planes": planes, "page": page, "heads": heads, "HD": 256}
    b = _log(rng, 1, 64)
    rows = [8 * _log(rng, 1, 2176) for _ in range(rng.choice([1, 1, 2, 3]))]
    rows = [r + 8 if r == 3072 else r for r in rows]
    k = 256 * _log(rng, 1, 20)
    return {"kind": kind, "B": b, "K": k + 256 if k == 3072 else k, "rows": ",".join(map(str, rows)), "rank": rng.choice([8, 16, 16, 32, 64]),
            "adapters": _log(rng, 1, 48), "f32": rng.random() < 0.5}


# ---- what follows from a case alone ---------------------------------------------------

def _attn_lens(c):
    """(rows of each sequence with its new ones, new tokens of each sequence)"""
    new = [max(1, c["T"] - (b * 3) % c["T"]) for b in range(c["B"])]
    own_rows = [c["suffix"] if b == 0 else 1 + (b * 2654435761 >> 7) % c["suffix"] for b in range(c["B"])]
    return [c["prefix"] + max(s, n) for s, n in zip(own_rows, new)], new


def _lora_ids(c):
    return [-1 if b % 8 == 5 else (b * 5) % c["adapters"] for b in range(c["B"])]


def _lora_rows(c):
    return [int(r) for r in c["rows"].split(",")]


def _beam_lens(c):
    return [max(1, c["len"] - (p * 37) % c["page"]) for p in range(c["parents"])]


def _pages(rows, page):
    return (rows + page - 1) // page


def _compact_used(c):
    return max(1, int(c["pages"] * c["used"]))


# ---- inputs ------------------------------------------------------------------------

def _gen(seed, stream):
    g = torch.Generator(device="cuda")
    g.manual_seed((int(seed) * 1000003 + stream) & 0x7FFFFFFF)
    return g


def _bf16(shape, g, std=1.0):
    return (torch.randn(shape, device="cuda", generator=g) * std).bfloat16()


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _pool(planes, pages, c, g):
    """Pool contents as 16-bit patterns of any value: [plane][page][head][row][HD]"""
    n = planes * pages * c["heads"] * c["page"] * c["HD"]
    return torch.randint(-2**31, 2**31, ((n + 1) // 2,), dtype=torch.int32, device="cuda", generator=g).view(torch.int16)[:n].view(
        planes, pages, c["heads"], c["page"], c["HD"])


def _handle(s, name, pool, ref, table, lens):
    """The pool as a user of the framework holds it."""
    from bunker_b200.pages import PagePool
    planes, pages, heads, rows, hd = pool.shape
    s[name] = PagePool(base=pool.data_ptr(), n_planes=planes, n_pages=pages, heads=heads, page_rows=rows, row_bytes=2 * hd, n_seqs=table.shape[0],
                       max_pages=table.shape[1], ref=ref.data_ptr(), table=table.data_ptr(), lens=lens.data_ptr(),
                       scratch=s["scratch"].data_ptr(), scratch_bytes=s["scratch"].numel())


def prepare(case, seed):
    s = {"case": dict(case), "seed": int(seed)}
    g = _gen(seed, 7)
    {"attn": _prepare_attn, "beam": _prepare_beam, "compact": _prepare_compact, "copy": _prepare_copy, "lora": _prepare_lora}[case["kind"]](s, case, g)
    torch.cuda.synchronize()
    return s


def _prepare_attn(s, c, g):
    B, T, P, Hq, Hkv, HD, page = c["B"], c["T"], c["prefix"], c["Hq"], c["Hkv"], c["HD"], c["page"]
    lens, new = _attn_lens(c)
    shared = P // page
    tail = [_pages(n, page) - shared for n in lens]      # pages of a sequence behind the shared ones
    n_pages = shared + sum(tail) + 7
    ids = torch.randperm(n_pages, device="cuda", generator=g, dtype=torch.int32)
    max_pages = shared + max(tail)
    table = torch.full((B, max_pages), -1, dtype=torch.int32, device="cuda")
    table[:, :shared] = ids[:shared]
    at = shared
    for b in range(B):
        table[b, shared:shared + tail[b]] = ids[at:at + tail[b]]
        at += tail[b]
    k_pages, v_pages = _bf16((n_pages, Hkv, page, HD), g), _bf16((n_pages, Hkv, page, HD), g)
    if P % page:    # the page that the preamble ends in: every sequence has its copy of those rows
        own_page = table[:, shared].long()
        k_pages[own_page, :, :P % page] = k_pages[own_page[0], :, :P % page].clone()
        v_pages[own_page, :, :P % page] = v_pages[own_page[0], :, :P % page].clone()
    max_len = max_pages * page
    ang = torch.outer(torch.arange(max_len, device="cuda", dtype=torch.float64),
                      1e7 ** (-torch.arange(ROT, device="cuda", dtype=torch.float64) / ROT))
    s.update(qg=_bf16((T * B, Hq, 2 * HD), g), k=_bf16((T * B, Hkv, HD), g), v=_bf16((T * B, Hkv, HD), g), q_norm_w=_bf16((HD,), g, 0.02),
             k_norm_w=_bf16((HD,), g, 0.02), cos=ang.cos().float(), sin=ang.sin().float(), k_pages=k_pages, v_pages=v_pages, table=table, len=_i32(lens),
             new=_i32(new), out=torch.zeros((T * B, Hq * HD), dtype=torch.bfloat16, device="cuda"), scale=1.0 / math.sqrt(HD))
    if own:
        from bunker_b200 import ops, runtime as R
        R.cu(0)
        s["scratch"] = torch.zeros(ops.paged_attn_scratch_bytes(B, T, Hq, Hkv, HD, P), dtype=torch.uint8, device="cuda")
        s["args"] = ops.paged_attn_args(
            qg=s["qg"].data_ptr(), k=s["k"].data_ptr(), v=s["v"].data_ptr(), q_norm_w=s["q_norm_w"].data_ptr(), k_norm_w=s["k_norm_w"].data_ptr(),
            cos_t=s["cos"].data_ptr(), sin_t=s["sin"].data_ptr(), k_pages=k_pages.data_ptr(), v_pages=v_pages.data_ptr(), table=table.data_ptr(),
            len=s["len"].data_ptr(), n_new=s["new"].data_ptr(), out=s["out"].data_ptr(), scratch=s["scratch"].data_ptr(),
            scratch_bytes=s["scratch"].numel(), B=B, T=T, Hq=Hq, Hkv=Hkv, HD=HD, rot_half=ROT, n_pages=n_pages, page_rows=page, max_pages=max_pages,
            prefix_rows=P, max_len=max_len, scale=s["scale"], eps=EPS, fused_norm_rope=1)


def _prepare_beam(s, c, g):
    parents, children, page = c["parents"], c["children"], c["page"]
    lens = _beam_lens(c)
    held = [_pages(n, page) for n in lens]
    max_pages = max(held) + 1
    n_pages = sum(held) + 2 * children + 20
    ids = torch.randperm(n_pages, device="cuda", generator=g, dtype=torch.int32)
    n_seqs = parents + children
    table = torch.full((n_seqs, max_pages), -1, dtype=torch.int32, device="cuda")
    at = 0
    for p in range(parents):
        table[p, :held[p]] = ids[at:at + held[p]]
        at += held[p]
    ref = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
    ref[ids[:at].long()] = 1
    s.update(pool=_pool(c["planes"], n_pages, c, g), table=table, ref=ref, len=_i32(lens + [0] * children),
             src=_i32([i % parents for i in range(children)]), dst=_i32([parents + i for i in range(children)]),
             add=_i32([1 + i % 3 for i in range(children)]), ok=torch.zeros((2, children), dtype=torch.int32, device="cuda"))
    if own:
        from bunker_b200 import pages, runtime as R
        R.cu(0)
        s["scratch"] = torch.zeros(pages.scratch_bytes(n_pages, n_seqs), dtype=torch.uint8, device="cuda")
        _handle(s, "handle", s["pool"], ref, table, s["len"])


def _prepare_compact(s, c, g):
    n_pages, seqs, used = c["pages"], c["seqs"], _compact_used(c)
    ids = torch.randperm(n_pages, device="cuda", generator=g, dtype=torch.int32)[:used]
    common = min(used - 1, 4)                                  # pages that all sequences share
    each = -(-(used - common) // seqs)
    table = torch.full((seqs, common + each + 1), -1, dtype=torch.int32, device="cuda")
    table[:, :common] = ids[:common]
    rest = torch.full((seqs * each,), -1, dtype=torch.int32, device="cuda")
    rest[:used - common] = ids[common:]
    table[:, common:common + each] = rest.view(each, seqs).t()
    ref = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
    ref.scatter_add_(0, table[table >= 0].long(), torch.ones_like(table[table >= 0]))
    s.update(pool=_pool(c["planes"], n_pages, c, g), table=table, ref=ref, len=((table >= 0).sum(1) * c["page"]).int(), table_out=torch.zeros_like(table),
             ref_out=torch.zeros_like(ref), map=torch.zeros_like(ref), used=_i32([0]))
    if own:
        from bunker_b200 import pages, runtime as R
        R.cu(0)
        s["scratch"] = torch.zeros(pages.scratch_bytes(n_pages, seqs), dtype=torch.uint8, device="cuda")
        _handle(s, "handle", s["pool"], ref, table, s["len"])


def _prepare_copy(s, c, g):
    a, b = _pool(c["planes"], c["from"], c, g), _pool(c["planes"], c["to"], c, g)
    src = torch.randperm(c["from"], device="cuda", generator=g, dtype=torch.int32)[:c["n"]]
    dst = torch.randperm(c["to"], device="cuda", generator=g, dtype=torch.int32)[:c["n"]]
    s.update(a=a, b=b, src=src.clone(), dst=dst.clone())
    if own:
        from bunker_b200 import pages, runtime as R
        R.cu(0)
        s["scratch"] = torch.zeros(pages.scratch_bytes(max(c["from"], c["to"]), 1), dtype=torch.uint8, device="cuda")
        for name, pool in (("a_handle", a), ("b_handle", b)):
            meta = [torch.zeros(pool.shape[1], dtype=torch.int32, device="cuda"), torch.zeros((1, 1), dtype=torch.int32, device="cuda"), _i32([0])]
            s[name + "_meta"] = meta
            _handle(s, name, pool, *meta)


def _prepare_lora(s, c, g):
    B, K, r, rows = c["B"], c["K"], c["rank"], _lora_rows(c)
    kind = torch.float32 if c["f32"] else torch.bfloat16
    s.update(x=_bf16((B, K), g), ids=_i32(_lora_ids(c)), scale=torch.rand(c["adapters"], device="cuda", generator=g) + 0.5,
             A=[_bf16((c["adapters"], r, K), g, 1 / math.sqrt(K)) for _ in rows], Bm=[_bf16((c["adapters"], n, r), g, 1 / math.sqrt(r)) for n in rows],
             base=[torch.randn((B, n), device="cuda", generator=g).to(kind) for n in rows], out=[torch.zeros((B, n), dtype=kind, device="cuda") for n in rows])
    if own:
        from bunker_b200 import ops, runtime as R
        R.cu(0)
        s["scratch"] = torch.zeros(ops.lora_scratch_bytes(K, B, r, len(rows)), dtype=torch.uint8, device="cuda")
        s["args"] = ops.lora_args(
            x=s["x"].data_ptr(), K=K, B=B, rank=r, n_adapters=c["adapters"], ids=s["ids"].data_ptr(), scale=s["scale"].data_ptr(),
            scratch=s["scratch"].data_ptr(), scratch_bytes=s["scratch"].numel(),
            segs=[ops.lora_seg(A=a.data_ptr(), Bm=m.data_ptr(), n_rows=n, base=y.data_ptr(), out=o.data_ptr(), bf16=not c["f32"])
                  for a, m, n, y, o in zip(s["A"], s["Bm"], rows, s["base"], s["out"])])


# ---- one pass ----------------------------------------------------------------------

def run(state):
    s, c = state, state["case"]
    return {"attn": _run_attn, "beam": _run_beam, "compact": _run_compact, "copy": _run_copy, "lora": _run_lora}[c["kind"]](s, c)


def _norm_rope(x, w, cos, sin):
    """x [n][heads][HD] in 32 bits, cos and sin [n][ROT]: head RMSNorm times 1 + w, then the rotation of the first 2 * ROT values"""
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * (1.0 + w)
    a, b, c, s = y[..., :ROT], y[..., ROT:2 * ROT], cos[:, None], sin[:, None]
    return torch.cat([a * c - b * s, b * c + a * s, y[..., 2 * ROT:]], -1)


def _run_attn(s, c):
    if own:
        from bunker_b200 import ops
        ops.paged_attn(s["args"])
        return {"out": s["out"], "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    B, T, P, Hq, Hkv, HD, page = c["B"], c["T"], c["prefix"], c["Hq"], c["Hkv"], c["HD"], c["page"]
    G, shared = Hq // Hkv, P // page
    t = torch.arange(T, device="cuda")[:, None]
    pos = (s["len"] - s["new"])[None] + t                          # [T][B]
    there = (t < s["new"][None]).reshape(-1)
    pos = torch.where(there, pos.reshape(-1), 0)
    cos, sin = s["cos"][pos], s["sin"][pos]
    q = _norm_rope(s["qg"][..., :HD].float(), s["q_norm_w"].float(), cos, sin)
    k = _norm_rope(s["k"].float(), s["k_norm_w"].float(), cos, sin)
    # append
    seq = torch.arange(B, device="cuda").repeat(T)[there]
    at = pos[there]
    pg, row = s["table"][seq, at // page].long(), at % page
    s["k_pages"][pg, :, row] = k[there].bfloat16()
    s["v_pages"][pg, :, row] = s["v"][there]
    # rows of the common pages once, the others by sequence
    qr = q.view(T, B, Hkv, G, HD)
    pre = s["table"][0, :shared].long()
    kp = s["k_pages"][pre].float().permute(1, 0, 2, 3).reshape(Hkv, shared * page, HD)
    vp = s["v_pages"][pre].float().permute(1, 0, 2, 3).reshape(Hkv, shared * page, HD)
    sp = torch.matmul(qr.permute(2, 0, 1, 3, 4).reshape(Hkv, T * B * G, HD), kp.transpose(1, 2)) * s["scale"]
    rest = s["table"][:, shared:].clamp_min(0).long()
    n = rest.shape[1] * page
    ks = s["k_pages"][rest].float().permute(0, 2, 1, 3, 4).reshape(B, Hkv, n, HD)
    vs = s["v_pages"][rest].float().permute(0, 2, 1, 3, 4).reshape(B, Hkv, n, HD)
    ss = torch.matmul(qr.permute(1, 2, 0, 3, 4).reshape(B, Hkv, T * G, HD), ks.transpose(2, 3)) * s["scale"]
    key = shared * page + torch.arange(n, device="cuda")
    seen = key <= pos.view(T, B).t()[:, :, None]                   # [B][T][n]
    ss = ss.view(B, Hkv, T, G, n).masked_fill(~seen[:, None, :, None], float("-inf"))
    sp = sp.view(Hkv, T, B, G, shared * page).permute(2, 0, 1, 3, 4)   # [B][Hkv][T][G][keys]
    m = ss.amax(-1, keepdim=True)
    if shared:
        m = torch.maximum(m, sp.amax(-1, keepdim=True))
    ep, es = torch.exp(sp - m), torch.exp(ss - m)
    z = ep.sum(-1, keepdim=True) + es.sum(-1, keepdim=True)
    op = torch.matmul(ep.permute(1, 2, 0, 3, 4).reshape(Hkv, T * B * G, shared * page), vp).view(Hkv, T, B, G, HD).permute(2, 0, 1, 3, 4)
    os = torch.matmul(es.reshape(B, Hkv, T * G, n), vs).view(B, Hkv, T, G, HD)
    o = ((op + os) / z).permute(2, 0, 1, 3, 4).reshape(T * B, Hq, HD)
    o = o * torch.sigmoid(s["qg"][..., HD:].float())
    s["out"].copy_(torch.where(there[:, None], o.reshape(T * B, Hq * HD), 0.0))
    return {"out": s["out"], "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _run_beam(s, c):
    if own:
        n = c["children"]
        s["handle"].free(s["dst"].data_ptr(), n)
        s["handle"].fork(s["src"].data_ptr(), s["dst"].data_ptr(), n, s["ok"].data_ptr())
        s["handle"].grow(s["dst"].data_ptr(), s["add"].data_ptr(), n, s["ok"].data_ptr() + 4 * n)
        return {k: s[k] for k in ("pool", "table", "ref", "len", "ok")}
    page, table, ref, lens = c["page"], s["table"], s["ref"], s["len"]
    src, dst = s["src"].long(), s["dst"].long()
    col = torch.arange(table.shape[1], device="cuda")
    # free
    held = (col < ((lens[dst] + page - 1) // page)[:, None])
    gone = table[dst][held].long()
    ref.scatter_add_(0, gone, torch.full_like(gone, -1, dtype=torch.int32))
    table[dst] = torch.where(held, -1, table[dst])
    lens[dst] = 0
    # fork
    n = lens[src]
    part = n % page
    need = (part > 0).int()
    free = torch.nonzero(ref == 0).flatten()
    s["ok"][0] = ((need == 0) | (need.cumsum(0) <= free.numel())).int()
    whole = col < (n // page)[:, None]
    kept = table[src]
    table[dst] = torch.where(whole, kept, -1)
    also = kept[whole].long()
    ref.scatter_add_(0, also, torch.ones_like(also, dtype=torch.int32))
    take = need > 0
    fresh = free[:int(need.sum())]
    ref[fresh] = 1
    last = (n // page).long()
    old = kept[take, last[take]].long()
    table[dst[take], last[take]] = fresh.int()
    filled = torch.arange(page, device="cuda") < part[take][:, None]             # [forks][page]
    f, r = torch.nonzero(filled, as_tuple=True)
    s["pool"][:, fresh[f], :, r] = s["pool"][:, old[f], :, r]
    lens[dst] = n
    # grow
    before, after = (lens[dst] + page - 1) // page, (lens[dst] + s["add"] + page - 1) // page
    need = after - before
    free = torch.nonzero(ref == 0).flatten()
    s["ok"][1] = ((need == 0) | (need.cumsum(0) <= free.numel())).int()
    more = (col >= before[:, None]) & (col < after[:, None])
    i, j = torch.nonzero(more, as_tuple=True)
    fresh = free[:i.numel()]
    table[dst[i], j] = fresh.int()
    ref[fresh] = 1
    lens[dst] = lens[dst] + s["add"]
    return {k: s[k] for k in ("pool", "table", "ref", "len", "ok")}


def _run_compact(s, c):
    if own:
        s["handle"].compact(s["table_out"].data_ptr(), s["ref_out"].data_ptr(), s["map"].data_ptr(), s["used"].data_ptr())
        return {k: s[k] for k in ("pool", "table_out", "ref_out", "map", "used")}
    ref = s["ref"]
    page = torch.arange(ref.numel(), device="cuda")
    held = ref > 0
    n = int(held.sum())
    old, new = torch.nonzero(held & (page >= n)).flatten(), torch.nonzero(~held & (page < n)).flatten()
    s["pool"][:, new] = s["pool"][:, old]
    to = torch.where(held, page, -1).int()
    to[old] = new.int()
    s["map"].copy_(to)
    s["used"].fill_(n)
    s["ref_out"].zero_()
    s["ref_out"][to[held].long()] = ref[held]
    s["table_out"].copy_(torch.where(s["table"] >= 0, to[s["table"].clamp_min(0).long()], -1))
    return {k: s[k] for k in ("pool", "table_out", "ref_out", "map", "used")}


def _run_copy(s, c):
    if own:
        s["a_handle"].copy(s["b_handle"], s["src"].data_ptr(), s["dst"].data_ptr(), c["n"])
    else:
        s["b"][:, s["dst"].long()] = s["a"][:, s["src"].long()]
    return {"pool": s["b"]}


def _run_lora(s, c):
    if own:
        from bunker_b200 import ops
        ops.lora(s["args"])
        return {"out": s["out"]}
    x, a = s["x"].float(), s["ids"].clamp_min(0).long()
    scale = torch.where(s["ids"] >= 0, s["scale"][a], 0.0)[:, None]

    def segment(A, Bm, base, out):
        u = torch.matmul(A[a].float(), x[:, :, None])               # [B][rank][1]
        out.copy_(base.float() + scale * torch.matmul(Bm[a].float(), u).squeeze(-1))
        return out

    return {"out": list(map(segment, s["A"], s["Bm"], s["base"], s["out"]))}


# ---- the definition in 64 bits ---------------------------------------------------------

def exact(case, seed):
    c = case
    if c["kind"] not in ("attn", "lora"):
        return None     # whole numbers and copied patterns
    s = prepare(c, seed)
    if c["kind"] == "lora":
        outs = []
        for A, Bm, base in zip(s["A"], s["Bm"], s["base"]):
            y = base.double()
            for b, a in enumerate(s["ids"].tolist()):
                if a >= 0:
                    y[b] += s["scale"][a].double() * (Bm[a].double() @ (A[a].double() @ s["x"][b].double()))
            outs.append(y)
        return {"out": outs}
    B, T, Hq, Hkv, HD, page = c["B"], c["T"], c["Hq"], c["Hkv"], c["HD"], c["page"]
    lens, new = s["len"].tolist(), s["new"].tolist()
    kp, out = s["k_pages"].double(), torch.zeros((T * B, Hq, HD), dtype=torch.float64, device="cuda")

    def turned(x, w, p):
        y = x / torch.sqrt((x ** 2).sum(-1, keepdim=True) / HD + EPS) * (w.double() + 1)
        c64, s64 = s["cos"][p].double(), s["sin"][p].double()
        z = y.clone()
        z[..., :ROT] = y[..., :ROT] * c64 - y[..., ROT:2 * ROT] * s64
        z[..., ROT:2 * ROT] = y[..., ROT:2 * ROT] * c64 + y[..., :ROT] * s64
        return z

    for b in range(B):
        for t in range(new[b]):
            p = lens[b] - new[b] + t
            kp[s["table"][b, p // page].item(), :, p % page] = turned(s["k"][t * B + b].double(), s["k_norm_w"], p)
            s["v_pages"][s["table"][b, p // page].item(), :, p % page] = s["v"][t * B + b]
    for b in range(B):
        pages = s["table"][b, :_pages(lens[b], page)].long()
        K = kp[pages].transpose(0, 1).reshape(Hkv, -1, HD)
        V = s["v_pages"][pages].double().transpose(0, 1).reshape(Hkv, -1, HD)
        for t in range(new[b]):
            p = lens[b] - new[b] + t
            e = t * B + b
            q = turned(s["qg"][e, :, :HD].double(), s["q_norm_w"], p).view(Hkv, Hq // Hkv, HD)
            w = torch.softmax(q @ K[:, :p + 1].transpose(1, 2) * s["scale"], -1)
            out[e] = (w @ V[:, :p + 1]).reshape(Hq, HD) / (1 + torch.exp(-s["qg"][e, :, HD:].double()))
    return {"out": out.view(T * B, Hq * HD), "k_pages": kp, "v_pages": None}


# ---- what a pass cannot do without ----------------------------------------------------

def work(case):
    c = case
    if c["kind"] == "attn":
        B, T, Hq, Hkv, HD, page = c["B"], c["T"], c["Hq"], c["Hkv"], c["HD"], c["page"]
        lens, new = _attn_lens(c)
        shared = c["prefix"] // page * page
        rows = shared + sum(n - shared for n in lens)
        keys = sum(n * m - m * (m - 1) // 2 for n, m in zip(lens, new))
        return {"bytes": rows * Hkv * HD * 4 + sum(new) * (Hq * 3 + Hkv * 2) * HD * 2, "flops": keys * Hq * HD * 4}
    if c["kind"] == "lora":
        rows, ids = _lora_rows(c), _lora_ids(c)
        distinct, active, size = len(set(ids) - {-1}), sum(a >= 0 for a in ids), 4 if c["f32"] else 2
        return {"bytes": distinct * c["rank"] * sum(c["K"] + n for n in rows) * 2 + c["B"] * (c["K"] * 2 + 2 * sum(rows) * size),
                "flops": 2 * active * c["rank"] * sum(c["K"] + n for n in rows)}
    row = c["heads"] * c["HD"] * 2 * c["planes"]     # one cached position of all planes
    if c["kind"] == "beam":
        lens = _beam_lens(c)
        forked = [i % c["parents"] for i in range(c["children"])]
        meta = 4 * (3 * sum(_pages(lens[p], c["page"]) for p in forked) + 8 * c["children"])
        return {"bytes": row * (sum(lens[p] % c["page"] for p in forked) + sum(lens[p] % c["page"] for p in set(forked))) + meta, "flops": 0}
    if c["kind"] == "compact":
        used = _compact_used(c)
        # of the used pages, scattered at random, this share lies behind the first `used`
        return {"bytes": 2 * row * c["page"] * used * (c["pages"] - used) / c["pages"] + 12 * c["pages"], "flops": 0}
    return {"bytes": 2 * row * c["page"] * c["n"] + 8 * c["n"], "flops": 0}
