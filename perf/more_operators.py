"""Verifying drafted trees of tokens for many requests on one paged cache, as measurable cases.

``kind`` names the operator that one pass goes through, in the order of a step:

  batch    tables, lengths, positions, slots and masks of a list of sequences and their trees    (bkPagesBatch)
  tree     store the trees' rows and attend: the rows before a tree, then a node's ancestors       (bkTreeAttn)
  logits   penalties for repeated tokens, biases and grammar masks on the nodes' logits            (bkAdjustLogits)
  commit   room for the trees, then the longest path that the model agrees with stays              (bkPagesGrow / bkPagesCommit)

With ``own`` false ``run`` computes the same with elementary torch operations in 32 bits.  Head counts, widths, layer counts and
vocabularies are those of the two benchmark models and of the small test model, or log-uniform between them.
"""
import math
import random

import torch

own = False

ROT = 32   # rotary pairs of a head: the first 2 * ROT values
EPS = 1e-6


def listed():
    return [
        # one chat with a short draft: the smallest attention call, latency counts
        {"name": "tree_b1_t8", "kind": "tree", "B": 1, "T": 8, "prefix": 0, "suffix": 300, "Hq": 16, "Hkv": 2, "HD": 256, "page": 16, "fused": True},
        # a server batch behind one long system prompt, drafts of up to 16 nodes, the 24-layer model's heads
        {"name": "tree_b16_t16", "kind": "tree", "B": 16, "T": 16, "prefix": 8192, "suffix": 512, "Hq": 16, "Hkv": 2, "HD": 256, "page": 64, "fused": True},
        # wide trees over ready queries of narrow heads, a common part that ends inside a page
        {"name": "tree_b4_t100", "kind": "tree", "B": 4, "T": 100, "prefix": 1000, "suffix": 3333, "Hq": 24, "Hkv": 4, "HD": 128, "page": 32, "fused": False},
        # the largest: 32 requests with long contexts of their own, full trees, the 64-layer model's heads
        {"name": "tree_b32_t64", "kind": "tree", "B": 32, "T": 64, "prefix": 0, "suffix": 16384, "Hq": 24, "Hkv": 4, "HD": 256, "page": 64, "fused": True},
        # one chat's next token: penalties alone
        {"name": "logits_b1", "kind": "logits", "B": 1, "T": 1, "V": 151936, "history": 700, "bias": 0, "masks": 0, "allow": 1.0},
        # a server batch of single tokens, every second one under a grammar that allows few tokens
        {"name": "logits_b64", "kind": "logits", "B": 64, "T": 1, "V": 151936, "history": 5000, "bias": 40, "masks": 12, "allow": 0.03},
        # all nodes of the trees of sixteen requests, each in its own state of a grammar
        {"name": "logits_b16_t32", "kind": "logits", "B": 16, "T": 32, "V": 151936, "history": 16000, "bias": 300, "masks": 60, "allow": 0.4},
        # one sequence, one token
        {"name": "batch_1", "kind": "batch", "B": 1, "T": 1, "seqs": 7, "len": 300, "page": 16},
        # a full server's trees
        {"name": "batch_256_t64", "kind": "batch", "B": 256, "T": 64, "seqs": 400, "len": 32768, "page": 16},
        # one request's tree, the cache of the small test model
        {"name": "commit_1", "kind": "commit", "B": 1, "T": 8, "len": 100, "page": 16, "planes": 2, "heads": 1, "HD": 256},
        # the 24-layer model's cache (six attention layers)
        {"name": "commit_16_t24", "kind": "commit", "B": 16, "T": 24, "len": 2000, "page": 16, "planes": 12, "heads": 2, "HD": 256},
        # the 64-layer model's cache (sixteen attention layers), a full batch
        {"name": "commit_64_t64", "kind": "commit", "B": 64, "T": 64, "len": 4096, "page": 64, "planes": 32, "heads": 4, "HD": 256},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    kind = rng.choice(["tree", "tree", "tree", "logits", "logits", "batch", "commit", "commit"])
    b = _log(rng, 1, 64)
    t = _log(rng, 1, min(128, 1024 // b))
    if kind == "tree":
        hq, hkv = rng.choice([(16, 2), (24, 4), (4, 1)])
        longest = max(64, (32 * 64 * 24 * 8192) // (2 * b * t * hq))       # the prefix and the longest suffix, which is twice the mean
        return {"kind": kind, "B": b, "T": t, "prefix": _log(rng, 16, min(16384, longest)) if rng.random() < 0.6 else 0,
                "suffix": t + _log(rng, 1, min(16384, longest)), "Hq": hq, "Hkv": hkv, "HD": rng.choice([256, 256, 128]),
                "page": rng.choice([16, 32, 64, 128]), "fused": rng.random() < 0.7}
    if kind == "logits":
        v = rng.choice([151936, 4096, _log(rng, 1000, 160000)])
        t = max(1, min(t, 512 // b, 10**8 // (v * b)))
        return {"kind": kind, "B": b, "T": t, "V": v, "history": _log(rng, 1, 32000), "bias": rng.choice([0, _log(rng, 1, 1000)]),
                "masks": rng.choice([0, _log(rng, 1, 60)]), "allow": round(rng.uniform(0.01, 0.99), 2)}
    page = rng.choice([16, 32, 64])
    if kind == "batch":
        return {"kind": kind, "B": b, "T": t, "seqs": b + rng.randint(0, 100), "len": t + _log(rng, 1, 32768), "page": page}
    planes, heads = rng.choice([(12, 2), (32, 4), (2, 1)])
    t = min(t, 64)
    return {"kind": kind, "B": b, "T": t, "len": t + _log(rng, 1, 2000), "page": page, "planes": planes, "heads": heads, "HD": 256}


# ---- what follows from a case alone ---------------------------------------------------

def _new(c):
    """Nodes of each sequence's tree: 1 to T."""
    return [max(1, c["T"] - (b * 3) % c["T"]) for b in range(c["B"])]


def _parent(b, t):
    """A spine of the likeliest tokens, then branches anywhere."""
    return t - 1 if t < 6 else ((b + 1) * 2654435761 + t * 40503 >> 4) % t


def _parents(c):
    return [[_parent(b, t) for t in range(c["T"])] for b in range(c["B"])]


def _paths(parents):
    """For each sequence and node the node and its ancestors, as bits of an integer."""
    out = []
    for p in parents:
        bits = []
        for t, q in enumerate(p):
            bits.append((bits[q] if q >= 0 else 0) | 1 << t)
        out.append(bits)
    return out


def _tree_lens(c):
    """rows of each sequence, its tree among them"""
    rows = [c["suffix"] if b == 0 else 1 + (b * 2654435761 >> 7) % c["suffix"] for b in range(c["B"])]
    return [c["prefix"] + max(s, n) for s, n in zip(rows, _new(c))]


def _batch_lens(c):
    return [max(n, c["len"] - (b * 40503) % c["len"]) for b, n in enumerate(_new(c))]


def _commit_lens(c):
    return [max(1, c["len"] - (b * 37) % min(c["len"], 3 * c["page"])) for b in range(c["B"])]


def _accepted(c):
    """The nodes on the path that the model agrees with."""
    paths, out = _paths(_parents(c)), []
    for b, n in enumerate(_new(c)):
        bits = paths[b][((b + 3) * 2654435761 >> 9) % n]
        out.append([t for t in range(n) if bits >> t & 1])
    return out


def _history_lens(c):
    return [max(1, c["history"] - (b * 2654435761 >> 8) % c["history"]) for b in range(c["B"])]


def _mask_ids(c):
    """every second row has a grammar (where there is one)"""
    return [r * 7 % c["masks"] if c["masks"] and r % 2 == 0 else -1 for r in range(c["T"] * c["B"])]


def _pages(rows, page):
    return (rows + page - 1) // page


# ---- inputs ------------------------------------------------------------------------

def _gen(seed, stream):
    g = torch.Generator(device="cuda")
    g.manual_seed((int(seed) * 1000003 + stream) & 0x7FFFFFFF)
    return g


def _bf16(shape, g, std=1.0):
    return (torch.randn(shape, device="cuda", generator=g) * std).bfloat16()


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _by_node(rows):
    """[sequence][node] -> int32 [node * B + sequence], as all inputs of nodes lie"""
    return _i32(rows).t().contiguous().view(-1)


def _words(paths, T):
    """[sequence][node] bits -> int32 [node * B + sequence][(T + 31) // 32]"""
    n = (T + 31) // 32
    w = [[[x >> 32 * k & 0xFFFFFFFF for k in range(n)] for x in p] for p in paths]
    v = torch.tensor(w, dtype=torch.int64, device="cuda").transpose(0, 1).reshape(-1, n)
    return torch.where(v >= 2**31, v - 2**32, v).int()


def _rope(rows):
    ang = torch.outer(torch.arange(rows, device="cuda", dtype=torch.float64), 1e7 ** (-torch.arange(ROT, device="cuda", dtype=torch.float64) / ROT))
    return ang.cos().float(), ang.sin().float()


def _pool(planes, pages, c, g):
    """Pool contents as 16-bit patterns of any value: [plane][page][head][row][HD]"""
    n = planes * pages * c["heads"] * c["page"] * c["HD"]
    return torch.randint(-2**31, 2**31, ((n + 1) // 2,), dtype=torch.int32, device="cuda", generator=g).view(torch.int16)[:n].view(
        planes, pages, c["heads"], c["page"], c["HD"])


def _handle(s, pool, ref, table, lens):
    """The pool as a user of the framework holds it."""
    from bunker_b200.pages import PagePool, scratch_bytes
    planes, pages, heads, rows, hd = pool.shape
    s["scratch"] = torch.zeros(scratch_bytes(pages, table.shape[0]), dtype=torch.uint8, device="cuda")
    s["handle"] = PagePool(base=pool.data_ptr(), n_planes=planes, n_pages=pages, heads=heads, page_rows=rows, row_bytes=2 * hd, n_seqs=table.shape[0],
                           max_pages=table.shape[1], ref=ref.data_ptr(), table=table.data_ptr(), lens=lens.data_ptr(),
                           scratch=s["scratch"].data_ptr(), scratch_bytes=s["scratch"].numel())


def prepare(case, seed):
    s = {"case": dict(case), "seed": int(seed)}
    g = _gen(seed, 11)
    if own:
        from bunker_b200 import runtime as R
        R.cu(0)
    {"tree": _prepare_tree, "logits": _prepare_logits, "batch": _prepare_batch, "commit": _prepare_commit}[case["kind"]](s, case, g)
    torch.cuda.synchronize()
    return s


def _prepare_tree(s, c, g):
    B, T, P, Hq, Hkv, HD, page = c["B"], c["T"], c["prefix"], c["Hq"], c["Hkv"], c["HD"], c["page"]
    lens, new = _tree_lens(c), _new(c)
    shared = P // page
    tail = [_pages(n, page) - shared for n in lens]      # pages of a sequence behind the shared ones
    n_pages = shared + sum(tail) + 7
    ids = torch.randperm(n_pages, device="cuda", generator=g, dtype=torch.int32)
    max_pages = shared + max(tail)
    col = torch.arange(max_pages - shared, device="cuda")[None]
    at = torch.tensor([0] + tail, device="cuda").cumsum(0)
    own_page = col < torch.tensor(tail, device="cuda")[:, None]
    table = torch.full((B, max_pages), -1, dtype=torch.int32, device="cuda")
    table[:, :shared] = ids[:shared]
    table[:, shared:] = torch.where(own_page, ids[(shared + at[:-1, None] + col).clamp_max(n_pages - 1)], -1)
    k_pages, v_pages = _bf16((n_pages, Hkv, page, HD), g), _bf16((n_pages, Hkv, page, HD), g)
    if P % page:    # the page that the preamble ends in: every sequence has its copy of those rows
        last = table[:, shared].long()
        k_pages[last, :, :P % page] = k_pages[last[0], :, :P % page].clone()
        v_pages[last, :, :P % page] = v_pages[last[0], :, :P % page].clone()
    max_len = max_pages * page
    paths = _paths(_parents(c))
    pos = [[lens[b] - new[b] + bin(paths[b][t]).count("1") - 1 if t < new[b] else -1 for t in range(T)] for b in range(B)]
    row = _i32([[lens[b] - new[b] + t if t < new[b] else 0 for t in range(T)] for b in range(B)]).long()       # [B][T]
    there = torch.arange(T, device="cuda")[None] < _i32(new)[:, None]
    slot = torch.where(there, table.gather(1, row // page).long() * page + row % page, -1).int()
    cos, sin = _rope(max_len)
    s.update(qg=_bf16((T * B, Hq, 2 * HD if c["fused"] else HD), g), k=_bf16((T * B, Hkv, HD), g), v=_bf16((T * B, Hkv, HD), g), gate=_bf16((T * B, Hq, HD), g),
             q_norm_w=_bf16((HD,), g, 0.02), k_norm_w=_bf16((HD,), g, 0.02), cos=cos, sin=sin, k_pages=k_pages, v_pages=v_pages, table=table, len=_i32(lens),
             new=_i32(new), pos=_by_node(pos), slot=slot.t().contiguous().view(-1), mask=_words(paths, T),
             out=torch.zeros((T * B, Hq * HD), dtype=torch.bfloat16, device="cuda"), scale=1.0 / math.sqrt(HD))
    if own:
        from bunker_b200 import ops
        s["scratch"] = torch.zeros(ops.tree_attn_scratch_bytes(B, T, Hq, Hkv, HD, P), dtype=torch.uint8, device="cuda")
        more = dict(q_norm_w=s["q_norm_w"].data_ptr(), k_norm_w=s["k_norm_w"].data_ptr(), cos_t=cos.data_ptr(), sin_t=sin.data_ptr(), rot_half=ROT,
                    eps=EPS) if c["fused"] else dict(gate=s["gate"].data_ptr())
        s["args"] = ops.tree_attn_args(
            qg=s["qg"].data_ptr(), k=s["k"].data_ptr(), v=s["v"].data_ptr(), k_pages=k_pages.data_ptr(), v_pages=v_pages.data_ptr(), table=table.data_ptr(),
            lens=s["len"].data_ptr(), n_new=s["new"].data_ptr(), pos=s["pos"].data_ptr(), slot=s["slot"].data_ptr(), mask=s["mask"].data_ptr(),
            mask_words=s["mask"].shape[1], out=s["out"].data_ptr(), scratch=s["scratch"].data_ptr(), scratch_bytes=s["scratch"].numel(), B=B, T=T, Hq=Hq, Hkv=Hkv,
            HD=HD, n_pages=n_pages, page_rows=page, max_pages=max_pages, prefix_rows=P, max_len=max_len, scale=s["scale"], fused_norm_rope=int(c["fused"]), **more)


def _prepare_logits(s, c, g):
    B, T, V = c["B"], c["T"], c["V"]
    lens = _history_lens(c)
    # words of a text: some are frequent, most are rare
    u = torch.rand((B, c["history"]), device="cuda", generator=g)
    hist = (V * u ** 4).int().clamp_max(V - 1)
    n_bias = c["bias"]
    s.update(logits=torch.randn((T * B, V), device="cuda", generator=g) * 3, history=hist, hist_len=_i32(lens), prompt_len=_i32([n // 3 for n in lens]),
             repetition=1 + 0.3 * torch.rand(B, device="cuda", generator=g), presence=0.5 * torch.rand(B, device="cuda", generator=g),
             frequency=0.2 * torch.rand(B, device="cuda", generator=g),
             draft=torch.randint(0, V, (T * B,), dtype=torch.int32, device="cuda", generator=g), path=_words(_paths(_parents(c)), T), mask_id=_i32(_mask_ids(c)))
    if n_bias:   # a request names a token once
        s.update(bias_token=torch.rand((B, V), device="cuda", generator=g).topk(min(n_bias, V), dim=1).indices.int().contiguous(),
                 bias_value=torch.randn((B, min(n_bias, V)), device="cuda", generator=g), bias_n=_i32([max(0, min(n_bias, V) - b % 3) for b in range(B)]))
    if c["masks"]:
        words = (V + 31) // 32
        allowed = torch.rand((c["masks"], words, 32), device="cuda", generator=g) < c["allow"]
        bits = (allowed.long() << torch.arange(32, device="cuda")).sum(-1)
        s["allowed"] = torch.where(bits >= 2**31, bits - 2**32, bits).int()
    if own:
        from bunker_b200 import ops
        more = {}
        if T > 1:
            more.update(draft=s["draft"].data_ptr(), path=s["path"].data_ptr(), path_words=s["path"].shape[1])
        if n_bias:
            more.update(bias_token=s["bias_token"].data_ptr(), bias_value=s["bias_value"].data_ptr(), bias_n=s["bias_n"].data_ptr(), bias_ld=s["bias_token"].shape[1])
        if c["masks"]:
            more.update(allowed=s["allowed"].data_ptr(), mask_id=s["mask_id"].data_ptr(), n_masks=c["masks"], allowed_words=s["allowed"].shape[1])
        s["args"] = ops.adjust_logits_args(
            logits=s["logits"].data_ptr(), V=V, B=B, T=T, history=hist.data_ptr(), history_ld=c["history"], hist_len=s["hist_len"].data_ptr(),
            prompt_len=s["prompt_len"].data_ptr(), repetition=s["repetition"].data_ptr(), presence=s["presence"].data_ptr(),
            frequency=s["frequency"].data_ptr(), **more)


def _sequences(c, n_seqs, lens, max_pages, spare, g):
    """A pool's table, counts and lengths where sequence seqs[b] has lens[b] rows in scattered pages."""
    held = torch.tensor([_pages(n, c["page"]) for n in lens], device="cuda")
    n_pages = int(held.sum()) + spare
    ids = torch.randperm(n_pages, device="cuda", generator=g, dtype=torch.int32)
    seqs = torch.randperm(n_seqs, device="cuda", generator=g)[:c["B"]]
    at, col = held.cumsum(0) - held, torch.arange(max_pages, device="cuda")[None]
    table = torch.full((n_seqs, max_pages), -1, dtype=torch.int32, device="cuda")
    table[seqs] = torch.where(col < held[:, None], ids[(at[:, None] + col).clamp_max(n_pages - 1)], -1)
    ref = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
    ref[ids[:int(held.sum())].long()] = 1
    length = torch.zeros(n_seqs, dtype=torch.int32, device="cuda")
    length[seqs] = _i32(lens)
    return seqs.int(), table, ref, length


def _prepare_batch(s, c, g):
    B, T = c["B"], c["T"]
    lens = _batch_lens(c)
    max_pages = _pages(max(lens), c["page"])
    seqs, table, ref, length = _sequences(c, c["seqs"], lens, max_pages, 3, g)
    words = (T + 31) // 32
    z = lambda *shape: torch.zeros(shape, dtype=torch.int32, device="cuda")  # noqa: E731
    s.update(seqs=seqs, table=table, ref=ref, len=length, new=_i32(_new(c)), parent=_by_node(_parents(c)), batch_table=z(B, max_pages), batch_len=z(B), pos=z(T * B),
             slot=z(T * B), mask=z(T * B, words))
    if own:
        s["pool"] = torch.zeros((1, ref.numel(), 1, c["page"], 8), dtype=torch.int16, device="cuda")
        _handle(s, s["pool"], ref, table, length)


def _prepare_commit(s, c, g):
    B, T, page = c["B"], c["T"], c["page"]
    new, accepted = _new(c), _accepted(c)
    before = _commit_lens(c)                                   # rows before the trees
    # A pass begins as the one before it ended: with the accepted rows of the same trees, for which it has room already.
    lens = [n + len(p) for n, p in zip(before, accepted)]
    max_pages = max(_pages(n + m, page) for n, m in zip(before, new))
    spare = sum(_pages(n + m, page) - _pages(n, page) for n, m in zip(before, new)) + 5
    seqs, table, ref, length = _sequences(c, B + 3, lens, max_pages, spare, g)
    token = torch.randperm(1 << 17, device="cuda", generator=g)[:B * T].int()      # [node * B + sequence], no two the same
    target = torch.full_like(token, 1 << 17) + torch.arange(B * T, device="cuda", dtype=torch.int32)
    at = [(p[i] * B + b, p[i + 1] * B + b) for b, p in enumerate(accepted) for i in range(len(p) - 1)]
    if at:
        target[torch.tensor([x for x, _ in at], device="cuda")] = token[torch.tensor([y for _, y in at], device="cuda")]
    z = lambda *shape: torch.zeros(shape, dtype=torch.int32, device="cuda")  # noqa: E731
    s.update(pool=_pool(c["planes"], ref.numel(), c, g), seqs=seqs, table=table, ref=ref, len=length, new=_i32(new), add=_i32([n - len(p) for n, p in zip(new, accepted)]),
             parent=_by_node(_parents(c)), token=token, target=target, path=z(T, B), n_path=z(B), next=z(B), ok=z(2, B))
    if own:
        _handle(s, s["pool"], ref, table, length)


# ---- one pass ----------------------------------------------------------------------

def run(state):
    s, c = state, state["case"]
    return {"tree": _run_tree, "logits": _run_logits, "batch": _run_batch, "commit": _run_commit}[c["kind"]](s, c)


def _bits(words, n):
    """int32 [..][words] -> bool [..][n]"""
    return ((words[..., None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1).bool().flatten(-2)[..., :n]


def _norm_rope(x, w, cos, sin):
    """x [n][heads][HD] in 32 bits, cos and sin [n][ROT]: head RMSNorm times 1 + w, then the rotation of the first 2 * ROT values"""
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * (1.0 + w)
    a, b, c, s = y[..., :ROT], y[..., ROT:2 * ROT], cos[:, None], sin[:, None]
    return torch.cat([a * c - b * s, b * c + a * s, y[..., 2 * ROT:]], -1)


def _run_tree(s, c):
    if own:
        from bunker_b200 import ops
        ops.tree_attn(s["args"])
        return {"out": s["out"], "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    B, T, P, Hq, Hkv, HD, page = c["B"], c["T"], c["prefix"], c["Hq"], c["Hkv"], c["HD"], c["page"]
    G, shared = Hq // Hkv, P // page
    there = (torch.arange(T, device="cuda")[:, None] < s["new"][None]).reshape(-1)
    if c["fused"]:
        pos = s["pos"].clamp_min(0).long()
        cos, sin = s["cos"][pos], s["sin"][pos]
        q = _norm_rope(s["qg"][..., :HD].float(), s["q_norm_w"].float(), cos, sin)
        k = _norm_rope(s["k"].float(), s["k_norm_w"].float(), cos, sin).bfloat16()
        gate = s["qg"][..., HD:].float()
    else:
        q, k, gate = s["qg"].float(), s["k"], s["gate"].float()
    # the trees' rows into their slots
    slot = s["slot"][there].long()
    s["k_pages"][slot // page, :, slot % page] = k[there]
    s["v_pages"][slot // page, :, slot % page] = s["v"][there]
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
    # rows before the tree, then those of the node's path
    node = shared * page + torch.arange(n, device="cuda")[None] - (s["len"] - s["new"])[:, None]      # [B][n]
    path = _bits(s["mask"], T).view(T, B, T).permute(1, 0, 2)                                         # [B][T][T]
    seen = (node < 0)[:, None] | (((node >= 0) & (node < s["new"][:, None]))[:, None] & path.gather(2, node.clamp(0, T - 1)[:, None].expand(B, T, n)))
    ss = ss.view(B, Hkv, T, G, n).masked_fill(~seen[:, None, :, None], float("-inf"))
    sp = sp.view(Hkv, T, B, G, shared * page).permute(2, 0, 1, 3, 4)   # [B][Hkv][T][G][keys]
    m = ss.amax(-1, keepdim=True)
    if shared:
        m = torch.maximum(m, sp.amax(-1, keepdim=True))
    ep, es = torch.exp(sp - m), torch.exp(ss - m)
    z = ep.sum(-1, keepdim=True) + es.sum(-1, keepdim=True)
    op = torch.matmul(ep.permute(1, 2, 0, 3, 4).reshape(Hkv, T * B * G, shared * page), vp).view(Hkv, T, B, G, HD).permute(2, 0, 1, 3, 4)
    os = torch.matmul(es.reshape(B, Hkv, T * G, n), vs).view(B, Hkv, T, G, HD)
    o = ((op + os) / z).permute(2, 0, 1, 3, 4).reshape(T * B, Hq, HD) * torch.sigmoid(gate)
    s["out"].copy_(torch.where(there[:, None], o.reshape(T * B, Hq * HD), 0.0))
    return {"out": s["out"], "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _run_logits(s, c):
    if own:
        from bunker_b200 import ops
        ops.adjust_logits(s["args"])
        return {"logits": s["logits"]}
    B, T, V = c["B"], c["T"], c["V"]
    at = torch.arange(c["history"], device="cuda")[None]
    prompt = at < s["prompt_len"][:, None]
    said = ~prompt & (at < s["hist_len"][:, None])
    hist = s["history"].long()
    in_prompt = torch.zeros((B, V), dtype=torch.int32, device="cuda").scatter_add_(1, hist, prompt.int()) > 0
    times = torch.zeros((B, V), dtype=torch.int32, device="cuda").scatter_add_(1, hist, said.int())
    times = times.repeat(T, 1)                                                              # [T * B][V]
    if T > 1:
        path = _bits(s["path"], T)                                                          # [T * B][T]
        drafted = s["draft"].view(T, B).t().long().repeat(T, 1)                             # [T * B][T]
        times.scatter_add_(1, drafted, path.int())
    by_row = lambda x: x.repeat(T)[:, None]  # noqa: E731
    x, rep = s["logits"], by_row(s["repetition"])
    y = torch.where((times > 0) | in_prompt.repeat(T, 1), torch.where(x > 0, x / rep, x * rep), x)
    y = y - (by_row(s["frequency"]) * times + by_row(s["presence"]) * (times > 0))
    if c["bias"]:
        some = torch.arange(s["bias_token"].shape[1], device="cuda")[None] < s["bias_n"][:, None]
        y = y + torch.zeros((B, V), device="cuda").scatter_add_(1, s["bias_token"].long(), s["bias_value"] * some).repeat(T, 1)
    if c["masks"]:
        allowed = _bits(s["allowed"], V)[s["mask_id"].clamp_min(0).long()] | (s["mask_id"] < 0)[:, None]
        y = torch.where(allowed, y, float("-inf"))
    s["logits"].copy_(y)
    return {"logits": s["logits"]}


def _ancestors(parent, B, T):
    """parent int32 [T * B] -> bool [B][T][T]: node t has node u on its path (itself among them)"""
    one = torch.eye(T, device="cuda")
    p = parent.view(T, B).t().long()
    step = one[p.clamp_min(0)] * (p >= 0)[..., None]       # the way up by one, then by 2, 4, ...
    path = one + step
    for _ in range(max(0, T - 1).bit_length()):
        step = torch.matmul(step, step)
        path = path + torch.matmul(path, step)
    return path > 0


def _run_batch(s, c):
    if own:
        s["handle"].batch(s["seqs"].data_ptr(), c["B"], T=c["T"], n_new=s["new"].data_ptr(), parent=s["parent"].data_ptr(), table=s["batch_table"].data_ptr(),
                          lens=s["batch_len"].data_ptr(), pos=s["pos"].data_ptr(), slot=s["slot"].data_ptr(), mask=s["mask"].data_ptr(),
                          mask_words=s["mask"].shape[1])
        return {k: s[k] for k in ("batch_table", "batch_len", "pos", "slot", "mask")}
    B, T, page = c["B"], c["T"], c["page"]
    seqs, new = s["seqs"].long(), s["new"]
    lens, table = s["len"][seqs], s["table"][seqs]
    col = torch.arange(table.shape[1], device="cuda")[None]
    s["batch_table"].copy_(torch.where(col < ((lens + page - 1) // page)[:, None], table, -1))
    s["batch_len"].copy_(lens)
    t = torch.arange(T, device="cuda")[None]
    there, row = t < new[:, None], (lens - new)[:, None] + t                      # [B][T]
    path = _ancestors(s["parent"], B, T)
    pos = (lens - new)[:, None] + path.sum(-1).int() - 1
    s["pos"].copy_(torch.where(there, pos, -1).t().reshape(-1))
    slot = table.gather(1, (row // page).clamp(0, table.shape[1] - 1).long()) * page + row % page
    s["slot"].copy_(torch.where(there, slot, -1).t().reshape(-1))
    words = s["mask"].shape[1]
    bits = torch.zeros((B, T, words * 32), dtype=torch.int64, device="cuda")
    bits[..., :T] = path & there[..., None]
    w = (bits.view(B, T, words, 32) << torch.arange(32, device="cuda")).sum(-1)
    s["mask"].copy_(torch.where(w >= 2**31, w - 2**32, w).transpose(0, 1).reshape(T * B, words))
    return {k: s[k] for k in ("batch_table", "batch_len", "pos", "slot", "mask")}


def _run_commit(s, c):
    names = ("pool", "table", "ref", "len", "path", "n_path", "next", "ok")
    B, T, page = c["B"], c["T"], c["page"]
    if own:
        s["handle"].grow(s["seqs"].data_ptr(), s["add"].data_ptr(), B, s["ok"].data_ptr())
        s["handle"].commit(s["seqs"].data_ptr(), B, T=T, n_new=s["new"].data_ptr(), parent=s["parent"].data_ptr(), token=s["token"].data_ptr(),
                           target=s["target"].data_ptr(), path=s["path"].data_ptr(), n_path=s["n_path"].data_ptr(), next=s["next"].data_ptr(),
                           ok=s["ok"].data_ptr() + 4 * B)
        return {k: s[k] for k in names}
    table, ref, lens, new = s["table"], s["ref"], s["len"], s["new"]
    seqs = s["seqs"].long()
    col = torch.arange(table.shape[1], device="cuda")[None]
    # room: the lowest free pages, in the list's order
    before, after = (lens[seqs] + page - 1) // page, (lens[seqs] + s["add"] + page - 1) // page
    need, free = after - before, torch.nonzero(ref == 0).flatten()
    s["ok"][0] = ((need == 0) | (need.cumsum(0) <= free.numel())).int()
    i, j = torch.nonzero((col >= before[:, None]) & (col < after[:, None]), as_tuple=True)
    fresh = free[:i.numel()]
    table[seqs[i], j] = fresh.int()
    ref[fresh] = 1
    lens[seqs] = lens[seqs] + s["add"]
    # a node stays if its token is what the model says after its parent, and no node before it has the same parent and token, all the way up
    path = _ancestors(s["parent"], B, T)
    parent, token, target = (s[k].view(T, B).t() for k in ("parent", "token", "target"))        # [B][T]
    up = parent.clamp_min(0).long()
    there = torch.arange(T, device="cuda")[None] < new[:, None]
    said = (token == target.gather(1, up)) & (parent >= 0) & there
    earlier = torch.ones((T, T), dtype=torch.bool, device="cuda").tril(-1)
    again = (said[:, None, :] & (parent[:, None, :] == parent[:, :, None]) & earlier).any(-1)
    agrees = (said & ~again) | (torch.arange(T, device="cuda")[None] == 0)
    kept = ~(path & ~agrees[:, None, :]).any(-1) & there
    n = kept.sum(-1).int()
    b, node = torch.nonzero(kept, as_tuple=True)
    rank = (kept.cumsum(-1) - 1)[b, node]
    s["path"].fill_(-1)
    s["path"][rank, b] = node.int()
    s["n_path"].copy_(n)
    last = (kept * torch.arange(T, device="cuda")[None]).amax(-1)
    s["next"].copy_(target.gather(1, last[:, None])[:, 0])
    s["ok"][1] = 1
    # their rows move up
    base = lens[seqs] - new
    src, dst = base[b] + node, base[b] + rank
    ps, pd = table[seqs[b], src // page].long(), table[seqs[b], dst // page].long()
    s["pool"][:, pd, :, dst % page] = s["pool"][:, ps, :, src % page]
    # pages behind them go back
    held, kept_pages = (lens[seqs] + page - 1) // page, (base + n + page - 1) // page
    i, j = torch.nonzero((col >= kept_pages[:, None]) & (col < held[:, None]), as_tuple=True)
    gone = table[seqs[i], j].long()
    ref.scatter_add_(0, gone, torch.full_like(gone, -1, dtype=torch.int32))
    table[seqs[i], j] = -1
    lens[seqs] = base + n
    return {k: s[k] for k in names}


# ---- the definition in 64 bits ---------------------------------------------------------

def exact(case, seed):
    c = case
    if c["kind"] not in ("tree", "logits"):
        return None     # whole numbers and copied patterns
    s = prepare(c, seed)
    B, T = c["B"], c["T"]
    if c["kind"] == "logits":
        y, V = s["logits"].double(), c["V"]
        lens, prompts, draft, paths = s["hist_len"].tolist(), s["prompt_len"].tolist(), s["draft"].tolist(), _paths(_parents(c))
        rep, pres, freq = (s[k].double() for k in ("repetition", "presence", "frequency"))
        for b in range(B):
            h = s["history"][b].long()
            seen_before = torch.zeros(V, dtype=torch.bool, device="cuda")
            seen_before[h[:prompts[b]]] = True
            count = torch.bincount(h[prompts[b]:lens[b]], minlength=V)
            for t in range(T):
                r, n = t * B + b, count
                if T > 1:
                    drafted = torch.tensor([draft[u * B + b] for u in range(T) if paths[b][t] >> u & 1], device="cuda")
                    n = count + torch.bincount(drafted, minlength=V)
                i = torch.nonzero((n > 0) | seen_before).flatten()
                x, k = y[r, i], n[i].double()
                y[r, i] = torch.where(x > 0, x / rep[b], x * rep[b]) - freq[b] * k - pres[b] * (k > 0)
                if c["bias"]:
                    m = int(s["bias_n"][b])
                    y[r, s["bias_token"][b, :m].long()] += s["bias_value"][b, :m].double()
                a = int(s["mask_id"][r])
                if a >= 0:
                    word = s["allowed"][a].long() & 0xFFFFFFFF
                    v = torch.arange(V, device="cuda")
                    y[r, (word[v // 32] >> v % 32) % 2 == 0] = -math.inf
        return {"logits": y}
    Hq, Hkv, HD, page = c["Hq"], c["Hkv"], c["HD"], c["page"]
    lens, new, paths = s["len"].tolist(), s["new"].tolist(), _paths(_parents(c))
    kp, out = s["k_pages"].double(), torch.zeros((T * B, Hq, HD), dtype=torch.float64, device="cuda")

    def turned(x, w, p):
        """x [n][heads][HD] of nodes at positions p [n]"""
        y = x / torch.sqrt((x ** 2).sum(-1, keepdim=True) / HD + EPS) * (w.double() + 1)
        c64, s64 = s["cos"][p].double()[:, None], s["sin"][p].double()[:, None]
        z = y.clone()
        z[..., :ROT] = y[..., :ROT] * c64 - y[..., ROT:2 * ROT] * s64
        z[..., ROT:2 * ROT] = y[..., ROT:2 * ROT] * c64 + y[..., :ROT] * s64
        return z

    for b in range(B):
        n, first = new[b], lens[b] - new[b]
        e = torch.arange(n, device="cuda") * B + b
        rows = first + torch.arange(n, device="cuda")
        depth = torch.tensor([bin(paths[b][t]).count("1") - 1 for t in range(n)], device="cuda")
        k, q, gate = s["k"][e].double(), s["qg"][e].double(), s["gate"][e].double()
        if c["fused"]:
            q, gate = turned(q[..., :HD], s["q_norm_w"], first + depth), q[..., HD:]
            k = turned(k, s["k_norm_w"], first + depth)
        at = s["table"][b].long()[rows // page]
        kp[at, :, rows % page] = k
        s["v_pages"][at, :, rows % page] = s["v"][e]
        pages = s["table"][b, :_pages(lens[b], page)].long()
        K = kp[pages].transpose(0, 1).reshape(Hkv, -1, HD)[:, :lens[b]]
        V = s["v_pages"][pages].double().transpose(0, 1).reshape(Hkv, -1, HD)[:, :lens[b]]
        hidden = torch.zeros((n, lens[b]), dtype=torch.bool, device="cuda")
        hidden[:, first:] = torch.tensor([[not paths[b][t] >> u & 1 for u in range(n)] for t in range(n)], device="cuda")
        qh = q.view(n, Hkv, Hq // Hkv, HD).permute(1, 2, 0, 3)                        # [Hkv][G][n][HD]
        w = torch.softmax((qh @ K[:, None].transpose(2, 3) * s["scale"]).masked_fill(hidden, -math.inf), -1)
        out[e] = (w @ V[:, None]).permute(2, 0, 1, 3).reshape(n, Hq, HD) / (1 + torch.exp(-gate))
    return {"out": out.view(T * B, Hq * HD), "k_pages": kp if c["fused"] else None, "v_pages": None}


# ---- what a pass cannot do without ----------------------------------------------------

def work(case):
    c = case
    B, T, new = c["B"], c["T"], _new(c)
    if c["kind"] == "tree":
        Hq, Hkv, HD, page = c["Hq"], c["Hkv"], c["HD"], c["page"]
        lens, paths = _tree_lens(c), _paths(_parents(c))
        shared = c["prefix"] // page * page
        rows = shared + sum(n - shared for n in lens)
        keys = sum(n * (m - n) + sum(bin(x).count("1") for x in p[:n]) for n, m, p in zip(new, lens, paths))
        return {"bytes": rows * Hkv * HD * 4 + sum(new) * (Hq * 3 + Hkv * 2) * HD * 2, "flops": keys * Hq * HD * 4}
    if c["kind"] == "logits":
        lens, ids = _history_lens(c), _mask_ids(c)
        masked = sum(a >= 0 for a in ids)
        # a token of the history is read; a logit that it, a node or a bias names is read and written once (here: three quarters of the words are new ones),
        # unless the grammar hides it; one that the grammar hides is written
        named = T * sum(0.75 * min(n, c["V"]) + c["bias"] for n in lens) + sum(new)
        return {"bytes": 4 * sum(lens) + 8 * B * c["bias"] + 8 * named * (1 - masked / len(ids) * (1 - c["allow"])) + masked * 4 * c["V"] * (1 - c["allow"])
                + len(set(ids) - {-1}) * c["V"] / 8, "flops": 0}
    if c["kind"] == "batch":
        lens, words = _batch_lens(c), (T + 31) // 32
        return {"bytes": 4 * (sum(_pages(n, c["page"]) for n in lens) + B * _pages(max(lens), c["page"])) + 4 * B * 4 + 4 * T * B * (3 + words), "flops": 0}
    before, accepted = _commit_lens(c), _accepted(c)
    row = c["heads"] * c["HD"] * 2 * c["planes"]     # one cached position of all planes
    moved = sum(sum(i != t for i, t in enumerate(p)) for p in accepted)
    pages = sum(_pages(n + m, c["page"]) - _pages(n, c["page"]) for n, m in zip(before, new))
    return {"bytes": 2 * row * moved + 4 * (4 * sum(new) + 6 * B + 4 * pages), "flops": 0}
