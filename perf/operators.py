"""The serving operators of this package as measurable cases: attention of drafted-token trees over the paged KV arena,
committing an accepted path of such a tree, sampling the next token, and copying the rows of a slot to other slots.

`listed` and `draw` give cases, `prepare` what a serving loop holds before the call, `run` one pass: the plain form in
elementary torch operations, or, where `own` is true, the package's entry points.  `exact` states the same results in 64
bits, row by row, and `work` the bytes and operations that a pass cannot do without.

Shapes are those of the package's own model configurations: 14 query and 2 KV heads of 64 over 24 layers with a vocabulary
of 151936; 12 and 2 heads of 128 over 28 layers; 12 heads of 64 over 12 layers with a vocabulary of 50257.
"""
import math

import numpy as np
import torch

own = False

PAGE = 64                      # positions per page of the KV arena
DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one stream decoding one token at a short context: what a single user waits for
        {"name": "tree one token", "op": "tree", "q": "f16", "kv": "f16", "heads": 14, "kv_heads": 2, "hd": 64,
         "seqs": 1, "nodes_lo": 1, "nodes_hi": 1, "len_lo": 300, "len_hi": 300, "width": 1, "window": 0},
        # one stream, a small draft, a long document in the cache
        {"name": "tree long context", "op": "tree", "q": "bf16", "kv": "bf16", "heads": 12, "kv_heads": 2, "hd": 128,
         "seqs": 1, "nodes_lo": 9, "nodes_hi": 9, "len_lo": 30011, "len_hi": 30011, "width": 3, "window": 0},
        # the model path's own types: fp32 queries over the fp16 arena, ragged drafts and contexts
        {"name": "tree batch fp32", "op": "tree", "q": "f32", "kv": "f16", "heads": 14, "kv_heads": 2, "hd": 64,
         "seqs": 32, "nodes_lo": 1, "nodes_hi": 17, "len_lo": 65, "len_hi": 1900, "width": 4, "window": 0},
        # every query head with its own K and V, a sliding window
        {"name": "tree all heads windowed", "op": "tree", "q": "f16", "kv": "f16", "heads": 12, "kv_heads": 12, "hd": 64,
         "seqs": 24, "nodes_lo": 5, "nodes_hi": 26, "len_lo": 100, "len_hi": 990, "width": 5, "window": 512},
        # large drafts over long contexts: the operation-bound end
        {"name": "tree large drafts", "op": "tree", "q": "bf16", "kv": "bf16", "heads": 12, "kv_heads": 2, "hd": 128,
         "seqs": 16, "nodes_lo": 48, "nodes_hi": 64, "len_lo": 6000, "len_hi": 10000, "width": 8, "window": 0},
        # the next token of one stream
        {"name": "sample one row", "op": "sample", "rows": 1, "vocab": 151936, "type": "f32", "mix": "nucleus"},
        # a serving batch in which every request has its own settings
        {"name": "sample batch", "op": "sample", "rows": 128, "vocab": 151936, "type": "f32", "mix": "mixed"},
        # many rows of a smaller vocabulary, temperature alone
        {"name": "sample many rows", "op": "sample", "rows": 1000, "vocab": 50257, "type": "f32", "mix": "temperature"},
        # one stream's accepted draft
        {"name": "commit one stream", "op": "commit", "layers": 24, "kv_dim": 128, "seqs": 1, "nodes": 17, "width": 4, "len": 700},
        # a batch of streams, each with another number of accepted tokens
        {"name": "commit batch", "op": "commit", "layers": 28, "kv_dim": 256, "seqs": 128, "nodes": 41, "width": 5, "len": 333},
        # a short prompt continued twice
        {"name": "fork short prompt", "op": "copy", "layers": 12, "kv_dim": 768, "copies": 1, "first": 0, "count": 45},
        # a shared prompt continued by sixteen streams
        {"name": "fork to many", "op": "copy", "layers": 28, "kv_dim": 256, "copies": 16, "first": 0, "count": 1733},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tree", "tree", "tree", "sample", "sample", "commit", "copy"])
    if op == "tree":
        heads, kv_heads, hd = rng.choice([(14, 2, 64), (12, 2, 128), (12, 12, 64), (8, 1, 128), (6, 3, 80), (4, 4, 32), (16, 4, 256)])
        q, kv = rng.choice([("f16", "f16"), ("bf16", "bf16"), ("f32", "f16"), ("f32", "bf16")])
        seqs = _log(rng, 1, 64)
        hi = _log(rng, 1, 130)
        top = min(30000, max(40, 2500 * 32 // seqs))
        length = min(_log(rng, 1, top), int(7e9 / (seqs * hi * heads * hd)) + 1)
        return {"op": "tree", "q": q, "kv": kv, "heads": heads, "kv_heads": kv_heads, "hd": hd, "seqs": seqs,
                "nodes_lo": rng.randint(1, hi), "nodes_hi": hi, "len_lo": rng.randint(0, length), "len_hi": length,
                "width": rng.randint(1, 9), "window": rng.choice([0, 0, 0, _log(rng, 3, 4000)])}
    if op == "sample":
        vocab = _log(rng, 100, 152000)
        return {"op": "sample", "rows": min(_log(rng, 1, 1000), max(1, int(4.5e7) // vocab)), "vocab": vocab,
                "type": rng.choice(["f32", "f32", "f16", "bf16"]), "mix": rng.choice(["nucleus", "mixed", "temperature"])}
    layers, kv_dim = rng.choice([(24, 128), (28, 256), (12, 768), (2, 1024), (5, 72)])
    if op == "commit":
        return {"op": "commit", "layers": layers, "kv_dim": kv_dim, "seqs": _log(rng, 1, 128), "nodes": _log(rng, 1, 200),
                "width": rng.randint(1, 9), "len": _log(rng, 1, 400)}
    return {"op": "copy", "layers": layers, "kv_dim": kv_dim, "copies": _log(rng, 1, 16), "first": rng.choice([0, 0, rng.randint(1, 300)]),
            "count": _log(rng, 1, 1400)}


# ---- inputs ----------------------------------------------------------------------------------------------------------------

def _spread(lo, hi, n):
    """n sizes from lo to hi, both among them where n allows."""
    return [hi] if n == 1 else [lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _trees(sizes, width, rs):
    """Drafted trees in levels of `width` nodes under a root: each node's parent is a random node of the level above.  The
    ancestors of every node, itself among them, as bits of 64-bit words (int64 [sum of sizes][words]), and their parents."""
    most = max(sizes)
    words = (most + 63) // 64
    n = len(sizes)
    bits = np.zeros((n, most, words), np.uint64)
    parents = np.full((n, most), -1, np.int64)
    every = np.arange(n)
    for i in range(most):
        if i:
            level = (i - 1) // width
            parents[:, i] = 0 if level == 0 else 1 + (level - 1) * width + rs.randint(0, width, n)
            bits[:, i] = bits[every, parents[:, i]]
        bits[:, i, i // 64] |= np.uint64(1 << (i % 64))
    inside = np.arange(most)[None, :] < np.array(sizes)[:, None]
    return bits[inside].view(np.int64).reshape(-1, words), parents, inside


def _arena(layers, pages, kv_dim, kind, gen):
    shape = (layers, pages, PAGE, kv_dim)
    return tuple(torch.randn(shape, generator=gen, device=DEV, dtype=TYPES[kind]) for _ in range(2))


def _tables(slots, per_slot, pages, rs):
    """A page table [slots][per_slot] whose pages lie in the pool in no order."""
    return torch.from_numpy(rs.permutation(pages)[: slots * per_slot].reshape(slots, per_slot).astype(np.int32)).to(DEV)


def prepare(case, seed):
    rs = np.random.RandomState(seed % (1 << 31))
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    dev = lambda v, t=np.int32: torch.from_numpy(np.ascontiguousarray(np.asarray(v).astype(t))).to(DEV)  # noqa: E731
    s = dict(case)
    if case["op"] == "tree":
        n = case["seqs"]
        sizes = [int(v) for v in rs.permutation(_spread(min(case["nodes_lo"], case["nodes_hi"]), case["nodes_hi"], n))]
        base = rs.permutation(_spread(min(case["len_lo"], case["len_hi"]), case["len_hi"], n))
        words, _, _ = _trees(sizes, case["width"], rs)
        most = int(max(base)) + max(sizes)
        per_slot = -(-most // PAGE)
        pages = n * per_slot + 3
        k, v = _arena(1, pages, case["kv_heads"] * case["hd"], case["kv"], gen)
        rows = sum(sizes)
        s.update(k=k[0].view(pages, PAGE, case["kv_heads"], case["hd"]), v=v[0].view(pages, PAGE, case["kv_heads"], case["hd"]),
                 q_rows=torch.randn((rows, case["heads"] * case["hd"]), generator=gen, device=DEV).to(TYPES[case["q"]]),
                 out=torch.empty((rows, case["heads"] * case["hd"]), device=DEV, dtype=TYPES[case["q"]]),
                 table=_tables(n, per_slot, pages, rs), slots=dev(rs.permutation(n)), row_start=dev(np.cumsum([0] + sizes)),
                 base=dev(base), mask=dev(words, np.int64), most=most, most_nodes=max(sizes),
                 work=torch.empty(64 << 20, device=DEV, dtype=torch.uint8))
    elif case["op"] == "sample":
        m, n = case["rows"], case["vocab"]
        # a model's logits: a broad body, and a few dozen tokens that fit the context, some far ahead of the rest
        logits = torch.randn((m, n), generator=gen, device=DEV).mul_(2.0)
        few = min(48, n)
        at = (torch.randint(0, n, (m, 1), generator=gen, device=DEV) + torch.arange(few, device=DEV) * (n // few)) % n
        logits.scatter_add_(1, at, torch.rand((m, few), generator=gen, device=DEV).mul_(12.0))
        s.update(logits=logits.to(TYPES[case["type"]]), u=torch.rand(m, generator=gen, device=DEV),
                 ids=torch.empty(m, device=DEV, dtype=torch.int32), prob=torch.empty(m, device=DEV))
        pick = lambda values, t: dev(rs.choice(values, m), t)  # noqa: E731
        s["temperature"] = pick([0.6, 0.8, 1.0, 1.3] + ([0.0] if case["mix"] == "mixed" else []), np.float32)
        s["top_k"] = s["top_p"] = s["min_p"] = None
        if case["mix"] == "nucleus":
            s["top_k"], s["top_p"] = pick([50], np.int32), pick([0.95], np.float32)
        elif case["mix"] == "mixed":
            s["top_k"] = pick([0, 0, 1, 40, 1000], np.int32)
            s["top_p"] = pick([1.0, 0.8, 0.95, 0.99], np.float32)
            s["min_p"] = pick([0.0, 0.0, 0.02, 0.1], np.float32)
    elif case["op"] == "commit":
        n, nodes, width = case["seqs"], case["nodes"], case["width"]
        words, parents, _ = _trees([nodes] * n, width, rs)
        tokens = rs.randint(0, 50000, (n, nodes))
        for j in range(1, nodes):        # siblings of a draft are different tokens
            tokens[:, j] = 8 * tokens[:, j] + (j - 1) % 8 if width <= 8 else 16 * tokens[:, j] + (j - 1) % 16
        picked = rs.randint(1 << 20, 1 << 21, (n, nodes))
        depth = -(-(nodes - 1) // width)
        for b in range(n):               # sequence b accepts b mod (depth + 1) drafted tokens, one after the other
            want = depth if n == 1 else b % (depth + 1)
            node = min(1 + (want - 1) * width + int(rs.randint(0, width)), nodes - 1) if want else 0
            while node > 0:
                picked[b, parents[b, node]] = tokens[b, node]
                node = parents[b, node]
        per_slot = -(-(case["len"] + nodes) // PAGE)
        pages = n * per_slot + 2
        k, v = _arena(case["layers"], pages, case["kv_dim"], "f16", gen)
        s.update(k=k, v=v, table=_tables(n, per_slot, pages, rs), slots=dev(rs.permutation(n)),
                 row_start=dev(np.arange(n + 1) * nodes), base=dev(case["len"] - rs.randint(0, min(60, case["len"]), n)),
                 mask=dev(words, np.int64), tokens=dev(tokens.reshape(-1)), picked=dev(picked.reshape(-1)), most_path=depth + 1,
                 accepted=torch.empty((n, depth + 1), device=DEV, dtype=torch.int32),
                 n_accepted=torch.empty(n, device=DEV, dtype=torch.int32), new_base=torch.empty(n, device=DEV, dtype=torch.int32))
    else:
        n = case["copies"]
        per_slot = -(-(case["first"] + case["count"]) // PAGE)
        pages = (n + 1) * per_slot + 1
        k, v = _arena(case["layers"], pages, case["kv_dim"], "f16", gen)
        order = rs.permutation(n + 1)
        s.update(k=k, v=v, table=_tables(n + 1, per_slot, pages, rs), src=dev(np.full(n, order[0])), dst=dev(order[1:]),
                 start=dev(np.full(n, case["first"])), end=dev(np.full(n, case["first"] + case["count"])))
    return s


# ---- the package's operators, as a serving loop calls them -----------------------------------------------------------------

def _own(s):
    import edgecore_b200 as ec
    stream = torch.cuda.current_stream().cuda_stream
    if s["op"] == "tree":
        ec.tree_attention(s["out"], s["q_rows"], s["k"], s["v"], s["table"], s["row_start"], s["base"], s["mask"], slots=s["slots"],
                          window=s["window"], max_len=s["most"], workspace=s["work"], stream=stream)
        return s["out"]
    if s["op"] == "sample":
        ec.sample(s["ids"], s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"],
                  prob=s["prob"], stream=stream)
        return {"ids": s["ids"], "prob": s["prob"]}
    if s["op"] == "commit":
        ec.tree_commit(s["k"], s["v"], s["table"], s["row_start"], s["base"], s["mask"], s["tokens"], s["picked"], s["accepted"],
                       s["n_accepted"], s["new_base"], slots=s["slots"], stream=stream)
        return {"k": s["k"], "v": s["v"], "accepted": s["accepted"], "n": s["n_accepted"], "base": s["new_base"]}
    ec.kv_copy(s["k"], s["v"], s["table"], s["src"], s["dst"], s["start"], s["end"], stream=stream)
    return {"k": s["k"], "v": s["v"]}


# ---- the plain forms -------------------------------------------------------------------------------------------------------

def _bits(mask, most):
    """bool [rows][most]: bit j of each row of the mask words."""
    j = torch.arange(most, device=DEV)
    return ((mask[:, j // 64] >> (j % 64)) & 1).bool()


def _rows_of(table, slots, positions):
    """Arena rows of positions [seqs][n] of the slots; positions behind the table's end give any row."""
    page = (positions // PAGE).clamp(max=table.shape[1] - 1)
    return table[slots.long()].long().gather(1, page) * PAGE + positions % PAGE


def _plain_tree(s):
    q, start, base = s["q_rows"], s["row_start"].long(), s["base"].long()
    heads, kvh, hd, n, most, t = s["heads"], s["kv_heads"], s["hd"], s["seqs"], s["most"], s["most_nodes"]
    size = start[1:] - start[:-1]
    node = torch.arange(t, device=DEV)
    real = node[None] < size[:, None]                                    # [seqs][nodes]
    row = (start[:-1, None] + node).clamp(max=q.shape[0] - 1)
    qf = q.float().view(-1, kvh, heads // kvh, hd)[row]                  # [seqs][nodes][kv heads][group][hd]
    pos = torch.arange(most, device=DEV).expand(n, most)
    at = _rows_of(s["table"], s["slots"], pos)
    k = s["k"].view(-1, kvh, hd)[at].float()                             # [seqs][positions][kv heads][hd]
    score = torch.einsum("btkgd,bpkd->bktgp", qf, k) / math.sqrt(hd)
    del k
    kin = _bits(s["mask"], t)[row]                                       # [seqs][nodes][nodes]
    depth = kin.sum(-1) - 1
    rel = pos - base[:, None]                                            # index of a position among the nodes
    drafted = (rel >= 0) & (rel < size[:, None])
    j = rel.clamp(0, t - 1)
    seen = torch.where((rel < 0)[:, None], torch.ones_like(real)[..., None], drafted[:, None] & kin.gather(2, j[:, None].expand(n, t, most)))
    if s["window"]:
        key_pos = torch.where(rel < 0, pos, base[:, None] + depth.gather(1, j))
        seen = seen & (key_pos[:, None] > (base[:, None] + depth)[..., None] - s["window"])
    seen = seen[:, None, :, None]
    score = score.masked_fill(~seen, -math.inf)
    high = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(high == -math.inf, 0.0, high))
    v = s["v"].view(-1, kvh, hd)[at].float()
    total = p.sum(-1)
    out = torch.einsum("bktgp,bpkd->btkgd", p, v) / torch.where(total == 0, 1.0, total).permute(0, 2, 1, 3)[..., None]
    s["out"].copy_(out.reshape(n, t, heads * hd)[real])
    return s["out"]


def _plain_sample(s):
    logits = s["logits"].double()
    m, n = logits.shape
    logits = torch.where(logits.isnan(), -math.inf, logits)
    off = lambda v, none: torch.full((m, 1), none, device=DEV, dtype=torch.float64) if v is None else v.double()[:, None]  # noqa: E731
    t, p, least = off(s["temperature"], 1.0), off(s["top_p"], 1.0), off(s["min_p"], 0.0)
    k = off(s["top_k"], 0.0)
    k = torch.where(k <= 0, float(n), k)
    high, order = torch.sort(logits, dim=1, descending=True, stable=True)  # ties: the lowest index first
    greedy = t <= 0
    w = torch.exp((high - high[:, :1]) / torch.where(greedy, 1.0, t))
    rank = torch.arange(n, device=DEV, dtype=torch.float64)[None]
    w = torch.where((rank < k) & ~(greedy & (rank > 0)), w, 0.0)
    before = w.cumsum(1) - w
    w = torch.where((p >= 1) | (before < p * w.sum(1, keepdim=True)) | (rank == 0), w, 0.0)
    w = torch.where((w >= least) | (rank == 0), w, 0.0)
    w = torch.zeros_like(w).scatter_(1, order, w)                         # back in the vocabulary's order
    sums = w.cumsum(1)
    total = sums[:, -1:]
    ids = (sums <= s["u"].double()[:, None] * total).sum(1, keepdim=True)
    last = (w > 0).double().mul_(rank).amax(1, keepdim=True).long()
    ids = torch.minimum(ids, last)
    return {"ids": ids[:, 0].int(), "prob": (w.gather(1, ids) / total)[:, 0].float()}


def _plain_commit(s):
    start, n, nodes, longest = s["row_start"].long(), s["seqs"], s["nodes"], s["most_path"]
    kin = _bits(s["mask"], nodes).view(n, nodes, nodes)
    j = torch.arange(nodes, device=DEV)
    own_bit = torch.eye(nodes, device=DEV, dtype=torch.bool)
    above = kin & ~own_bit
    parent = torch.where(above, j, -1).amax(2)                            # the nearest ancestor has the highest index
    token, picked = s["tokens"].view(n, nodes), s["picked"].view(n, nodes)
    match = (parent >= 0) & (token == picked.gather(1, parent.clamp(min=0)))
    same = match[:, :, None] & match[:, None, :] & (parent[:, :, None] == parent[:, None, :]) & (j[None, :] < j[:, None])
    good = (match & ~same.any(2)) | (j == 0)                              # of equal siblings the first
    taken = good & ~(kin & ~good[:, None, :]).any(2) & (kin[:, :, 0])
    count = taken.sum(1)
    path = torch.where(taken, j, nodes).sort(1).values[:, :longest]
    step = torch.arange(longest, device=DEV)[None]
    real = step < count[:, None]
    path = path.clamp(max=nodes - 1)
    at = s["base"].long()[:, None]
    src = _rows_of(s["table"], s["slots"], at + path)[real]
    dst = _rows_of(s["table"], s["slots"], at + step.expand(n, longest))[real]
    layers = s["layers"]
    k, v = s["k"].view(layers, -1, s["kv_dim"]), s["v"].view(layers, -1, s["kv_dim"])
    k[:, dst] = k[:, src]
    v[:, dst] = v[:, src]
    s["accepted"].copy_(torch.where(real, picked.gather(1, path), -1))    # the token that follows each accepted node
    s["n_accepted"].copy_(count)
    s["new_base"].copy_(s["base"] + count)
    return {"k": s["k"], "v": s["v"], "accepted": s["accepted"], "n": s["n_accepted"], "base": s["new_base"]}


def _plain_copy(s):
    layers, first, count = s["layers"], s["first"], s["count"]
    pos = (first + torch.arange(count, device=DEV)).expand(s["copies"], count)
    src, dst = _rows_of(s["table"], s["src"], pos).view(-1), _rows_of(s["table"], s["dst"], pos).reshape(-1)
    k, v = s["k"].view(layers, -1, s["kv_dim"]), s["v"].view(layers, -1, s["kv_dim"])
    k[:, dst] = k[:, src]
    v[:, dst] = v[:, src]
    return {"k": s["k"], "v": s["v"]}


def run(state):
    if own:
        return _own(state)
    return {"tree": _plain_tree, "sample": _plain_sample, "commit": _plain_commit, "copy": _plain_copy}[state["op"]](state)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------------

def work(case):
    if case["op"] == "tree":
        size = {"f32": 4, "f16": 2, "bf16": 2}[case["q"]]
        n = case["seqs"]
        nodes, lens = (_spread(min(case[a], case[b]), case[b], n) for a, b in (("nodes_lo", "nodes_hi"), ("len_lo", "len_hi")))
        mean_nodes, rows = sum(nodes) / n, sum(nodes)
        seen = sum(min(v, case["window"]) if case["window"] else v for v in lens)
        kv_rows = seen + rows
        wide = case["heads"] * case["hd"]
        return {"bytes": 2 * rows * wide * size + kv_rows * 2 * case["kv_heads"] * case["hd"] * 2 + rows * 8 * ((max(nodes) + 63) // 64),
                "flops": 4 * wide * (mean_nodes * seen + rows)}
    if case["op"] == "sample":
        size = 4 if case["type"] == "f32" else 2
        return {"bytes": case["rows"] * (case["vocab"] * size + 24), "flops": 4 * case["rows"] * case["vocab"]}
    row = case["layers"] * 2 * case["kv_dim"] * 2
    if case["op"] == "commit":
        n, depth = case["seqs"], -(-(case["nodes"] - 1) // case["width"])
        moved = depth if n == 1 else sum(b % (depth + 1) for b in range(n))
        return {"bytes": 2 * moved * row + n * case["nodes"] * (8 * ((case["nodes"] + 63) // 64) + 8), "flops": 0}
    return {"bytes": (1 + case["copies"]) * case["count"] * row, "flops": 0}


# ---- the definitions in 64 bits, row by row --------------------------------------------------------------------------------

def _exact_tree(s):
    heads, kvh, hd, window = s["heads"], s["kv_heads"], s["hd"], s["window"]
    start, base, slots, table = (s[x].tolist() for x in ("row_start", "base", "slots", "table"))
    words = s["mask"].cpu().numpy().view(np.uint64)
    out = torch.zeros((start[-1], heads, hd), device=DEV, dtype=torch.float64)
    for b in range(s["seqs"]):
        r0, t, length = start[b], start[b + 1] - start[b], base[b]
        pages = torch.tensor(table[slots[b]], device=DEV)
        k, v = (s[x][pages].reshape(-1, kvh, hd)[: length + t].double() for x in ("k", "v"))
        anc = np.array([[bool(int(words[r0 + i, j // 64]) >> (j % 64) & 1) for j in range(t)] for i in range(t)])
        depth = anc.sum(1) - 1
        allow = np.ones((t, length + t), bool)
        allow[:, length:] = anc
        if window:
            where = np.concatenate([np.arange(length), length + depth])
            allow &= where[None, :] > (length + depth)[:, None] - window
        blocked = torch.from_numpy(~allow).to(DEV)
        q = s["q_rows"][r0:r0 + t].double().view(t, heads, hd)
        for h in range(heads):
            score = (q[:, h] @ k[:, h // (heads // kvh)].T) * hd ** -0.5
            score[blocked] = -math.inf
            weights = torch.nan_to_num(torch.softmax(score, 1), nan=0.0)
            out[r0:r0 + t, h] = weights @ v[:, h // (heads // kvh)]
    return out.view(start[-1], heads * hd)


def _exact_sample(s):
    m, n = s["logits"].shape
    get = lambda x, none: [none] * m if s[x] is None else [float(v) for v in s[x].tolist()]  # noqa: E731
    t, k, p, least = get("temperature", 1.0), get("top_k", 0), get("top_p", 1.0), get("min_p", 0.0)
    u = s["u"].double().tolist()
    ids, prob = torch.empty(m, dtype=torch.int32), torch.empty(m, dtype=torch.float64)
    for r in range(m):
        row = s["logits"][r].double().cpu().numpy()
        if t[r] <= 0:
            ids[r], prob[r] = int(np.argmax(row)), 1.0
            continue
        z = np.exp((row - row.max()) / t[r])
        keep = np.ones(n, bool)
        if 0 < k[r] < n or p[r] < 1:
            order = np.argsort(-row, kind="stable")
            if 0 < k[r] < n:
                order = order[: int(k[r])]
            if p[r] < 1:
                mass = np.cumsum(z[order])
                order = order[: 1 + int(np.searchsorted(mass, p[r] * mass[-1]))]
            keep[:] = False
            keep[order] = True
        if least[r] > 0:
            keep &= z >= least[r]
        z[~keep] = 0.0
        mass = np.cumsum(z)
        i = min(int(np.searchsorted(mass, u[r] * mass[-1], side="right")), int(np.flatnonzero(z)[-1]))
        ids[r], prob[r] = i, z[i] / mass[-1]
    return {"ids": ids, "prob": prob}


def _exact_commit(s):
    n, nodes, longest = s["seqs"], s["nodes"], s["most_path"]
    words = s["mask"].cpu().numpy().view(np.uint64).reshape(n, nodes, -1)
    token, picked = (s[x].cpu().numpy().reshape(n, nodes) for x in ("tokens", "picked"))
    table, slots, base = s["table"].cpu().numpy(), s["slots"].tolist(), s["base"].tolist()
    out = {"k": s["k"].double(), "v": s["v"].double()}
    accepted, count = np.full((n, longest), -1), np.zeros(n, np.int64)
    src, dst = [], []
    for b in range(n):
        up = [-1] + [(sum(int(w) << (64 * i) for i, w in enumerate(words[b, c])) & ((1 << c) - 1)).bit_length() - 1 for c in range(1, nodes)]
        path, here = [], 0
        while here is not None:
            path.append(here)
            here = next((c for c in range(1, nodes) if up[c] == path[-1] and token[b, c] == picked[b, path[-1]]), None)
        for step, node in enumerate(path):
            accepted[b, step] = picked[b, node]
            at = [base[b] + node, base[b] + step]
            x, y = (int(table[slots[b], a // PAGE]) * PAGE + a % PAGE for a in at)
            src.append(x)
            dst.append(y)
        count[b] = len(path)
    src, dst = (torch.tensor(x, device=DEV) for x in (src, dst))
    for x in ("k", "v"):
        flat = out[x].view(s["layers"], -1, s["kv_dim"])
        flat[:, dst] = flat[:, src].clone()
    count = torch.from_numpy(count)
    return {**out, "accepted": torch.from_numpy(accepted).int(), "n": count.int(), "base": (count + torch.tensor(base)).int()}


def _exact_copy(s):
    out = {"k": s["k"].double(), "v": s["v"].double()}
    table = s["table"].cpu().numpy()
    for x in ("k", "v"):
        flat = out[x].view(s["layers"], -1, s["kv_dim"])
        for a, b, lo, hi in zip(*(s[y].tolist() for y in ("src", "dst", "start", "end"))):
            pos = np.arange(lo, hi)
            src, dst = (torch.from_numpy(table[c][pos // PAGE].astype(np.int64) * PAGE + pos % PAGE).to(DEV) for c in (a, b))
            flat[:, dst] = flat[:, src]
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"tree": _exact_tree, "sample": _exact_sample, "commit": _exact_commit, "copy": _exact_copy}[case["op"]](s)
