"""Cases of the paged K/V cache and of the attention over it.

Four operators on one cache of pages (a page is `page` rows of every layer's K and V; a slot is one sequence, its row of the
page table names its pages):

  tree     attention of drafted tokens over the cache: row i of a sequence sees the committed rows and, of the drafted rows that
           follow them, those that its mask names (its ancestors and itself); with a chain instead of a mask, those up to itself
  fork     sequences that continue another one: they share its full pages and get a copy of the page that is partly filled; then
           room for the next tokens, in the lowest free pages
  accept   the accepted path of a drafted tree: its rows move up behind the committed ones, the rest is cut off and the pages
           behind it are freed
  compact  pages move down into the holes of the pool, so that the used ones are the first ones

A pass of the last three starts from the page table that the program hands over (one copy of the integers), as a scheduler does
that keeps its own.
"""
import math

import numpy as np
import torch

own = False

NEG = float("-inf")
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
# heads (query, key/value) and head size of the layer shapes that the benchmark and the tests use
HEADS = {"9x3x64": (9, 3, 64), "14x2x64": (14, 2, 64), "32x4x64": (32, 4, 64), "16x8x128": (16, 8, 128)}


def listed():
    return [
        # one user, a small tree on a short conversation: what a step costs at least
        tree("tree-one", seqs=1, ctx=500, ragged=False, drafts=8, mask="tree", heads="16x8x128", q="bf16", kv="bf16", page=16),
        # plain decode of many users, one token each, at all lengths
        tree("decode-256", seqs=256, ctx=4096, ragged=True, drafts=1, mask="chain", heads="32x4x64", q="f16", kv="f16", page=16),
        # one long document and a wide tree
        tree("tree-long", seqs=1, ctx=131000, ragged=False, drafts=64, mask="tree", heads="16x8x128", q="bf16", kv="bf16", page=64),
        # many users with trees of different sizes; seven query heads to a key head, several tiles of rows to a sequence
        tree("tree-batch", seqs=48, ctx=6000, ragged=True, drafts=45, mask="tree", heads="14x2x64", q="f16", kv="f16", page=32),
        # 32-bit activations over a 16-bit cache, the layout of the engine's GPU path
        tree("tree-f32", seqs=8, ctx=2000, ragged=True, drafts=13, mask="tree", heads="9x3x64", q="f32", kv="f16", page=16),
        # a chunk of a prompt behind what the cache holds already
        tree("chain-chunk", seqs=4, ctx=9000, ragged=True, drafts=128, mask="chain", heads="16x8x128", q="bf16", kv="bf16", page=128),
        # one prompt, four samples of it
        pages("fork-few", "fork", seqs=1, per=4, ctx=500, grow=8, layers=28, row=2048, page=16, n_pages=96),
        # eight prompts, eight samples each
        pages("fork-many", "fork", seqs=8, per=8, ctx=300, grow=33, layers=28, row=2048, page=16, n_pages=400),
        # one user's accepted path
        pages("accept-one", "accept", seqs=1, per=4, ctx=900, grow=32, layers=28, row=2048, page=16, n_pages=64),
        # a batch of accepted paths
        pages("accept-batch", "accept", seqs=128, per=7, ctx=500, grow=63, layers=22, row=512, page=16, n_pages=4700),
        # a small pool, and one whose moved pages are past the on-chip cache
        pages("compact-small", "compact", seqs=6, per=0, ctx=100, grow=0, layers=24, row=256, page=16, n_pages=80),
        pages("compact-large", "compact", seqs=40, per=0, ctx=120, grow=0, layers=28, row=2048, page=16, n_pages=420),
    ]


def tree(name, **k):
    return {"name": name, "op": "tree", **k}


def pages(name, op, **k):
    return {"name": name, "op": op, **k}


def draw(rng):
    def log(a, b):
        return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))

    op = rng.choice(["tree", "tree", "tree", "fork", "accept", "compact"])
    page = rng.choice([8, 16, 16, 32, 64, 128])
    if op == "tree":
        heads = rng.choice(list(HEADS))
        q, kv = rng.choice([("bf16", "bf16"), ("bf16", "bf16"), ("f16", "f16"), ("f32", "f16"), ("f32", "bf16"), ("f32", "f32")])
        seqs = log(1, 128)
        ctx = log(min(40, 40000 // seqs), min(131000, (40000 if q == "f32" else 400000) // seqs))
        return dict(op="tree", seqs=seqs, ctx=ctx, ragged=rng.random() < 0.7, drafts=min(log(1, 128), max(1, 4096 // seqs), 8000000 // (seqs * ctx)),
                    mask=rng.choice(["tree", "tree", "chain"]), heads=heads, q=q, kv=kv, page=page)
    layers, row = rng.choice([(22, 512), (24, 256), (28, 2048), (30, 384)])
    seqs = log(1, 64)
    ctx = log(8, max(16, min(2000, int(4e8 / (2 * layers * row) / (2 * seqs)))))
    per, grow = (rng.randint(1, 6), log(1, 64)) if op != "compact" else (0, 0)
    if op == "fork":
        seqs = max(1, seqs // 4)
    if op == "accept":
        grow = max(grow, 2 * per + 1)

    def need():
        return seqs * (per + 1 if op == "fork" else 1) * (grow // page + 2) + seqs * (ctx // page + 2)

    while need() * page * row * 2 * layers > 3e8 and seqs > 1:
        seqs //= 2
    return dict(op=op, seqs=seqs, per=per, ctx=ctx, grow=grow, layers=layers, row=row, page=page,
                n_pages=int(need() * rng.uniform(1.2, 2.5)) + 4)


# ---- what a case holds, whatever the seed: lengths, trees, which rows were accepted ----

def shape_rng(case):
    return np.random.default_rng([len(case["op"])] + [int(case[k]) for k in ("seqs", "ctx", "page")])


def tree_shape(case):
    """Committed rows, drafted rows and parents (-1: a child of the last committed row) of each sequence."""
    rng = shape_rng(case)
    n = case["seqs"]
    ctx = rng.integers(0, case["ctx"] + 1, n) if case["ragged"] else np.full(n, case["ctx"])
    drafts = rng.integers(1, case["drafts"] + 1, n) if case["ragged"] else np.full(n, case["drafts"])
    drafts[0] = case["drafts"]
    parents = [np.array([-1 if j == 0 else int(rng.integers(max(-1, j - 12), j)) for j in range(d)]) for d in drafts]
    return ctx, drafts, parents


def page_shape(case):
    """Rows of each filled slot before the pass."""
    rng = shape_rng(case)
    return rng.integers(max(1, case["ctx"] // 2), case["ctx"] + 1, case["seqs"])


def work(case):
    if case["op"] == "tree":
        hq, hkv, hd = HEADS[case["heads"]]
        ctx, drafts, parents = tree_shape(case)
        rows, size = int(drafts.sum()), {"f32": 4, "f16": 2, "bf16": 2}
        seen = int((ctx * drafts).sum())
        for p in parents:
            depth = np.zeros(len(p), np.int64)
            for j, a in enumerate(p):
                depth[j] = 1 + (depth[a] if a >= 0 else 0)
            seen += int(depth.sum()) if case["mask"] == "tree" else len(p) * (len(p) + 1) // 2
        cache = int((ctx + drafts).sum()) * 2 * hkv * hd * size[case["kv"]]
        return {"bytes": cache + 2 * rows * hq * hd * size[case["q"]], "flops": 4 * seen * hq * hd}
    lens, page, stores = page_shape(case), case["page"], 2 * case["layers"]
    if case["op"] == "fork":
        moved, table = int((lens % page).sum()) * case["per"], int(lens.sum()) * case["per"] // page
    elif case["op"] == "accept":
        rows, counts = accepted_shape(case)
        moved, table = sum(int((a[:n] != np.arange(n)).sum()) for a, n in zip(rows, counts)), len(counts)
    else:
        moved, table = len(hole_pairs(case)) * page, case["n_pages"]
    return {"bytes": 2 * moved * case["row"] * stores + 8 * table, "flops": 0}


def accepted_shape(case):
    """Drafted rows that were accepted (ascending) and how many, per sequence. A row is taken from behind the places that the path
    moves to, or is at its place already, so that a pass over the same cache gives the same rows again."""
    rng = shape_rng(case)
    rows, counts = [], []
    for _ in range(case["seqs"]):
        n = int(rng.integers(1, case["per"] + 1))
        keep = int(rng.integers(0, n + 1))
        later = np.sort(rng.choice(np.arange(n, case["grow"]), n - keep, replace=False))
        rows.append(np.concatenate([np.arange(keep), later, np.zeros(case["per"] - n, np.int64)]).astype(np.int64))
        counts.append(n)
    return rows, np.array(counts)


def scattered(case):
    """Used pages of each slot for `compact`: anywhere in the pool."""
    lens = page_shape(case)
    order = shape_rng(case).permutation(case["n_pages"])
    held = np.concatenate([[0], np.cumsum(-(-lens // case["page"]))])
    return [order[a:b] for a, b in zip(held[:-1], held[1:])]


def hole_pairs(case):
    used = np.zeros(case["n_pages"], bool)
    for p in scattered(case):
        used[p] = True
    return np.flatnonzero(used[used.sum():])


# ---- inputs ----

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(shape, dtype):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)

    def whole(a, dtype=torch.int32):
        return torch.as_tensor(np.ascontiguousarray(a), device="cuda").to(dtype)

    s = {"case": case}
    return prepare_tree(case, seed, s, normal, whole) if case["op"] == "tree" else prepare_pages(case, seed, s, whole)


def prepare_tree(case, seed, s, normal, whole):
    hq, hkv, hd = HEADS[case["heads"]]
    page, n = case["page"], case["seqs"]
    ctx, drafts, parents = tree_shape(case)
    lens = ctx + drafts
    max_pages = int(-(-lens.max() // page))
    held = -(-lens // page)
    n_pages = int(held.sum()) + 3
    order = np.random.default_rng(seed).permutation(n_pages)
    table = np.full((n, max_pages), -1)
    at = 0
    for i in range(n):
        table[i, :held[i]] = order[at:at + held[i]]
        at += held[i]
    refs = np.zeros(n_pages, np.int64)
    refs[order[:at]] = 1
    starts = np.concatenate([[0], np.cumsum(drafts)])
    rows = int(starts[-1])
    words = -(-int(drafts.max()) // 64)
    mask = np.zeros((rows, words), np.uint64)
    for i, p in enumerate(parents):
        for j, a in enumerate(p):
            r = starts[i] + j
            if a >= 0:
                mask[r] = mask[starts[i] + a]
            mask[r, j // 64] |= np.uint64(1) << np.uint64(j % 64)
    s |= {"hq": hq, "hkv": hkv, "hd": hd, "page": page, "seqs": n, "rows": rows, "words": words, "max_drafts": int(drafts.max()),
          "max_len": int(lens.max()), "n_pages": n_pages, "max_pages": max_pages, "scale": 1.0 / math.sqrt(hd),
          "q": normal((rows, hq * hd), TYPES[case["q"]]), "out": torch.empty((rows, hq * hd), dtype=TYPES[case["q"]], device="cuda"),
          "k": normal((n_pages * page, hkv * hd), TYPES[case["kv"]]), "v": normal((n_pages * page, hkv * hd), TYPES[case["kv"]]),
          "table": whole(table), "lens": whole(lens), "refs": whole(refs), "q_start": whole(starts),
          "slots": whole(np.arange(n)), "mask": whole(mask.view(np.int64), torch.int64) if case["mask"] == "tree" else None}
    if own:
        s["pool"] = make_pool(s, [s["k"], s["v"]], s["k"].shape[1] * s["k"].element_size())
        s["work_bytes"] = context().tree_attn_workspace(rows=rows, n_q_heads=hq, n_kv_heads=hkv, head_dim=hd)
        s["work"] = torch.empty(max(16, s["work_bytes"]), dtype=torch.uint8, device="cuda")
    return s


def prepare_pages(case, seed, s, whole):
    page, n, n_pages, op = case["page"], case["seqs"], case["n_pages"], case["op"]
    lens = page_shape(case)
    per = case["per"] if op == "fork" else 0
    n_slots = n * (1 + per) + 1
    total = lens + case["grow"] if op == "accept" else lens
    max_pages = int(-(-(total.max() + case["grow"]) // page)) + 1
    table, refs, filled = np.full((n_slots, max_pages), -1), np.zeros(n_pages, np.int64), np.zeros(n_slots, np.int64)
    order = np.random.default_rng(seed).permutation(n_pages)
    sets = scattered(case) if op == "compact" else [None] * n
    at = 0
    for i in range(n):
        held = int(-(-total[i] // page))
        table[i, :held] = sets[i] if op == "compact" else order[at:at + held]
        at += held
        refs[table[i, :held]] += 1
        filled[i] = total[i]
    book = np.concatenate([table.reshape(-1), filled, refs])
    g = torch.Generator(device="cuda").manual_seed(seed)
    width = case["row"] // 2
    store = torch.randn((2 * case["layers"], n_pages * page, width), generator=g, device="cuda", dtype=torch.bfloat16)
    s |= {"page": page, "n_pages": n_pages, "n_slots": n_slots, "max_pages": max_pages, "store": store,
          "book0": whole(book), "book": whole(book)}
    a, b = n_slots * max_pages, n_slots * max_pages + n_slots
    s |= {"table": s["book"][:a].view(n_slots, max_pages), "lens": s["book"][a:b], "refs": s["book"][b:]}
    if op == "fork":
        src = np.repeat(np.arange(n), per)
        dst = n + np.arange(n * per)
        s |= {"src": whole(src), "dst": whole(dst), "every": whole(np.arange(n * (1 + per))),
              "room": whole(np.concatenate([lens, lens[src]]) + case["grow"])}
    elif op == "accept":
        rows, counts = accepted_shape(case)
        s |= {"slots": whole(np.arange(n)), "q_start": whole(np.arange(n + 1) * case["grow"]), "drafts": case["grow"],
              "accepted": whole(np.stack(rows)), "counts": whole(counts)}
    if own:
        s["pool"] = make_pool(s, list(store), case["row"])
    return s


# ---- the framework's calls ----

_context = None


def context():
    global _context
    if _context is None:
        import lokal_b200
        _context = lokal_b200.Context(torch.cuda.current_device())
    return _context


def make_pool(s, stores, row_bytes):
    import lokal_b200
    return lokal_b200.KvPool(context(), page_rows=s["page"], n_pages=s["n_pages"], n_slots=s["lens"].numel(), max_pages=s["max_pages"],
                             table=s["table"], lens=s["lens"], refs=s["refs"], stores=stores, row_bytes=row_bytes)


def own_run(s):
    stream = torch.cuda.current_stream().cuda_stream
    case = s["case"]
    if case["op"] == "tree":
        import lokal_b200
        context().tree_attn(s["pool"], s["q"], s["out"], k_store=0, v_store=1, slots=s["slots"], q_start=s["q_start"], n_seqs=s["seqs"],
                            rows=s["rows"], mask=s["mask"], mask_words=s["words"], n_q_heads=s["hq"], n_kv_heads=s["hkv"], head_dim=s["hd"],
                             scale=s["scale"], dtype=lokal_b200.dtype_id(s["q"]),
                            kv_dtype=lokal_b200.dtype_id(s["k"]), workspace=s["work"], workspace_bytes=s["work_bytes"], stream=stream)
        return s["out"]
    s["book"].copy_(s["book0"])
    if case["op"] == "fork":
        s["pool"].fork(s["src"], s["dst"], n=s["src"].numel(), stream=stream)
        s["pool"].reserve(s["every"], s["room"], n=s["every"].numel(), stream=stream)
    elif case["op"] == "accept":
        s["pool"].accept(s["slots"], s["q_start"], s["accepted"], s["counts"], n_seqs=case["seqs"], max_accept=case["per"], stream=stream)
    else:
        s["pool"].compact(stream=stream)
    return kept(s)


# ---- the plain forms ----

def run(s):
    if own:
        return own_run(s)
    op = s["case"]["op"]
    if op == "tree":
        return plain_tree(s)
    s["book"].copy_(s["book0"])
    {"fork": plain_fork, "accept": plain_accept, "compact": plain_compact}[op](s)
    return kept(s)


def kept(s):
    """The page table and the cache, whose values are copies: their bits have to be the same."""
    return {"book": s["book"], "store": s["store"].view(torch.int16)}


def plain_tree(s):
    hq, hkv, hd, page, n, length, most = s["hq"], s["hkv"], s["hd"], s["page"], s["seqs"], s["max_len"], s["max_drafts"]
    lens, starts = s["lens"].long(), s["q_start"].long()
    drafts = starts[1:] - starts[:-1]
    # the cache rows of every sequence, side by side
    pos = torch.arange(length, device="cuda")
    held = pos < lens[:, None]
    rows = s["table"].long()[:, pos // page].clamp(min=0) * page + pos % page
    k = s["k"][rows].float().view(n, length, hkv, hd).transpose(1, 2)
    v = s["v"][rows].float().view(n, length, hkv, hd).transpose(1, 2)
    # the drafted rows of every sequence, side by side
    j = torch.arange(most, device="cuda")
    there = j < drafts[:, None]
    at = (starts[:-1, None] + j).clamp(max=s["rows"] - 1)
    q = s["q"][at].float().view(n, most, hkv, hq // hkv, hd).permute(0, 2, 3, 1, 4).reshape(n, hkv, -1, hd)
    # which of its sequence's rows a drafted row sees
    node = pos - (lens - drafts)[:, None]
    if s["mask"] is None:
        seen = node[:, None, :] <= j[:, None]
    else:
        bits = (s["mask"][:, :, None] >> torch.arange(64, device="cuda")) & 1
        bits = bits.view(s["rows"], -1)[at]
        which = node.clamp(0, bits.shape[2] - 1)[:, None, :].expand(n, most, length)
        seen = (node < 0)[:, None, :] | (bits.gather(2, which) == 1)
    seen = seen & held[:, None, :]
    seen = seen[:, None, None].expand(n, 1, hq // hkv, most, length).reshape(n, 1, -1, length)
    score = (q @ k.transpose(2, 3) * s["scale"]).masked_fill(~seen, NEG)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == NEG, torch.zeros_like(top), top)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    out = (p @ v) / torch.where(total == 0, torch.ones_like(total), total)
    out = out.view(n, hkv, hq // hkv, most, hd).permute(0, 3, 1, 2, 4).reshape(n, most, hq * hd)
    s["out"].copy_(out[there])
    return s["out"]


def lowest_free(refs):
    """Free pages in ascending order, then as many -1 as there are others."""
    free = refs == 0
    place = torch.where(free, free.cumsum(0) - 1, refs.numel())
    out = torch.full((refs.numel() + 1,), -1, device="cuda", dtype=torch.long)
    out[place] = torch.arange(refs.numel(), device="cuda")
    out[-1] = -1
    return out


def plain_fork(s):
    page, table, lens, refs, store = s["page"], s["table"], s["lens"], s["refs"], s["store"]
    src, dst = s["src"].long(), s["dst"].long()
    col = torch.arange(s["max_pages"], device="cuda")
    n = lens[src].long()
    full, part = n // page, (n % page != 0)
    fresh = lowest_free(refs)[(part.cumsum(0) - 1).clamp(min=0)]
    old = table[src]
    shared = col < full[:, None]
    table[dst] = torch.where(shared, old, torch.where((col == full[:, None]) & part[:, None], fresh[:, None].int(), -1))
    lens[dst] = lens[src]
    refs.index_add_(0, old.clamp(min=0).long().view(-1), shared.int().view(-1))
    refs.index_add_(0, fresh.clamp(min=0), part.int())
    i = torch.arange(page, device="cuda")
    last = old.gather(1, ((n - 1) // page)[:, None])[:, 0].long()
    # behind the filled rows, the first is copied again (and where there is no such page, a row to itself)
    i = torch.where(i < (n % page)[:, None], i, 0)
    get = last[:, None] * page + i
    put = torch.where(part, fresh, last)[:, None] * page + i
    store[:, put.view(-1)] = store[:, get.view(-1)]
    # room for the next tokens
    slots, room = s["every"].long(), s["room"].long()
    have, want = -(-lens[slots].long() // page), -(-room // page)
    need = (want - have).clamp(min=0)
    new = (col >= have[:, None]) & (col < want[:, None])
    rank = (need.cumsum(0) - need)[:, None] + col - have[:, None]
    got = lowest_free(refs)[torch.where(new, rank, 0)]
    table[slots] = torch.where(new, got.int(), table[slots])
    refs.index_add_(0, torch.where(new, got, 0).view(-1), new.int().view(-1))
    lens[slots] = torch.maximum(lens[slots], s["room"])


def plain_accept(s):
    page, table, lens, refs, store = s["page"], s["table"], s["lens"], s["refs"], s["store"]
    slots, take, count = s["slots"].long(), s["accepted"].long(), s["counts"].long()
    base = lens[slots].long() - s["drafts"]
    j = torch.arange(take.shape[1], device="cuda").expand_as(take)
    there = j < count[:, None]
    # where there is no row to move, the first move is made again (or, with none, a row moves to itself)
    take = torch.where(there, take, torch.where(count > 0, take[:, 0], 0)[:, None])
    j = torch.where(there, j, 0)
    pages_of = table[slots].long()

    def row(p):
        return pages_of.gather(1, p // page) * page + p % page

    store[:, row(base[:, None] + j).view(-1)] = store[:, row(base[:, None] + take).view(-1)]
    now = base + count
    col = torch.arange(s["max_pages"], device="cuda")
    gone = (col >= -(-now // page)[:, None]) & (pages_of >= 0)
    refs.index_add_(0, pages_of.clamp(min=0).view(-1), -gone.int().view(-1))
    table[slots] = torch.where(gone, -1, table[slots])
    lens[slots] = now.int()


def plain_compact(s):
    table, refs, store = s["table"], s["refs"], s["store"]
    used = refs > 0
    index = torch.arange(refs.numel(), device="cuda")
    low = index < used.sum()
    to = (low & ~used).nonzero()[:, 0]
    source = (~low & used).nonzero()[:, 0]
    both = store.view(store.shape[0], refs.numel(), -1)
    both[:, to] = both[:, source]
    place = index.clone()
    place[source] = to
    table.copy_(torch.where(table >= 0, place[table.clamp(min=0).long()].int(), -1))
    refs[to] = refs[source]
    refs[source] = 0


# ---- from the definition, in 64 bits ----

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "tree":
        return exact_tree(case, s)
    return {"book": {"fork": exact_fork, "accept": exact_accept, "compact": exact_compact}[case["op"]](case, s), "store": None}


def exact_tree(case, s):
    ctx, drafts, parents = tree_shape(case)
    group = s["hq"] // s["hkv"]
    out = torch.zeros((s["rows"], s["hq"], s["hd"]), dtype=torch.float64, device="cuda")
    table, at = s["table"].cpu().numpy(), 0
    for i in range(case["seqs"]):
        c, d = int(ctx[i]), int(drafts[i])
        where = np.arange(c + d)
        where = torch.as_tensor(table[i, where // case["page"]].astype(np.int64) * case["page"] + where % case["page"], device="cuda")
        sees = np.zeros((d, c + d), bool)
        sees[:, :c] = True
        for j in range(d):
            if case["mask"] == "chain":
                sees[j, c:c + j + 1] = True
            else:
                a = j
                while a >= 0:
                    sees[j, c + a] = True
                    a = int(parents[i][a])
        sees = torch.as_tensor(sees, device="cuda")
        for h in range(s["hkv"]):
            cols = slice(h * s["hd"], (h + 1) * s["hd"])
            k, v = s["k"][where, cols].double(), s["v"][where, cols].double()
            for e in range(h * group, (h + 1) * group):
                q = s["q"][at:at + d, e * s["hd"]:(e + 1) * s["hd"]].double()
                z = (q @ k.T) / math.sqrt(s["hd"])
                z[~sees] = NEG
                w = torch.softmax(z, 1)
                out[at:at + d, e] = w @ v
        at += d
    return out.view(s["rows"], -1)


def as_lists(s):
    table, lens, refs = s["table"].cpu().numpy().copy(), s["lens"].cpu().numpy().copy(), s["refs"].cpu().numpy().copy()
    return table, lens, refs


def joined(table, lens, refs):
    return torch.as_tensor(np.concatenate([table.reshape(-1), lens, refs]).astype(np.int32))


def exact_fork(case, s):
    table, lens, refs = as_lists(s)
    page = case["page"]

    def take():
        p = int(np.flatnonzero(refs == 0)[0])
        refs[p] = 1
        return p

    for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
        for c in range(lens[a] // page):
            table[b, c] = table[a, c]
            refs[table[a, c]] += 1
        if lens[a] % page:
            table[b, lens[a] // page] = take()
        lens[b] = lens[a]
    for a, room in zip(s["every"].tolist(), s["room"].tolist()):
        for c in range(-(-int(lens[a]) // page), -(-room // page)):
            table[a, c] = take()
        lens[a] = max(lens[a], room)
    return joined(table, lens, refs)


def exact_accept(case, s):
    table, lens, refs = as_lists(s)
    for i, n in enumerate(s["counts"].tolist()):
        lens[i] = lens[i] - case["grow"] + n
        for c in range(-(-int(lens[i]) // case["page"]), table.shape[1]):
            if table[i, c] >= 0:
                refs[table[i, c]] -= 1
                table[i, c] = -1
    return joined(table, lens, refs)


def exact_compact(case, s):
    table, lens, refs = as_lists(s)
    low, high = 0, len(refs) - 1
    holes = [p for p in range(len(refs)) if refs[p] == 0]
    live = len(refs) - len(holes)
    movers = [p for p in range(live, len(refs)) if refs[p] > 0]
    for low, high in zip(holes, movers):
        table[table == high] = low
        refs[low], refs[high] = refs[high], 0
    return joined(table, lens, refs)
