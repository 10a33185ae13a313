"""Performance cases of the operators for long caches (``dgi.ops.longctx``): the append that keeps page bounds, their rebuilding, the
selection of pages by them, attention over selected pages, attention of drafted trees.

Sizes are those of the Llama-3, Qwen2.5 and GLM-4 attention layers (heads, kv heads of 64 or 128 dims, pages of 16 tokens).  ``seqs`` sequences
of ``low`` to ``high`` tokens bring ``rows`` rows each: 1 for decode steps, more for the last rows of a prompt portion.

Kinds of case (``kind``):

* ``append``   rotate queries and keys of a step's rows, write keys and values into the paged cache, bring the pages' bounds up to date
* ``bounds``   the bounds of ``pages`` pages from the keys that they hold
* ``select``   the ``count`` pages of a context that each row's group of heads is to read
* ``attend``   attention of every row over its selected pages
* ``tree``     attention of up to ``nodes`` drafted tokens a sequence over its cache, each seeing its ancestors among them

``own``: whether ``run`` goes through the framework's kernels; otherwise it computes the same from elementary operations.
"""
import math

import torch

own = False

DEV = "cuda"
PAGE = 16
THETA = 500000.0
F32, F64, BF16, I32 = torch.float32, torch.float64, torch.bfloat16, torch.int32


def listed():
    return [
        # one user chatting: a row of an 8B model, bound by latency
        {"name": "append_1", "kind": "append", "heads": 32, "kv": 8, "dim": 128, "rd": 128, "mode": 0, "seqs": 1, "rows": 1, "low": 600, "high": 600},
        # ragged prompt portions of a 70B model, most behind a cached prefix
        {"name": "append_prompts", "kind": "append", "heads": 64, "kv": 8, "dim": 128, "rd": 128, "mode": 0, "seqs": 5, "rows": 823, "low": 900,
         "high": 5000},
        # a short prefix that came from another worker
        {"name": "bounds_37", "kind": "bounds", "kv": 4, "dim": 128, "pages": 37},
        # a long document that comes back from the host tier
        {"name": "bounds_16k", "kind": "bounds", "kv": 8, "dim": 128, "pages": 16384},
        # one user with a long chat
        {"name": "select_1", "kind": "select", "heads": 32, "kv": 8, "dim": 128, "seqs": 1, "rows": 1, "low": 8000, "high": 8000, "count": 64},
        # a busy server of long contexts
        {"name": "select_64", "kind": "select", "heads": 64, "kv": 8, "dim": 128, "seqs": 64, "rows": 1, "low": 4000, "high": 32000, "count": 128},
        # portions of two long prompts, seven query heads on each kv head
        {"name": "select_prompts", "kind": "select", "heads": 28, "kv": 4, "dim": 128, "seqs": 2, "rows": 509, "low": 6000, "high": 16000, "count": 64},
        # one user with a very long chat
        {"name": "attend_1", "kind": "attend", "heads": 32, "kv": 8, "dim": 128, "seqs": 1, "rows": 1, "low": 32000, "high": 32000, "count": 128},
        # a busy server of long contexts
        {"name": "attend_64", "kind": "attend", "heads": 64, "kv": 8, "dim": 128, "seqs": 64, "rows": 1, "low": 2000, "high": 16000, "count": 128},
        # portions of two long prompts
        {"name": "attend_prompts", "kind": "attend", "heads": 28, "kv": 4, "dim": 128, "seqs": 2, "rows": 509, "low": 6000, "high": 16000, "count": 64},
        # one user, a short draft after a short chat
        {"name": "tree_1", "kind": "tree", "heads": 32, "kv": 8, "dim": 128, "seqs": 1, "nodes": 8, "low": 600, "high": 600},
        # sixteen users of a 70B model, full drafts of ragged size
        {"name": "tree_16", "kind": "tree", "heads": 64, "kv": 8, "dim": 128, "seqs": 16, "nodes": 60, "low": 1000, "high": 8000},
    ]


#: heads, kv heads, dims, rotated dims, pairing: Llama-3 8B and 70B, Qwen2.5 7B and 0.5B, GLM-4 9B, one of the test models
LAYERS = [(32, 8, 128, 128, 0), (64, 8, 128, 128, 0), (28, 4, 128, 128, 0), (14, 2, 64, 64, 0), (32, 2, 128, 64, 1), (8, 1, 64, 64, 0)]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["append", "bounds", "select", "attend", "tree"])
    heads, kv, dim, rd, mode = rng.choice(LAYERS)
    if kind == "bounds":
        return {"kind": kind, "kv": kv, "dim": dim, "pages": _log(rng, 4, 16384)}
    layer = {"kind": kind, "heads": heads, "kv": kv, "dim": dim}
    if kind == "append":
        seqs = _log(rng, 1, 64)
        rows = 1 if rng.random() < 0.4 else _log(rng, 2, max(2, 4000 // seqs))
        low = rows + _log(rng, 1, 2000)
        return {**layer, "rd": rd, "mode": mode, "seqs": seqs, "rows": rows, "low": low, "high": low + _log(rng, 1, 2000)}
    if kind == "tree":
        seqs, nodes = _log(rng, 1, 16), _log(rng, 2, 60)
        low = nodes + _log(rng, 16, 3000)
        return {**layer, "seqs": seqs, "nodes": nodes, "low": low, "high": low + _log(rng, 1, 2000)}
    prompt = rng.random() < 0.4
    seqs = rng.choice([1, 2]) if prompt else _log(rng, 1, 64)
    rows = _log(rng, 2, min(28000 // heads, 4000 // kv) // seqs) if prompt else 1
    low = rows + _log(rng, 100, 8000)
    high = low + _log(rng, 100, 7000 if kind == "attend" or prompt else 20000)
    return {**layer, "seqs": seqs, "rows": rows, "low": low, "high": high, "count": rng.choice([16, 32, 50, 64]) if prompt else rng.choice([16, 32, 64, 100, 128])}


def _lengths(case):
    """Tokens of each sequence, spread over low to high; the last is the longest."""
    n, low, high = case["seqs"], case["low"], case["high"]
    return [low + int((high - low) * ((i + 1) * 0.618034 % 1.0)) for i in range(n - 1)] + [high]


def _nodes(case):
    """Nodes of each sequence's tree: ragged, the last one's full."""
    n, most = case["seqs"], case["nodes"]
    return [max(1, most - (i * 7) % max(1, most // 2)) for i in range(1, n)] + [most]


def _pages_of(lengths):
    return [-(-x // PAGE) for x in lengths]


def _tables(lengths, gen):
    """Block tables [seqs, longest] over shuffled pages (page 0 belongs to nobody), and the pool's pages."""
    need = _pages_of(lengths)
    ids = torch.randperm(sum(need), generator=gen, device=DEV).to(I32) + 1
    table = torch.zeros(len(need), max(need), dtype=I32, device=DEV)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = ids[at:at + n]
        at += n
    return table, sum(need) + 1


def _randn(gen, *shape, dtype=BF16):
    return torch.randn(*shape, generator=gen, device=DEV, dtype=dtype)


def _keys(gen, pages, kv, dim):
    """Cached keys: every channel has a level of its own, every page a subject, every token what is new in it."""
    return (_randn(gen, pages, kv, PAGE, dim) * 0.7).add_(_randn(gen, pages, kv, 1, dim) * 0.7).add_(_randn(gen, 1, kv, 1, dim))


def _queries(gen, case, tables, lengths, pool):
    """Queries that look for the subject of some page of their context; neighbouring rows of a prompt mostly for the same one."""
    seqs, rows, kv, dim = case["seqs"], case["rows"], case["kv"], case["dim"]
    group = case["heads"] // kv
    spots = -(-rows // 32)
    far = torch.tensor(_pages_of(lengths), device=DEV)[:, None] - 1
    at = (torch.rand(seqs, spots, generator=gen, device=DEV) * far).long()
    page = torch.gather(tables.long(), 1, at).repeat_interleave(32, 1)[:, :rows]
    subject = pool[page]                                                     # [seqs, rows, kv, dim]
    q = subject[:, :, :, None] * 0.8 + _randn(gen, seqs, rows, kv, group, dim)
    return q.reshape(seqs * rows, kv * group * dim).to(BF16)


def _selection(gen, case, lengths):
    """A selection like the operator's: the first and last page of every row, others that neighbouring rows mostly share, ascending."""
    seqs, rows, kv, count = case["seqs"], case["rows"], case["kv"], case["count"]
    most = max(_pages_of(lengths))
    ctx = torch.tensor(lengths, device=DEV)[:, None] - rows + 1 + torch.arange(rows, device=DEV)
    have = (ctx + PAGE - 1) // PAGE                                          # [seqs, rows]
    shared = torch.rand(seqs, -(-rows // 32), kv, most, generator=gen, device=DEV).repeat_interleave(32, 1)[:, :rows]
    want = shared * 4 + torch.rand(seqs, rows, kv, most, generator=gen, device=DEV)
    page = torch.arange(most, device=DEV)
    want = torch.where((page == 0) | (page == have[..., None, None] - 1), 9.0, want)
    want = torch.where(page < have[..., None, None], want, -1.0)
    best = want.topk(min(count, most), -1)
    sel = torch.where(best.values >= 0, best.indices, most).sort(-1).values
    sel = torch.where(sel < most, sel, -1)
    sel = torch.nn.functional.pad(sel, (0, count - sel.shape[-1]), value=-1)
    return sel.reshape(seqs * rows, kv, count).to(I32).contiguous()


def _angles(length, rd):
    inv = 1.0 / THETA ** (torch.arange(0, rd, 2, dtype=F64, device=DEV) / rd)
    turn = torch.outer(torch.arange(length, dtype=F64, device=DEV), inv)
    return torch.cat([turn.cos(), turn.sin()], -1).float()


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(int(seed))
    kind, kv, dim = case["kind"], case["kv"], case["dim"]
    s = dict(case)
    if kind == "bounds":
        n = case["pages"]
        s["k_cache"] = _keys(gen, n + n // 8 + 1, kv, dim)
        s["bounds"] = _randn(gen, n + n // 8 + 1, kv, 2, dim)
        s["pages_at"] = torch.randperm(n + n // 8 + 1, generator=gen, device=DEV)[:n].to(I32)
        s["lens"] = torch.full((n,), PAGE, dtype=I32, device=DEV)
        s["lens"][-1] = 1 + seed % PAGE                                      # the sequence's last page is not full
        return s
    lengths = _lengths(case)
    tables, pool = _tables(lengths, gen)
    s["tables"] = tables
    if kind == "tree":
        nodes = _nodes(case)
        most = max(nodes)
        s["ctx"] = torch.tensor(lengths, dtype=I32, device=DEV)
        s["cu"] = torch.tensor([sum(nodes[:i]) for i in range(len(nodes) + 1)], dtype=I32, device=DEV)
        s["k_cache"], s["v_cache"] = _keys(gen, pool, kv, dim), _randn(gen, pool, kv, PAGE, dim)
        s["q"] = _randn(gen, sum(nodes), case["heads"] * dim)
        parent = (torch.rand(len(nodes), most, generator=gen, device=DEV) * torch.arange(most, device=DEV)).long().cpu()
        bits = torch.zeros(len(nodes), 64, dtype=torch.int64)
        for a in range(most):
            up = bits.gather(1, parent[:, a:a + 1])[:, 0] if a else torch.zeros(len(nodes), dtype=torch.int64)
            bits[:, a] = up | (1 << a)
        s["mask"] = bits.to(DEV)
        s["node_row"] = torch.tensor([[sum(nodes[:i]) + min(a, n - 1) for a in range(most)] for i, n in enumerate(nodes)], device=DEV)
        s["row_at"] = torch.tensor([i * most + a for i, n in enumerate(nodes) for a in range(n)], device=DEV)
        s["node_count"] = torch.tensor(nodes, device=DEV)
        return s
    rows, seqs = case["rows"], case["seqs"]
    ends = torch.tensor(lengths, dtype=I32, device=DEV)[:, None]
    s["ctx"] = (ends - rows + 1 + torch.arange(rows, dtype=I32, device=DEV)).reshape(-1).contiguous()
    s["seq"] = torch.arange(seqs, dtype=I32, device=DEV).repeat_interleave(rows)
    if kind == "append":
        pos = s["ctx"] - 1
        s["positions"] = pos
        page = torch.gather(tables.long(), 1, (pos.long() // PAGE).view(seqs, rows)).reshape(-1)
        s["slots"] = (page * PAGE + pos % PAGE).to(I32)
        s["cos_sin"] = _angles(case["high"] + 1, case["rd"])
        s["qkv"] = _randn(gen, seqs * rows, (case["heads"] + 2 * kv) * dim)
        s["k_cache"], s["v_cache"] = _keys(gen, pool, kv, dim), _randn(gen, pool, kv, PAGE, dim)
        s["bounds"] = torch.stack([s["k_cache"].amin(2), s["k_cache"].amax(2)], 2)
    elif kind == "select":
        middle = _randn(gen, pool, kv, dim) * 0.7
        level = _randn(gen, 1, kv, dim)
        reach = 1.0 + 0.6 * torch.rand(pool, kv, 2, dim, generator=gen, device=DEV)
        s["bounds"] = torch.stack([middle + level - reach[:, :, 0], middle + level + reach[:, :, 1]], 2).to(BF16)
        s["q"] = _queries(gen, case, tables, lengths, middle)
        s["first"], s["recent"] = 1, 2
    else:
        s["k_cache"], s["v_cache"] = _keys(gen, pool, kv, dim), _randn(gen, pool, kv, PAGE, dim)
        s["q"] = _queries(gen, case, tables, lengths, s["k_cache"][:, :, 3])
        s["pages"] = _selection(gen, case, lengths)
    return s


def run(s):
    kind = s["kind"]
    if own:
        from dgi.ops import longctx
        if kind == "append":
            q = longctx.rope_cache_bounds(s["qkv"], s["positions"], s["cos_sin"], s["heads"], s["kv"], s["dim"], s["slots"], s["k_cache"],
                                          s["v_cache"], s["bounds"], s["mode"])
            return q, s["k_cache"], s["v_cache"], s["bounds"]
        if kind == "bounds":
            longctx.page_bounds(s["k_cache"], s["bounds"], s["pages_at"], s["lens"])
            return s["bounds"]
        if kind == "select":
            return longctx.select_pages(s["q"], s["bounds"], s["tables"], s["ctx"], s["heads"], s["kv"], PAGE, s["count"], s["first"],
                                        s["recent"], row_seq=s["seq"])
        if kind == "attend":
            return longctx.paged_selected(s["q"], s["k_cache"], s["v_cache"], s["tables"], s["ctx"], s["pages"], s["heads"], s["kv"],
                                          1.0 / math.sqrt(s["dim"]), row_seq=s["seq"])
        return longctx.paged_tree(s["q"], s["k_cache"], s["v_cache"], s["tables"], s["cu"], s["ctx"], s["mask"], s["heads"], s["kv"],
                                  1.0 / math.sqrt(s["dim"]), max_nodes=s["nodes"])
    return {"append": _append, "bounds": _bounds, "select": _select, "attend": _attend, "tree": _tree}[kind](s)


# ---- plain forms -----------------------------------------------------------------------------------------------------------------------

def _rotated(x, cs, mode):
    """x [rows, heads, dim] in fp32, the first dims rotated by the rows [cos | sin] of cs."""
    half = cs.shape[-1] // 2
    cos, sin, part, rest = cs[:, None, :half], cs[:, None, half:], x[..., :2 * half], x[..., 2 * half:]
    if mode == 0:
        a, b = part[..., :half], part[..., half:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = part[..., 0::2], part[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([turned, rest], -1)


def _append(s):
    nh, kv, dim, T = s["heads"], s["kv"], s["dim"], s["qkv"].shape[0]
    rows = s["qkv"].view(T, nh + 2 * kv, dim)
    turned = _rotated(rows[:, :nh + kv].float(), s["cos_sin"][s["positions"].long()], s["mode"]).to(BF16)
    q, k, v = turned[:, :nh], turned[:, nh:], rows[:, nh + kv:]
    slots = s["slots"].long()
    page, off = slots // PAGE, slots % PAGE
    s["k_cache"][page, :, off] = k
    s["v_cache"][page, :, off] = v
    low, high = s["bounds"][:, :, 0].float(), s["bounds"][:, :, 1].float()
    begun = torch.zeros(low.shape[0], dtype=F32, device=DEV).index_add_(0, page, (off == 0).float())[:, None, None] > 0
    low, high = torch.where(begun, math.inf, low), torch.where(begun, -math.inf, high)
    at = page[:, None, None].expand(-1, kv, dim)
    low = low.scatter_reduce(0, at, k.float(), "amin")
    high = high.scatter_reduce(0, at, k.float(), "amax")
    s["bounds"][:] = torch.stack([low, high], 2).to(BF16)
    return q.reshape(T, nh * dim), s["k_cache"], s["v_cache"], s["bounds"]


def _bounds(s):
    k = s["k_cache"][s["pages_at"].long()].float()
    there = (torch.arange(PAGE, device=DEV) < s["lens"][:, None])[:, None, :, None]
    low, high = torch.where(there, k, math.inf).amin(2), torch.where(there, k, -math.inf).amax(2)
    s["bounds"][s["pages_at"].long()] = torch.stack([low, high], 2).to(BF16)
    return s["bounds"]


def _select(s):
    seqs, rows, kv, dim, count = s["seqs"], s["rows"], s["kv"], s["dim"], s["count"]
    # 64 bits: a page at the border is kept or not, whatever the order of the sum
    q = s["q"].view(seqs, rows, kv, -1, dim).to(F64)
    up, down = q.clamp(min=0).sum(3).transpose(1, 2), q.clamp(max=0).sum(3).transpose(1, 2)          # [seqs, kv, rows, dim]
    b = s["bounds"][s["tables"].long()].to(F64).permute(0, 2, 3, 4, 1)                               # [seqs, kv, 2, dim, pages]
    score = up @ b[:, :, 1] + down @ b[:, :, 0]
    score = torch.nan_to_num(score, nan=torch.finfo(F64).min)
    have = ((s["ctx"].view(seqs, 1, rows, 1) + PAGE - 1) // PAGE).long()
    page = torch.arange(score.shape[-1], device=DEV)
    score = torch.where((page < s["first"]) | (page >= have - s["recent"]), math.inf, score)
    score = torch.where(page < have, score, -math.inf)
    order = score.sort(dim=-1, descending=True, stable=True).indices[..., :count]
    order = torch.where(order < have, order, score.shape[-1]).sort(-1).values
    order = torch.where(order < score.shape[-1], order, -1)
    order = torch.nn.functional.pad(order, (0, count - order.shape[-1]), value=-1)
    return order.transpose(1, 2).reshape(seqs * rows, kv, count).to(I32)


def _softmax(x):
    e = torch.exp(x - x.amax(-1, keepdim=True).clamp(min=-1e30))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total > 0, total, 1.0)


def _attend(s):
    kv, dim, count, T = s["kv"], s["dim"], s["count"], s["q"].shape[0]
    pages = s["pages"].long()
    at = s["tables"].long()[s["seq"].long()[:, None, None], pages.clamp(min=0)]
    head = torch.arange(kv, device=DEV)[None, :, None]
    k = s["k_cache"][at, head].view(T, kv, count * PAGE, dim).float()
    v = s["v_cache"][at, head].view(T, kv, count * PAGE, dim).float()
    key = (pages[..., None] * PAGE + torch.arange(PAGE, device=DEV)).view(T, kv, 1, -1)
    seen = (key < s["ctx"].view(T, 1, 1, 1)) & (pages >= 0).repeat_interleave(PAGE, -1).unsqueeze(2)
    q = s["q"].view(T, kv, -1, dim).float()
    score = (q @ k.transpose(2, 3).contiguous()) * (1.0 / math.sqrt(dim))
    return (_softmax(torch.where(seen, score, -math.inf)) @ v).reshape(T, -1).to(BF16)


def _tree(s):
    kv, dim, seqs, most = s["kv"], s["dim"], s["seqs"], s["nodes"]
    tables = s["tables"].long()
    keys = tables.shape[1] * PAGE
    k = s["k_cache"][tables].transpose(1, 2).reshape(seqs, kv, keys, dim).float()
    v = s["v_cache"][tables].transpose(1, 2).reshape(seqs, kv, keys, dim).float()
    q = s["q"][s["node_row"]].view(seqs, most, kv, -1, dim).permute(0, 2, 3, 1, 4).reshape(seqs, kv, -1, dim).float()
    begin = (s["ctx"] - s["node_count"])[:, None, None]                                              # the tree's first key
    node = torch.arange(keys, device=DEV) - begin                                                    # [seqs, 1, keys]
    bit = (s["mask"][:, :most, None] >> node.clamp(0, 63)) & 1
    seen = (node < 0) | ((bit == 1) & (node < s["node_count"][:, None, None]))
    score = (q @ k.transpose(2, 3).contiguous()) * (1.0 / math.sqrt(dim))
    score = torch.where(seen[:, None, None], score.view(seqs, kv, -1, most, keys), -math.inf)
    out = _softmax(score).view(seqs, kv, -1, keys) @ v
    out = out.view(seqs, kv, -1, most, dim).permute(0, 3, 1, 2, 4).reshape(seqs * most, -1)
    return out[s["row_at"]].to(BF16)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------------------------

def work(case):
    kind, kv, dim = case["kind"], case["kv"], case["dim"]
    page = PAGE * kv * dim * 2                                               # bytes of a page's keys
    edge = kv * 2 * dim * 2                                                  # bytes of a page's bounds
    if kind == "bounds":
        return {"bytes": case["pages"] * (page + edge + 8), "flops": 2 * case["pages"] * PAGE * kv * dim}
    nh, lengths = case["heads"], _lengths(case)
    if kind == "tree":
        nodes = _nodes(case)
        return {"bytes": sum(lengths) * kv * dim * 4 + sum(nodes) * (nh * dim * 4 + 8),
                "flops": 4 * nh * dim * sum(n * c for n, c in zip(nodes, lengths))}
    rows = case["rows"]
    T = rows * case["seqs"]
    if kind == "append":
        touched = sum(-(-c // PAGE) - (c - rows) // PAGE for c in lengths)
        begun = sum(1 for c in lengths if (c - rows) % PAGE)                 # pages that go on: their bounds are read
        return {"bytes": T * (nh + 2 * kv) * dim * 4 + T * (case["rd"] * 4 + 8) + (touched + begun) * edge,
                "flops": 3 * T * (nh + kv) * case["rd"]}
    pages = _pages_of(lengths)
    if kind == "select":
        return {"bytes": sum(pages) * (edge + 4) + T * (nh * dim * 2 + kv * case["count"] * 4 + 8),
                "flops": 4 * dim * kv * rows * sum(pages)}
    kept = [min(n, case["count"]) for n in pages]
    read = sum(min(n, rows * m) for n, m in zip(pages, kept))
    return {"bytes": 2 * read * page + T * (nh * dim * 4 + kv * case["count"] * 4 + 8), "flops": 4 * nh * dim * PAGE * rows * sum(kept)}


# ---- from the definitions, in 64 bits --------------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    kind, kv, dim = case["kind"], case["kv"], case["dim"]
    if kind == "bounds":
        out = s["bounds"].double()
        full, last = s["pages_at"].long()[:-1], int(s["pages_at"][-1])
        keys = s["k_cache"].double()
        out[full, :, 0], out[full, :, 1] = keys[full].min(2).values, keys[full].max(2).values
        end = keys[last, :, :int(s["lens"][-1])]
        out[last, :, 0], out[last, :, 1] = end.min(1).values, end.max(1).values
        return out
    nh = case["heads"]
    group = nh // kv
    lengths = _lengths(case)
    if kind == "append":
        T, rd = s["qkv"].shape[0], case["rd"]
        x = s["qkv"].double().view(T, -1, dim)
        y = x.clone()
        table = s["cos_sin"].double()[s["positions"].long()]
        for i in range(rd // 2):
            a, b = (i, i + rd // 2) if case["mode"] == 0 else (2 * i, 2 * i + 1)
            c, d = table[:, i, None], table[:, rd // 2 + i, None]
            y[:, :nh + kv, a] = x[:, :nh + kv, a] * c - x[:, :nh + kv, b] * d
            y[:, :nh + kv, b] = x[:, :nh + kv, a] * d + x[:, :nh + kv, b] * c
        k, v, edges = s["k_cache"].double(), s["v_cache"].double(), s["bounds"].double()
        for i in range(case["seqs"]):
            lo, hi = lengths[i] - case["rows"], lengths[i]
            for p in range(lo // PAGE, -(-hi // PAGE)):
                t0, t1, at = max(lo, p * PAGE), min(hi, (p + 1) * PAGE), int(s["tables"][i, p])
                r = i * case["rows"] - lo
                new = y[r + t0:r + t1, nh:nh + kv]
                k[at, :, t0 - p * PAGE:t1 - p * PAGE] = new.transpose(0, 1)
                v[at, :, t0 - p * PAGE:t1 - p * PAGE] = y[r + t0:r + t1, nh + kv:].transpose(0, 1)
                low, high = new.min(0).values, new.max(0).values
                if t0 > p * PAGE:
                    low, high = torch.minimum(low, edges[at, :, 0]), torch.maximum(high, edges[at, :, 1])
                edges[at, :, 0], edges[at, :, 1] = low, high
        return y[:, :nh].reshape(T, -1), k, v, edges
    if kind == "tree":
        q = s["q"].double().view(-1, kv, group, dim)
        out = torch.zeros_like(q)
        row = 0
        for i, (n, c) in enumerate(zip(_nodes(case), lengths)):
            at = s["tables"][i, :-(-c // PAGE)].long()
            see = torch.ones(n, c, dtype=torch.bool)
            for a, bits in enumerate(s["mask"][i, :n].tolist()):
                see[a, c - n:] = torch.tensor([bool(bits >> b & 1) for b in range(n)])
            see = see.to(DEV)
            for h in range(kv):
                k, v = s["k_cache"][at, h].reshape(-1, dim)[:c].double(), s["v_cache"][at, h].reshape(-1, dim)[:c].double()
                for g in range(group):
                    x = torch.mm(q[row:row + n, h, g], k.t()) / math.sqrt(dim)
                    out[row:row + n, h, g] = torch.mm(torch.softmax(x.masked_fill(~see, -math.inf), 1), v)
            row += n
        return out.view(-1, nh * dim)
    rows = case["rows"]
    if kind == "select":
        count, first, recent = case["count"], s["first"], s["recent"]
        out = torch.full((rows * case["seqs"], kv, count), -1, dtype=I32, device=DEV)
        for i in range(case["seqs"]):
            edges = s["bounds"][s["tables"][i].long()].double()                                      # [pages, kv, 2, dim]
            for h in range(kv):
                q = s["q"][i * rows:(i + 1) * rows].view(rows, kv, group, dim)[:, h].double()
                # a key within the bounds gives a head at most q.k with every channel at the end that suits it
                most = sum(torch.mm(q[:, g] * (q[:, g] > 0), edges[:, h, 1].t()) + torch.mm(q[:, g] * (q[:, g] < 0), edges[:, h, 0].t())
                           for g in range(group))
                have = (s["ctx"][i * rows:(i + 1) * rows].long() + PAGE - 1) // PAGE
                page = torch.arange(most.shape[1], device=DEV)[None]
                rank = most.masked_fill((page < first) | (page >= have[:, None] - recent), math.inf).masked_fill(page >= have[:, None], -math.inf)
                best = torch.argsort(rank, dim=1, descending=True, stable=True)[:, :count]
                best = best.masked_fill(best >= have[:, None], 1 << 30).sort(1).values
                out[i * rows:(i + 1) * rows, h, :best.shape[1]] = best.masked_fill(best == 1 << 30, -1).to(I32)
        return out
    q = s["q"].double().view(-1, kv, group, dim)
    out = torch.zeros_like(q)
    spot = torch.arange(PAGE, device=DEV)
    for lo in range(0, q.shape[0], 64):
        part = slice(lo, min(lo + 64, q.shape[0]))
        for h in range(kv):
            sel = s["pages"][part, h].long()
            at = torch.gather(s["tables"].long()[s["seq"][part].long()], 1, sel.clamp(min=0))
            k, v = s["k_cache"][at, h].flatten(1, 2).double(), s["v_cache"][at, h].flatten(1, 2).double()
            hidden = ((sel[..., None] < 0) | (sel[..., None] * PAGE + spot >= s["ctx"][part, None, None])).flatten(1)
            x = torch.bmm(k, q[part, h].transpose(1, 2).contiguous()) / math.sqrt(dim)               # [rows, keys, group]
            w = torch.softmax(x.masked_fill(hidden[..., None], -math.inf), 1)
            out[part, h] = torch.bmm(w.transpose(1, 2).contiguous(), v)
    return out.view(-1, nh * dim)
