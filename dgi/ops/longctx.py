"""Ops for long caches (``dgi/_C_longctx.so``, sources in ``dgi/csrc/longctx``): rows that read the pages of their context that matter
to them, and drafted trees over long contexts.

* ``rope_cache_bounds``  the append: rotation, paged write, and the bounds (least and largest key of every channel) of the pages written
* ``page_bounds``        bounds of pages that came by another way (another worker, the host tier, keys moved between pages)
* ``select_pages``       per (row, kv head) the pages whose bounds promise the largest scores
* ``paged_selected``     attention over the selected pages
* ``paged_tree``         attention of drafted trees, split along the context, a group's heads sharing the keys

A decode step runs ``rope_cache_bounds`` -> ``select_pages`` -> ``paged_selected``; portions of prompts do the same with ``row_seq``
(the sequence of every row).  Same contract as the rest of ``dgi.ops``: the HIP kernel runs whenever the tensors are on the GPU (and raises
if the library is missing), the ``*_ref`` function — plain PyTorch — on CPU tensors.  On the GPU activations, caches and bounds are bf16 and
start on 16 bytes, heads have 64, 128 or 256 dims and at most 16 of them share a kv head; what does not fit is refused with ``ValueError``.
Nothing synchronises, scratch memory comes from torch's allocator, and every call may be captured into a graph.  Ids of pages outside
the cache, and selected pages behind a row's context, count as not there.
"""
from __future__ import annotations

import math
import os
from typing import Optional

import torch

import dgi.ops as ops

_LIB = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "_C_longctx.so")
_loaded = False


def load_native(required: bool = False) -> bool:
    """Load ``dgi/_C_longctx.so`` once (built by ``python -m dgi.build longctx``)."""
    global _loaded
    if _loaded:
        return True
    err = f"{_LIB} not built (run `python -m dgi.build longctx`)"
    if os.path.exists(_LIB):
        try:
            torch.ops.load_library(_LIB)
            _loaded = True
            return True
        except Exception as e:  # pragma: no cover - depends on the box
            err = repr(e)
    if required:
        raise RuntimeError(f"dgi long-cache kernels unavailable: {err}")
    return False


def _native(t: torch.Tensor) -> bool:
    return t.is_cuda and (_loaded or load_native(required=True))


def _call(name: str, *args):
    r = getattr(torch.ops.dgi, name)(*args)
    if ops._DEBUG_SYNC:
        from dgi.utils.debug import after_op
        after_op(name, *args)
    return r


def _need(ok: bool, op: str, what: str) -> None:
    if not ok:
        raise ValueError(f"{op}: {what}")


def _check_heads(op, nh, nkv):
    _need(nkv > 0 and nh > 0 and nh % nkv == 0 and nh // nkv <= 16, op, "heads must be 1 to 16 for each kv head")


def _check_rows(op, t, cols, name):
    _need(t.dim() == 2 and t.shape[1] >= cols, op, f"{name} must be rows of at least {cols} values")
    _need(not (t.requires_grad and torch.is_grad_enabled()), op, f"no gradient goes through {name}")


def _check_ints(op, t, dtype, name, n=None):
    _need(t.dtype == dtype and t.is_contiguous(), op, f"{name} must be contiguous {dtype}")
    _need(n is None or t.numel() == n, op, f"{name} must have {n} numbers")


def _check_row_seq(op, row_seq, tables, T):
    if row_seq is None:
        _need(tables.shape[0] >= T, op, "block_tables must have a row for each row of q (or row_seq says which)")
    else:
        _check_ints(op, row_seq, torch.int32, "row_seq", T)


def _check_attention(op, q, k_cache, v_cache, block_tables, nh, nkv, out):
    _check_heads(op, nh, nkv)
    _need(k_cache.dim() == 4 and k_cache.shape == v_cache.shape and k_cache.shape[1] == nkv and k_cache.is_contiguous()
          and v_cache.is_contiguous(), op, "k_cache and v_cache must be contiguous [blocks, kv heads, block size, dims]")
    _need(k_cache.shape[0] > 0 and k_cache.shape[2] > 0 and k_cache.shape[2] & (k_cache.shape[2] - 1) == 0, op, "pages of a power of two")
    _check_rows(op, q, nh * k_cache.shape[3], "q")
    _check_ints(op, block_tables, torch.int32, "block_tables")
    _need(block_tables.dim() == 2, op, "block_tables must be [sequences, pages]")
    _need(out is None or (out.dim() == 2 and out.shape[0] == q.shape[0] and out.shape[1] >= nh * k_cache.shape[3]), op,
          "out must have the rows of q")


# ----------------------------------------------------------------------------
# Page bounds
# ----------------------------------------------------------------------------

def empty_bounds(k_cache: torch.Tensor) -> torch.Tensor:
    """Bounds [blocks, kv heads, 2, dims] of a cache whose pages hold nothing yet: (inf, -inf)."""
    nb, nkv, _, hd = k_cache.shape
    b = torch.empty(nb, nkv, 2, hd, dtype=k_cache.dtype, device=k_cache.device)
    b[:, :, 0] = math.inf
    b[:, :, 1] = -math.inf
    return b


def rope_cache_bounds_ref(qkv, positions, cos_sin, nh, nkv, hd, slot_mapping, k_cache, v_cache, bounds, mode: int = 0) -> torch.Tensor:
    T, page = qkv.shape[0], k_cache.shape[2]
    rows = qkv[:, : (nh + 2 * nkv) * hd].clone()
    slots = slot_mapping.long()
    slots = torch.where(slots < k_cache.shape[0] * page, slots, -1)
    ops.rope_cache_ref(rows, positions.clamp(0, cos_sin.shape[0] - 1), cos_sin, nh, nkv, hd, slots, k_cache, v_cache, mode)
    for t in range(T):
        if slots[t] < 0:
            continue
        at, off = int(slots[t]) // page, int(slots[t]) % page
        k = k_cache[at, :, off]
        bounds[at, :, 0] = k if off == 0 else torch.minimum(bounds[at, :, 0], k)
        bounds[at, :, 1] = k if off == 0 else torch.maximum(bounds[at, :, 1], k)
    return rows[:, : nh * hd].contiguous()


def rope_cache_bounds(qkv, positions, cos_sin, nh: int, nkv: int, hd: int, slot_mapping, k_cache, v_cache, bounds, mode: int = 0,
                      out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``rope_cache`` that returns the rotated queries [T, nh * hd] (the rows of ``qkv`` stay as they are) and keeps ``bounds``
    [blocks, nkv, 2, hd]: the least and the largest cached key of every channel of a page.

    A page's bounds start anew with its slot 0 and go on otherwise; they never shrink, so keys that are overwritten or given up (rejected
    drafts) leave them wider than need be, never too narrow.  Rows of one page lie side by side, by rising slots, each slot once, as the
    steps of ``ModelRunner`` lay them out; slots may be left out.  Rows with a slot outside the cache (-1) are rotated and not cached, wherever
    they lie."""
    if _native(qkv):
        if out is None:
            return _call("rope_cache_bounds_new", qkv, positions, cos_sin, nh, nkv, hd, slot_mapping, k_cache, v_cache, bounds, mode)
        _call("rope_cache_bounds", out, qkv, positions, cos_sin, nh, nkv, hd, slot_mapping, k_cache, v_cache, bounds, mode)
        return out
    op = "rope_cache_bounds"
    _check_heads(op, nh, nkv)
    _check_rows(op, qkv, (nh + 2 * nkv) * hd, "qkv")
    _need(k_cache.dim() == 4 and k_cache.shape == v_cache.shape and k_cache.shape[1] == nkv and k_cache.shape[3] == hd, op,
          "k_cache and v_cache must be [blocks, kv heads, block size, dims]")
    _need(bounds.shape == (k_cache.shape[0], nkv, 2, hd), op, "bounds must be [blocks, kv heads, 2, dims]")
    _check_ints(op, positions, torch.int32, "positions", qkv.shape[0])
    _check_ints(op, slot_mapping, torch.int32, "slot_mapping", qkv.shape[0])
    _need(mode in (0, 1), op, "mode is 0 (halves) or 1 (interleaved pairs)")
    _need(cos_sin.dim() == 2 and cos_sin.shape[0] > 0, op, "cos_sin must be [positions, rotated dims]")
    rd = cos_sin.shape[1]
    _need(0 < rd <= hd and rd % (8 if mode else 16) == 0, op, "rotated dims must be a multiple of 16 (mode 1: 8) and at most the head's")
    _need(out is None or (out.is_contiguous() and out.shape == (qkv.shape[0], nh * hd)), op, "out must be contiguous [rows, heads * dims]")
    r = rope_cache_bounds_ref(qkv, positions, cos_sin, nh, nkv, hd, slot_mapping, k_cache, v_cache, bounds, mode)
    return r if out is None else out.copy_(r)


def page_bounds_ref(k_cache, bounds, pages, lens) -> None:
    page = k_cache.shape[2]
    for p, n in zip(pages.tolist(), lens.tolist()):
        if not 0 <= p < k_cache.shape[0]:
            continue
        n = min(max(n, 0), page)
        bounds[p, :, 0] = k_cache[p, :, :n].amin(1) if n else math.inf
        bounds[p, :, 1] = k_cache[p, :, :n].amax(1) if n else -math.inf


def page_bounds(k_cache, bounds, pages, lens) -> None:
    """Bounds of ``pages`` [n] int32, each given once, from the first ``lens`` [n] int32 keys that they hold; (inf, -inf) for none."""
    if _native(k_cache):
        _call("page_bounds", k_cache, bounds, pages, lens)
        return
    op = "page_bounds"
    _need(k_cache.dim() == 4, op, "k_cache must be contiguous [blocks, kv heads, block size, dims]")
    _need(bounds.shape == (*k_cache.shape[:2], 2, k_cache.shape[3]), op, "bounds must be [blocks, kv heads, 2, dims]")
    _check_ints(op, pages, torch.int32, "pages")
    _check_ints(op, lens, torch.int32, "lens", pages.numel())
    page_bounds_ref(k_cache, bounds, pages, lens)


# ----------------------------------------------------------------------------
# Selection
# ----------------------------------------------------------------------------

def select_pages_ref(q, bounds, block_tables, context_lens, nh, nkv, page, count, first, recent, row_seq=None) -> torch.Tensor:
    T, hd = q.shape[0], bounds.shape[-1]
    out = torch.full((T, nkv, count), -1, dtype=torch.int32)
    for t in range(T):
        n = min((int(context_lens[t]) + page - 1) // page, block_tables.shape[1])
        seq = t if row_seq is None else int(row_seq[t])
        if n <= count:
            out[t, :, : max(n, 0)] = torch.arange(max(n, 0), dtype=torch.int32)
            continue
        ids = block_tables[seq, :n].long() if 0 <= seq < block_tables.shape[0] else torch.full((n,), -1)
        there = (ids >= 0) & (ids < bounds.shape[0])
        b = bounds[ids.clamp(0, bounds.shape[0] - 1)].double()                    # [n, nkv, 2, hd]
        x = q[t, : nh * hd].double().view(nkv, -1, hd)
        score = (x.clamp(min=0).sum(1) * b[:, :, 1]).sum(-1) + (x.clamp(max=0).sum(1) * b[:, :, 0]).sum(-1)
        score = torch.nan_to_num(score, nan=-math.inf, posinf=math.inf, neginf=-math.inf).t()      # [nkv, n]
        best = torch.sort(score[:, first:n - recent].masked_fill(~there[first:n - recent], -math.inf), dim=1, descending=True, stable=True)
        keep = (best.indices[:, : count - first - recent] + first).sort(1).values
        out[t, :, :first] = torch.arange(first, dtype=torch.int32)
        out[t, :, first:count - recent] = keep.to(torch.int32)
        out[t, :, count - recent:] = torch.arange(n - recent, n, dtype=torch.int32)
    return out


def select_pages(q, bounds, block_tables, context_lens, nh: int, nkv: int, page: int, count: int, first: int = 1, recent: int = 1,
                 row_seq: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The pages that each row and kv head is to read: ordinals within the row's sequence, ascending, int32 [T, nkv, count], -1 behind
    them where the context has fewer.

    ``q`` [T, >= nh * hd] rotated; ``block_tables`` [sequences, pages], row t's is ``row_seq[t]`` (None: t); ``context_lens`` [T] the keys
    that row t sees, ``page`` tokens a page.  The first ``first`` and last ``recent`` pages are kept (the page that holds the row itself
    is among the latter, so keys behind the row decide nothing), then those with the largest
    P . largest + N . least, P and N the sums over the group's heads of max(q, 0) and min(q, 0), which no key of the page can exceed.
    Pages are compared by these sums in 64 bits; ties go to the lowest page, a sum that is no number (zero times infinite) counts as
    -inf."""
    if _native(q):
        if out is None:
            return _call("select_pages_new", q, bounds, block_tables, context_lens, nh, nkv, page, count, first, recent, row_seq)
        _need(out.dim() == 3 and out.shape[2] == count, "select_pages", "out must be [rows, kv heads, count]")
        _call("select_pages", out, q, bounds, block_tables, context_lens, nh, nkv, page, first, recent, row_seq)
        return out
    op = "select_pages"
    _check_heads(op, nh, nkv)
    _need(bounds.dim() == 4 and bounds.shape[1] == nkv and bounds.shape[2] == 2, op, "bounds must be [blocks, kv heads, 2, dims]")
    _check_rows(op, q, nh * bounds.shape[3], "q")
    _check_ints(op, block_tables, torch.int32, "block_tables")
    _check_ints(op, context_lens, torch.int32, "context_lens", q.shape[0])
    _need(page > 0, op, "a page has tokens")
    _need(first >= 0 and recent >= 1 and first + recent <= count, op, "first >= 0, recent >= 1 and both within count")
    _check_row_seq(op, row_seq, block_tables, q.shape[0])
    _need(out is None or (out.dtype == torch.int32 and out.shape == (q.shape[0], nkv, count)), op, "out must be [rows, kv heads, count]")
    r = select_pages_ref(q, bounds, block_tables, context_lens, nh, nkv, page, count, first, recent, row_seq)
    return r if out is None else out.copy_(r)


# ----------------------------------------------------------------------------
# Attention
# ----------------------------------------------------------------------------

def _attend_ref(q, k, v, see, scale):
    """q [n, d] over k, v [m, d]; ``see`` [n, m]; rows that see nothing are zero."""
    s = (q.float() @ k.float().t() * scale).masked_fill(~see, -math.inf)
    p = torch.softmax(s, -1).masked_fill(~see, 0.0)
    used = see.any(0)
    return torch.where(see.any(1, keepdim=True), p[:, used] @ v.float()[used], 0.0)


def paged_selected_ref(q, k_cache, v_cache, block_tables, context_lens, pages, nh, nkv, scale, row_seq=None) -> torch.Tensor:
    T, (nb, _, page, hd), G = q.shape[0], k_cache.shape, nh // nkv
    out = torch.zeros(T, nh * hd, dtype=q.dtype, device=q.device)
    for t in range(T):
        ctx, seq = int(context_lens[t]), t if row_seq is None else int(row_seq[t])
        if ctx <= 0 or not 0 <= seq < block_tables.shape[0]:
            continue
        for h in range(nkv):
            keys = [(int(block_tables[seq, p]), min(page, ctx - p * page)) for p in pages[t, h].tolist()
                    if 0 <= p < block_tables.shape[1] and p * page < ctx]
            keys = [(i, n) for i, n in keys if 0 <= i < nb]
            if not keys:
                continue
            k = torch.cat([k_cache[i, h, :n] for i, n in keys])
            v = torch.cat([v_cache[i, h, :n] for i, n in keys])
            x = q[t, h * G * hd:(h + 1) * G * hd].view(G, hd)
            o = _attend_ref(x, k, v, torch.ones(G, k.shape[0], dtype=torch.bool), scale)
            out[t, h * G * hd:(h + 1) * G * hd] = o.reshape(-1).to(q.dtype)
    return out


def paged_selected(q, k_cache, v_cache, block_tables, context_lens, pages, nh: int, nkv: int, scale: float,
                   row_seq: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of every row over its selected pages [T, nh * hd].

    ``pages`` [T, nkv, count] int32: ordinals of pages within the row's sequence (``select_pages``), in any order; -1 and pages behind
    the row's ``context_lens`` [T] are empty, a page named twice counts twice.  ``block_tables`` and ``row_seq`` as there.  Rows that
    see nothing are zero."""
    if _native(q):
        if out is None:
            return _call("paged_selected_new", q, k_cache, v_cache, block_tables, context_lens, pages, nh, nkv, scale, row_seq)
        _call("paged_selected", out, q, k_cache, v_cache, block_tables, context_lens, pages, nh, nkv, scale, row_seq)
        return out
    op = "paged_selected"
    _check_attention(op, q, k_cache, v_cache, block_tables, nh, nkv, out)
    _check_ints(op, context_lens, torch.int32, "context_lens", q.shape[0])
    _check_ints(op, pages, torch.int32, "pages")
    _need(pages.dim() == 3 and pages.shape[:2] == (q.shape[0], nkv) and pages.shape[2] > 0, op, "pages must be [rows, kv heads, count]")
    _check_row_seq(op, row_seq, block_tables, q.shape[0])
    r = paged_selected_ref(q, k_cache, v_cache, block_tables, context_lens, pages, nh, nkv, scale, row_seq)
    if out is None:
        return r
    out[:, : r.shape[1]] = r
    return out


def paged_tree_ref(q, k_cache, v_cache, block_tables, cu_seqlens_q, context_lens, tree_mask, nh, nkv, scale, max_nodes: int = 64,
                   out=None) -> torch.Tensor:
    (nb, _, page, hd), G = k_cache.shape, nh // nkv
    if out is None:
        out = torch.zeros(q.shape[0], nh * hd, dtype=q.dtype, device=q.device)
    cu = cu_seqlens_q.tolist()
    for s in range(len(cu) - 1):
        r0, n = cu[s], min(min(cu[s + 1], q.shape[0]) - cu[s], max_nodes)
        if r0 < 0 or n <= 0:
            continue
        ctx = min(max(int(context_lens[s]), 0), block_tables.shape[1] * page)
        ids = block_tables[s, : (ctx + page - 1) // page].long()
        there = ((ids >= 0) & (ids < nb)).repeat_interleave(page)[:ctx]
        ids = ids.clamp(0, nb - 1)
        node = torch.arange(ctx) - (ctx - n)
        bits = tree_mask[s, :n, None] >> node.clamp(0, 63)
        see = there & ((node < 0) | ((bits & 1) == 1))
        for h in range(nkv):
            k, v = k_cache[ids, h].reshape(-1, hd)[:ctx], v_cache[ids, h].reshape(-1, hd)[:ctx]
            for g in range(G):
                cols = slice((h * G + g) * hd, (h * G + g + 1) * hd)
                for a in range(n):      # a row alone: what others see does not reach it
                    m = see[a]
                    out[r0 + a, cols] = _attend_ref(q[r0 + a, cols][None], k[m], v[m], torch.ones(1, int(m.sum()), dtype=torch.bool),
                                                    scale)[0].to(out.dtype)
    return out


def paged_tree(q, k_cache, v_cache, block_tables, cu_seqlens_q, context_lens, tree_mask, nh: int, nkv: int, scale: float,
               max_nodes: int = 64, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of drafted trees over their paged caches [T, nh * hd].

    Rows ``cu_seqlens_q[s]`` .. ``cu_seqlens_q[s + 1]`` are the nodes of sequence s, at most ``max_nodes`` (<= 64) of them; their keys are
    the last of the ``context_lens[s]`` cached ones, in the same order.  A node sees all keys before the tree's and those nodes whose
    bits ``tree_mask[s, node]`` (int64 [sequences, >= max_nodes], as ``tree_mask`` makes them) has set.  Rows that see nothing are zero; rows of no
    sequence are left as they are in ``out``, and are not set where it is None."""
    if _native(q):
        if out is None:
            return _call("paged_tree_new", q, k_cache, v_cache, block_tables, cu_seqlens_q, context_lens, tree_mask, nh, nkv, scale, max_nodes)
        _call("paged_tree", out, q, k_cache, v_cache, block_tables, cu_seqlens_q, context_lens, tree_mask, nh, nkv, scale, max_nodes)
        return out
    op = "paged_tree"
    _check_attention(op, q, k_cache, v_cache, block_tables, nh, nkv, out)
    S = context_lens.numel()
    _check_ints(op, context_lens, torch.int32, "context_lens")
    _check_ints(op, cu_seqlens_q, torch.int32, "cu_seqlens_q", S + 1)
    _need(block_tables.shape[0] >= S, op, "block_tables must have a row for each sequence")
    _check_ints(op, tree_mask, torch.int64, "tree_mask")
    _need(1 <= max_nodes <= 64, op, "trees of 1 to 64 nodes")
    _need(tree_mask.dim() == 2 and tree_mask.shape[0] >= S and tree_mask.shape[1] >= max_nodes, op, "tree_mask must be [sequences, nodes]")
    return paged_tree_ref(q, k_cache, v_cache, block_tables, cu_seqlens_q, context_lens, tree_mask, nh, nkv, scale, max_nodes, out)
