"""Operators for long caches (``dgi.ops.longctx``) against a plain implementation in 64 bits, on the CPU's reference path and (``gpu``) on
the HIP kernels: layouts, lengths from none to long ones, pages that end inside a tile, rows that see nothing, values that are no numbers
in places that nobody sees, refusals, graphs, streams.

Tolerances count roundings.  A bf16 result is off by at most 2^-8 of itself; attention weights rounded to bf16 put at most
2^-8 of A = sum p |v| / sum p on top; a score is a sum of hd products in fp32, off by at most d = (hd + 4) 2^-24 scale max |q| . |k|, which puts
2 d on each weight and its sum; exp2 and the sums over n keys take (n + 16) 2^-24 of A.
"""
import ctypes
import math
import os
import random
import subprocess

import pytest
import torch

import dgi.build
from dgi import ops
from dgi.ops import longctx

gpu = pytest.mark.gpu
BF16, F64, I32 = torch.bfloat16, torch.float64, torch.int32
U8, U24 = 2.0 ** -8, 2.0 ** -24


@pytest.fixture(params=["cpu", pytest.param("cuda", marks=gpu)])
def dev(request):
    if request.param == "cuda":
        longctx.load_native(required=True)
    return request.param


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _randn(g, *shape, scale=1.0, dev="cpu", dtype=BF16):
    return (torch.randn(*shape, generator=g) * scale).to(dtype).to(dev)


def _tables(g, need, cols, pool, dev):
    """Shuffled page ids for sequences of ``need`` pages each."""
    ids = torch.randperm(pool, generator=g)[: sum(need)].to(I32)
    t = torch.full((len(need), cols), -1, dtype=I32)
    at = 0
    for i, n in enumerate(need):
        t[i, :n] = ids[at:at + n]
        at += n
    return t.to(dev)


def _close(got, want, tol, what=""):
    got, want, tol = got.double().cpu(), want.double().cpu(), tol.double().cpu()
    bad = ~((got - want).abs() <= tol) & ~((got == want) | (got.isnan() & want.isnan()))
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(((got - want).abs() / tol)[bad].max())} of its tolerance"


def _attention(q, k, v, scale):
    """q [G, hd] over k, v [n, hd] in 64 bits, and the tolerance."""
    if k.shape[0] == 0:
        return torch.zeros_like(q, dtype=F64), torch.zeros_like(q, dtype=F64)
    q, k, v = q.double(), k.double(), v.double()
    p = torch.softmax(q @ k.t() * scale, -1)
    o, a = p @ v, p @ v.abs()
    d = (q.shape[1] + 4) * U24 * abs(scale) * float((q.abs() @ k.abs().t()).max())
    return o, U8 * o.abs() + (U8 + 4 * d + (k.shape[0] + 16) * U24) * a + 1e-30


# ---- the append -------------------------------------------------------------------------------------------------------------------------

def _rotate64(x, cs, mode):
    """x [T, heads, hd] rotated in 64 bits, and the size of what is added up."""
    x, cs = x.double(), cs.double()
    y, size = x.clone(), x.abs()
    half = cs.shape[1] // 2
    for i in range(half):
        a, b = (i, i + half) if mode == 0 else (2 * i, 2 * i + 1)
        c, s = cs[:, i, None], cs[:, half + i, None]
        y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
        size[..., a] = size[..., b] = x[..., a].abs() + x[..., b].abs()
    return y, size


def _append_case(dev, nh, nkv, hd, rd, mode, page, spans, extra=0, seed=0, pool=None):
    """Portions ``spans`` = (first position, rows) of sequences whose pages hold what came before."""
    g = _gen(seed)
    need = [(p + n + page - 1) // page for p, n in spans]
    pool = pool or sum(need) + 5
    tables = _tables(g, need, max(need), pool, "cpu")
    pos = torch.cat([torch.arange(p, p + n) for p, n in spans]).to(I32)
    slots = torch.cat([tables[i, torch.arange(p, p + n) // page] * page + torch.arange(p, p + n) % page for i, (p, n) in enumerate(spans)]).to(I32)
    k, v = _randn(g, pool, nkv, page, hd), _randn(g, pool, nkv, page, hd)
    bounds = torch.stack([k.amin(2), k.amax(2)], 2) * 0.25      # narrow, so that keys of this step widen them
    qkv = _randn(g, len(pos), (nh + 2 * nkv) * hd + extra)
    cs = ops.rope_cos_sin(rd, int(pos.max()) + 3, 10000.0)
    return [x.to(dev) for x in (qkv, pos, cs, slots, k, v, bounds)]


def _append_check(dev, nh, nkv, hd, mode, page, case):
    qkv, pos, cs, slots, k, v, bounds = case
    k0, v0, b0, qkv0 = k.clone(), v.clone(), bounds.clone(), qkv.clone()
    q = longctx.rope_cache_bounds(qkv, pos, cs, nh, nkv, hd, slots, k, v, bounds, mode)
    T = qkv.shape[0]
    assert torch.equal(qkv, qkv0)
    rows = qkv[:, : (nh + 2 * nkv) * hd].reshape(T, nh + 2 * nkv, hd).cpu()
    want, size = _rotate64(rows[:, : nh + nkv], cs.cpu()[pos.cpu().long()], mode)
    tol = (U8 + 4 * U24) * want.abs() + 4 * U24 * size      # two products, a sum, each rounded, then bf16
    _close(q.view(T, nh, hd), want[:, :nh], tol[:, :nh], "q")
    k, v, bounds, k0, v0, b0 = (x.cpu() for x in (k, v, bounds, k0, v0, b0))
    for t, s in enumerate(slots.tolist()):
        if s < 0:
            continue
        at, off = s // page, s % page
        _close(k[at, :, off], want[t, nh:], tol[t, nh:], "k")
        assert torch.equal(v[at, :, off], rows[t, nh + nkv:])
        k0[at, :, off], v0[at, :, off] = k[at, :, off], v[at, :, off]
        if off == 0:
            b0[at, :, 0], b0[at, :, 1] = k[at, :, 0], k[at, :, 0]
        else:
            b0[at, :, 0], b0[at, :, 1] = torch.minimum(b0[at, :, 0], k[at, :, off]), torch.maximum(b0[at, :, 1], k[at, :, off])
    assert torch.equal(k, k0) and torch.equal(v, v0)      # nothing else is written
    assert torch.equal(bounds, b0)                        # a minimum rounds nothing


@pytest.mark.parametrize("nh,nkv,hd,rd,mode", [(8, 2, 64, 64, 0), (4, 4, 128, 128, 0), (16, 1, 128, 64, 1), (14, 2, 64, 16, 0), (7, 1, 256, 128, 0),
                                               (6, 3, 64, 8, 1)])
@pytest.mark.parametrize("page", [16, 8, 12])
def test_append(dev, nh, nkv, hd, rd, mode, page):
    """Decode rows at a page's first, middle and last slot, portions within a page, across pages, and of whole ones."""
    spans = [(0, 1), (page - 1, 1), (page, 1), (5, 1), (0, page), (3, 2), (2, 3 * page + 1), (page, 2 * page)]
    _append_check(dev, nh, nkv, hd, mode, page, _append_case(dev, nh, nkv, hd, rd, mode, page, spans))


def test_append_strided_rows_and_rows_without_a_slot(dev):
    case = _append_case(dev, 8, 2, 64, 64, 0, 16, [(3, 20), (16, 1), (30, 4)], extra=72)
    case[3][[1, 20, 24]] = -1      # inside a portion, a decode row, the last row
    _append_check(dev, 8, 2, 64, 0, 16, case)
    case = _append_case(dev, 8, 2, 64, 64, 0, 16, [(3, 20)])
    case[0] = case[0].repeat_interleave(2, 0)[::2]      # every other row of a buffer
    _append_check(dev, 8, 2, 64, 0, 16, case)


PAGE_RUNS = r"""
#include "page_runs.h"
template <class F> unsigned long long ballot(F f) {
  unsigned long long b = 0;
  for (int lane = 0; lane < 64; ++lane) b |= (unsigned long long)(bool)f(lane) << lane;
  return b;
}
extern "C" void runs(const int* slots, int T, long long n_slots, int page, int* out) {
  auto b = [](auto f) { return ballot(f); };
  for (int t = 0; t < T; ++t) {
    const int page0 = slots[t] / page * page;
    out[t] = 0;
    if (!dgi::has_slot(slots[t], n_slots) || !dgi::begins_page(b, slots, n_slots, page, t, page0)) continue;
    const dgi::PageRows r = dgi::page_rows(b, slots, n_slots, page, T, t, page0);
    out[t] = r.plain ? r.rows : -r.rows;
  }
}
"""


def test_append_a_page_has_one_writer(tmp_path):
    """Which rows write a page's bounds, and what rows they look at, as the kernel finds it, on the CPU: rows without a slot and slots that are left
    out between a page's rows make no second writer."""
    src, lib = tmp_path / "runs.cpp", tmp_path / "runs.so"
    src.write_text(PAGE_RUNS)
    folder = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "dgi", "csrc", "longctx")
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I", folder, str(src), "-o", str(lib)], check=True)
    runs = ctypes.CDLL(str(lib)).runs
    rng = random.Random(5)
    for case in range(400):
        page, n_pages = rng.choice([1, 5, 16, 64, 256]), rng.choice([3, 40])
        drop, hole = rng.choice([0, 0.1, 0.6]), rng.choice([0, 0.1, 0.9])
        slots = [-1] * rng.choice([0, 0, 70, 200, 1300])
        for at in rng.sample(range(n_pages), rng.randint(1, min(n_pages, 12))):
            for off in range(rng.randrange(page), rng.randint(1, page)):
                if rng.random() >= drop:
                    slots += [rng.choice([-1, -(1 << 31), page * n_pages, (1 << 31) - 1])] * (rng.random() < hole) * rng.choice([1, 1, 1, 1, 1, 65, 600])
                    slots.append(at * page + off)
        slots += [-1] * rng.choice([0, 0, 63, 64, 65, 130, 1300])
        T = len(slots)
        out = (ctypes.c_int * T)()
        runs((ctypes.c_int * T)(*slots), T, ctypes.c_longlong(page * n_pages), page, out)
        have = [s // page if 0 <= s < page * n_pages else -1 for s in slots]
        first, last = {}, {}
        for t, p in enumerate(have):
            if p >= 0:
                first.setdefault(p, t)
                last[p] = t
        want = [0] * T
        for p, t in first.items():
            want[t] = (last[p] - t + 1) * (1 if slots[t:last[p] + 1] == list(range(slots[t], slots[t] + last[p] + 1 - t)) else -1)
        assert list(out) == want, (case, page, slots)
        for p, t in first.items():      # the rows that it looks at have no other page's
            assert {x for x in have[t:t + abs(want[t])] if x >= 0} == {p}


@pytest.mark.parametrize("page", [16, 32])
def test_append_rows_without_a_slot_within_a_page(dev, page):
    """Every second row of a portion is not cached, slots are left out, and as many rows as a wave has lie between two of a page."""
    case = _append_case(dev, 8, 2, 64, 64, 0, page, [(3, 3 * page), (page, 100), (1, 2)])
    case[3][1: 3 * page: 2] = -1
    case[3][3 * page + 1: 3 * page + 99] = -1
    _append_check(dev, 8, 2, 64, 0, page, case)
    rows = [0, 1, 4, 5, 9, page - 4, page, 2 * page + 3, 3 * page + 1]
    qkv, pos, cs, slots, k, v, bounds = _append_case(dev, 8, 2, 64, 64, 0, page, [(3, 4 * page)], seed=1)
    _append_check(dev, 8, 2, 64, 0, page, [qkv[rows], pos[rows], cs, slots[rows], k, v, bounds])


def test_append_no_rows_one_row_many_rows(dev):
    for spans in ([(0, 1)], [(100, 1)] * 37, [(7, 700)]):
        _append_check(dev, 8, 2, 64, 0, 16, _append_case(dev, 8, 2, 64, 64, 0, 16, spans))
    case = _append_case(dev, 8, 2, 64, 64, 0, 16, [(0, 1)])
    case[0], case[1], case[3] = case[0][:0], case[1][:0], case[3][:0]
    _append_check(dev, 8, 2, 64, 0, 16, case)


def test_append_keeps_what_is_no_number(dev):
    """A key that is no number makes its channel's bounds no number until the page starts anew; infinities bound."""
    case = _append_case(dev, 2, 1, 64, 64, 0, 16, [(3, 4)])
    qkv, pos, cs, slots, k, v, bounds = case
    qkv[1, 2 * 64 + 5] = math.nan
    qkv[2, 2 * 64 + 60] = math.inf
    longctx.rope_cache_bounds(qkv, pos, cs, 2, 1, 64, slots, k, v, bounds)
    b = bounds[int(slots[0]) // 16, 0].float()
    assert b[:, [5, 37]].isnan().all() and not b[:, [4, 36]].isnan().any()
    assert torch.isinf(b[:, [60, 28]]).any(0).all()


@pytest.mark.parametrize("nkv,hd,page", [(1, 64, 16), (8, 128, 16), (3, 256, 32), (2, 128, 5), (2, 64, 128)])
def test_page_bounds(dev, nkv, hd, page):
    g = _gen(1)
    nb = 41
    k = _randn(g, nb, nkv, page, hd)
    k[7, 0, 2, 3] = math.nan
    k[9, nkv - 1, 0, 1] = -math.inf
    pages = torch.randperm(nb, generator=g)[:30].to(I32)
    pages[:2] = torch.tensor([7, 9], dtype=I32)
    pages = torch.tensor(list(dict.fromkeys(pages.tolist())) + [-1, nb, nb + 100], dtype=I32)
    lens = torch.randint(0, page + 1, (len(pages),), generator=g).to(I32)
    lens[:6] = torch.tensor([page, page, 0, 1, page + 3, -1], dtype=I32)      # clamped to the page
    bounds = longctx.empty_bounds(k.to(dev))
    old = bounds.cpu().clone()
    longctx.page_bounds(k.to(dev), bounds, pages.to(dev), lens.to(dev))
    for p, n in zip(pages.tolist(), lens.tolist()):
        if 0 <= p < nb and n > 0:
            old[p, :, 0], old[p, :, 1] = k[p, :, : min(n, page)].amin(1), k[p, :, : min(n, page)].amax(1)
    assert torch.equal(bounds.cpu().isnan(), old.isnan())
    assert torch.equal(bounds.cpu().nan_to_num(7.0), old.nan_to_num(7.0))
    longctx.page_bounds(k.to(dev), bounds, pages[:0].to(dev), lens[:0].to(dev))


# ---- the selection ----------------------------------------------------------------------------------------------------------------------

def _selection64(q, bounds, tables, ctx, nh, nkv, page, count, first, recent, seq):
    """By sorting, page by page, from the definition: what a key within the bounds can give each head at most."""
    out = torch.full((q.shape[0], nkv, count), -1, dtype=I32)
    hd = bounds.shape[-1]
    for t in range(q.shape[0]):
        n = min(-(-int(ctx[t]) // page), tables.shape[1])
        for h in range(nkv):
            x = q[t, : nh * hd].double().view(nkv, -1, hd)[h]
            if n <= count:
                keep = list(range(max(n, 0)))
            else:
                b = bounds[tables[int(seq[t]), :n].long(), h].double()
                most = sum(torch.where(x[i] > 0, x[i] * b[:, 1], x[i] * b[:, 0]).sum(-1) for i in range(x.shape[0]))
                most = torch.where(most.isnan(), -math.inf, most).tolist()
                forced = list(range(first)) + list(range(n - recent, n))
                rest = sorted(range(first, n - recent), key=lambda p: (-most[p], p))[: count - first - recent]
                keep = sorted(forced + rest)
            out[t, h, : len(keep)] = torch.tensor(keep, dtype=I32)
    return out


def _select_case(nh, nkv, hd, page, lens, rows, seed=0, whole=False, extra=0):
    """``rows`` rows at the end of each sequence of ``lens`` tokens; ``whole``: small whole numbers, so that many scores are alike."""
    g = _gen(seed)
    need = [-(-n // page) for n in lens]
    pool = sum(need) + 3
    tables = _tables(g, need, max(need) + 2, pool, "cpu")
    if whole:
        b = torch.randint(-1, 2, (pool, nkv, 2, hd), generator=g).to(BF16).sort(2).values
        q = torch.randint(-1, 2, (len(lens) * rows, nh * hd + extra), generator=g).to(BF16)
    else:
        b = _randn(g, pool, nkv, 2, hd).sort(2).values
        q = _randn(g, len(lens) * rows, nh * hd + extra)
    ctx = torch.cat([torch.arange(n - rows + 1, n + 1) for n in lens]).to(I32)
    seq = torch.arange(len(lens), dtype=I32).repeat_interleave(rows)
    return q, b, tables, ctx, seq


def _select_check(dev, nh, nkv, page, count, first, recent, q, b, tables, ctx, seq):
    got = longctx.select_pages(q.to(dev), b.to(dev), tables.to(dev), ctx.to(dev), nh, nkv, page, count, first, recent, row_seq=seq.to(dev))
    assert got.dtype == I32
    assert torch.equal(got.cpu(), _selection64(q, b, tables, ctx, nh, nkv, page, count, first, recent, seq))


@pytest.mark.parametrize("nh,nkv,hd", [(8, 2, 64), (7, 1, 128), (16, 1, 64), (4, 4, 256)])
@pytest.mark.parametrize("count,first,recent", [(8, 1, 2), (5, 0, 1), (3, 1, 2), (1, 0, 1), (64, 1, 1)])
def test_select(dev, nh, nkv, hd, count, first, recent):
    """Contexts of one token, of exactly ``count`` pages, of one page more, of many."""
    lens = [1, 16 * count, 16 * count + 1, 16 * count + 17, 700, 1601]
    _select_check(dev, nh, nkv, 16, count, first, recent, *_select_case(nh, nkv, hd, 16, lens, 1))


@pytest.mark.parametrize("rows,page,extra", [(37, 16, 0), (5, 64, 64), (64, 16, 8), (130, 32, 0)])
def test_select_rows_of_prompts(dev, rows, page, extra):
    """Rows that follow each other see one key more each; their sequence's table is given by ``row_seq``."""
    _select_check(dev, 8, 2, page, 6, 1, 2, *_select_case(8, 2, 64, page, [max(rows, 300), max(rows, 900), 1777], rows, extra=extra))


@pytest.mark.parametrize("lens", [[400, 1000, 2222], [40000]])
def test_select_alike_pages_go_to_the_lowest(dev, lens):
    _select_check(dev, 4, 2, 16, 12, 1, 1, *_select_case(4, 2, 64, 16, lens, 1, whole=True))
    q, b, tables, ctx, seq = _select_case(4, 2, 64, 16, lens, 1, whole=True)
    _select_check(dev, 4, 2, 16, 12, 1, 1, q * 0, b, tables, ctx, seq)      # all alike, zeros of both signs


def test_select_close_scores(dev):
    """Pages whose scores differ in the last bits of 64: one channel of the bounds is a little larger."""
    q, b, tables, ctx, seq = _select_case(4, 1, 128, 16, [3000], 1)
    b[:] = b[:1]
    b[:, 0, 1, 17] += (torch.randperm(b.shape[0], generator=_gen(3)) % 5).to(BF16) * 2.0 ** -6
    q[:, 17::128] = 2.0 ** -30
    _select_check(dev, 4, 1, 16, 40, 1, 1, q, b, tables, ctx, seq)


def test_select_values_that_are_no_numbers(dev):
    q, b, tables, ctx, seq = _select_case(4, 2, 64, 16, [900, 900, 900, 900], 1)
    b[tables[0, 7], 0, 1, 3] = math.nan
    b[tables[0, 9], 1] = torch.tensor([math.inf, -math.inf], dtype=BF16)[:, None]      # bounds of a page without keys
    b[tables[1, 11], :, 1, 5] = math.inf
    b[tables[1, 12], :, 0, 5] = -math.inf
    q[2, 70] = math.nan
    q[3, 70] = math.inf
    _select_check(dev, 4, 2, 16, 8, 1, 1, q, b, tables, ctx, seq)


def test_select_empty_rows_and_unknown_pages(dev):
    q, b, tables, ctx, seq = _select_case(4, 2, 64, 16, [900, 900, 500], 1)
    ctx[1] = 0
    got = longctx.select_pages(q.to(dev), b.to(dev), tables.to(dev), ctx.to(dev), 4, 2, 16, 8).cpu()
    assert (got[1] == -1).all()
    tables[0, [5, 6]] = torch.tensor([-1, 1 << 30], dtype=I32)      # never read, never preferred
    got = longctx.select_pages(q.to(dev), b.to(dev), tables.to(dev), ctx.to(dev), 4, 2, 16, 54, row_seq=seq.to(dev)).cpu()
    assert not torch.isin(got[0], torch.tensor([5, 6], dtype=I32)).any() and (got[0] >= 0).all()
    ctx[0] = 1 << 30      # more than the table has: its pages are all there are
    got = longctx.select_pages(q.to(dev), b.to(dev), tables.to(dev), ctx.to(dev), 4, 2, 16, 8).cpu()
    assert (got[0] < tables.shape[1]).all() and (got[0].diff() > 0).all()
    assert longctx.select_pages(q[:0].to(dev), b.to(dev), tables.to(dev), ctx[:0].to(dev), 4, 2, 16, 8).shape == (0, 2, 8)


@pytest.mark.parametrize("what", ["alike", "zeros", "close", "huge", "tiny", "no numbers", "a hundred alike", "two of a kind"])
@pytest.mark.parametrize("hd,pages", [(64, 300), (128, 1300)])
def test_select_prompts_that_need_every_bit(dev, what, hd, pages):
    """Rows of one sequence, whose scores leave fewer bits nothing to decide with: many alike, or out of the range of 32 bits."""
    q, b, tables, ctx, seq = _select_case(4, 2, hd, 4, [4 * pages], 33, whole=what == "alike")
    count = 24
    if what == "zeros":
        q[:, ::2] = 0.0
        q[3:9] = 0.0
        b[:, 0] = -b[:, 0].abs()
    elif what == "close":
        b[:] = b[:1]
        b[:, :, 1, 17] += (torch.randperm(b.shape[0], generator=_gen(3)) % 5).to(BF16)[:, None] * 2.0 ** -6
        q[:, 17::hd] = 2.0 ** -30
    elif what == "huge":
        q, b = q * 2.0 ** 100, b * 2.0 ** 100
    elif what == "tiny":
        q, b = q * 2.0 ** -100, b * 2.0 ** -100
    elif what == "no numbers":
        b[tables[0, 7], 0, 1, 3] = math.nan
        b[tables[0, 9], 1] = torch.tensor([math.inf, -math.inf], dtype=BF16)[:, None]
        b[tables[0, 11], 1, 1, 5] = math.inf
        q[2, 70], q[5, hd + 1], q[6, 0] = math.nan, math.inf, -math.inf
    elif what == "a hundred alike":      # the best ones, more than are kept
        b[tables[0, 40:140].long()] = b[tables[0, 40:41].long()] + 2
    elif what == "two of a kind":
        b[tables[0, 1:pages // 2].long()] = b[tables[0, pages // 2: 2 * (pages // 2) - 1].long()]
    if what != "no numbers":
        return _select_check(dev, 4, 2, 4, count, 1, 2, q, b, tables, ctx, seq)
    # a weight of zero times an infinite bound is no number, and what that makes of a page is said by the sum itself
    got = longctx.select_pages(q.to(dev), b.to(dev), tables.to(dev), ctx.to(dev), 4, 2, 4, count, 1, 2, row_seq=seq.to(dev)).cpu()
    for t in range(33):
        n = -(-int(ctx[t]) // 4)
        x, y = q[t].double().view(2, 2, 1, hd), b[tables[0, :n].long()].double()
        up, down = x.clamp(min=0).sum(1), x.clamp(max=0).sum(1)
        sums = (up * y[:, :, 1].transpose(0, 1) + down * y[:, :, 0].transpose(0, 1)).sum(-1)
        for h in range(2):
            most = [-math.inf if math.isnan(s) else s for s in sums[h].tolist()]
            best = sorted(range(1, n - 2), key=lambda p: (-most[p], p))[: count - 3]
            assert got[t, h].tolist() == [0] + sorted(best) + [n - 2, n - 1]


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("q_exp,b_exp", [(-122, 40), (-127, 60), (-112, 0), (60, -130), (100, -128)])
def test_select_prompts_of_the_least_numbers(dev, hd, q_exp, b_exp):
    """Weights whose lower bits, or bounds that are subnormal, against large ones."""
    q, b, tables, ctx, seq = _select_case(4, 2, hd, 4, [1200], 33)
    q, b = (q.double() * 2.0 ** q_exp).to(BF16), (b.double() * 2.0 ** b_exp).to(BF16)
    _select_check(dev, 4, 2, 4, 24, 1, 2, q, b, tables, ctx, seq)


@pytest.mark.parametrize("hd,pages", [(64, 200), (256, 1000), (128, 1090), (64, 5000), (128, 8300), (256, 9000)])
def test_select_rows_of_long_prompts(dev, hd, pages):
    _select_check(dev, 3, 1, 2, 50, 2, 3, *_select_case(3, 1, hd, 2, [2 * pages], 18))
    q, b, tables, ctx, seq = _select_case(3, 1, hd, 2, [2 * pages], 3, whole=True)
    q[2] = 0.0
    _select_check(dev, 3, 1, 2, 50, 2, 3, q, b, tables, ctx, seq)


@pytest.mark.parametrize("nh,nkv,hd", [(8, 2, 64), (18, 2, 128), (4, 4, 256)])
def test_select_prompts_beside_single_rows(dev, nh, nkv, hd):
    """Sixteen rows of one to sixteen sequences, rows without a context or a sequence, pages that are none."""
    lens = [500, 900, 31, 1, 640, 700, 410, 1200, 800, 333, 1000, 640, 555, 1500, 900]
    runs = [1] * 10 + [30, 3, 3, 3, 17]
    q, b, tables, ctx, seq = _select_case(nh, nkv, hd, 8, lens, 30)
    rows = torch.cat([torch.arange(30 * i + 30 - n, 30 * i + 30) for i, n in enumerate(runs)])
    q, ctx, seq = q[rows].contiguous(), ctx[rows].contiguous(), seq[rows].contiguous()
    ctx[[4, 20, 55]] = torch.tensor([0, -5, 0], dtype=I32)
    none, b = b.shape[0], torch.cat([b, torch.stack([torch.full_like(b[:1, :, 0], math.inf), torch.full_like(b[:1, :, 0], -math.inf)], 2)])
    tables[10, [3, 50]], tables[13, 7], tables[7, 9] = none, none, none
    given = torch.where(tables == none, torch.tensor([-1, 1 << 30], dtype=I32)[torch.arange(tables.shape[1]) % 2], tables)
    want = _selection64(q, b, tables, ctx, nh, nkv, 8, 20, 1, 2, seq)
    lost = torch.tensor([6, 30, 57])      # of no known sequence: all pages alike, so the lowest
    seq[lost] = torch.tensor([-1, 15, 1 << 30], dtype=I32)
    for t in lost.tolist():
        n = -(-int(ctx[t]) // 8)
        want[t] = torch.tensor(list(range(18)) + [n - 2, n - 1], dtype=I32) if n > 20 else torch.tensor(list(range(n)) + [-1] * (20 - n), dtype=I32)
    got = longctx.select_pages(q.to(dev), b.to(dev), given.to(dev), ctx.to(dev), nh, nkv, 8, 20, 1, 2, row_seq=seq.to(dev))
    assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("grouped", [False, True])
def test_select_wide_tables(dev, grouped):
    """Tables so wide that scores of all rows together would take 300 MB and more: rows go in several batches."""
    lens = [900 + 7 * i for i in range(104)] if not grouped else [700, 900]
    q, b, tables, ctx, seq = _select_case(8, 8, 64, 16, lens, 52 if grouped else 1)
    wide = torch.full((len(lens), 50000), -1, dtype=I32)
    wide[:, : tables.shape[1]] = tables
    _select_check(dev, 8, 8, 16, 10, 1, 1, q, b, wide, ctx, seq)
    if not grouped:
        got = longctx.select_pages(q.to(dev), b.to(dev), wide.to(dev), ctx.to(dev), 8, 8, 16, 10, 1, 1)
        assert torch.equal(got.cpu(), _selection64(q, b, tables, ctx, 8, 8, 16, 10, 1, 1, seq))


def test_select_whole_tables_of_rows(dev):
    """A table that has no more pages than are kept, and a row more than sequences."""
    q, b, tables, ctx, seq = _select_case(4, 2, 64, 16, [90, 160], 20)
    _select_check(dev, 4, 2, 16, tables.shape[1], 1, 1, q, b, tables, ctx, seq)
    _select_check(dev, 4, 2, 16, tables.shape[1] + 9, 1, 1, q, b, tables, ctx, seq)


# ---- attention over selected pages ------------------------------------------------------------------------------------------------------

def _selected_case(nh, nkv, hd, page, lens, count, rows=1, seed=0, extra=0):
    g = _gen(seed)
    need = [-(-max(n, 1) // page) for n in lens]
    pool = sum(need) + 3
    tables = _tables(g, need, max(need), pool, "cpu")
    k, v = _randn(g, pool, nkv, page, hd), _randn(g, pool, nkv, page, hd)
    q = _randn(g, len(lens) * rows, nh * hd + extra)
    ctx = torch.cat([torch.arange(n - rows + 1, n + 1) for n in lens]).to(I32)
    seq = torch.arange(len(lens), dtype=I32).repeat_interleave(rows)
    pages = torch.full((q.shape[0], nkv, count), -1, dtype=I32)
    for t in range(q.shape[0]):
        n = -(-int(ctx[t]) // page)
        for h in range(nkv):
            some = torch.randperm(n, generator=g)[:count].sort().values if n > 0 else torch.empty(0, dtype=torch.long)
            pages[t, h, : len(some)] = some.to(I32)
            if n > 0:
                pages[t, h, max(len(some) - 1, 0)] = n - 1      # the page that is not full
    return q, k, v, tables, ctx, pages, seq


def _selected_want(nh, nkv, scale, q, k, v, tables, ctx, pages, seq):
    T, page, hd, G = q.shape[0], k.shape[2], k.shape[3], nh // nkv
    o, tol = torch.zeros(T, nkv, G, hd, dtype=F64), torch.zeros(T, nkv, G, hd, dtype=F64)
    for t in range(T):
        for h in range(nkv):
            kk = [k[tables[seq[t], p], h, : int(ctx[t]) - p * page] for p in pages[t, h].tolist() if 0 <= p * page < int(ctx[t])]
            vv = [v[tables[seq[t], p], h, : int(ctx[t]) - p * page] for p in pages[t, h].tolist() if 0 <= p * page < int(ctx[t])]
            x = q[t, : nh * hd].view(nkv, G, hd)[h]
            o[t, h], tol[t, h] = _attention(x, torch.cat(kk) if kk else k[0, 0, :0], torch.cat(vv) if vv else v[0, 0, :0], scale)
    return o.view(T, -1), tol.view(T, -1)


def _selected_check(dev, nh, nkv, case, scale=None, **kw):
    scale = scale if scale is not None else case[1].shape[-1] ** -0.5
    q, k, v, tables, ctx, pages, seq = (x.to(dev) for x in case)
    got = longctx.paged_selected(q, k, v, tables, ctx, pages, nh, nkv, scale, row_seq=seq, **kw)
    want, tol = _selected_want(nh, nkv, scale, *case)
    _close(got[:, : want.shape[1]], want, tol)
    return got


@pytest.mark.parametrize("nh,nkv,hd", [(8, 2, 64), (7, 1, 128), (16, 1, 128), (4, 4, 256), (3, 3, 64)])
@pytest.mark.parametrize("page", [16, 8, 64])
def test_selected(dev, nh, nkv, hd, page):
    """Contexts of one token up to many pages, lists shorter than ``count``, last pages of every fill."""
    _selected_check(dev, nh, nkv, _selected_case(nh, nkv, hd, page, [1, 2, 15, 16, 17, 31, 33, 100, 777], 9))


@pytest.mark.parametrize("rows,lens", [(21, [21, 300]), (70, [1000])])
def test_selected_rows_of_prompts(dev, rows, lens):
    _selected_check(dev, 8, 2, _selected_case(8, 2, 64, 16, lens, 6, rows=rows, extra=24))


@pytest.mark.parametrize("count,lens", [(1, [5]), (2, [4000]), (200, [9000]), (700, [13000, 3]), (64, [2000] * 9)])
def test_selected_few_rows_long_lists(dev, count, lens):
    """Lists that are cut between workgroups, longer than a workgroup's list, or nearly empty."""
    _selected_check(dev, 4, 1, _selected_case(4, 1, 64, 16, lens, count))


def test_selected_lists_in_any_order(dev):
    """Empty entries anywhere, pages behind the context, pages twice, nothing at all."""
    case = _selected_case(4, 2, 64, 16, [500, 500, 500, 0, 40], 12)
    pages = case[5]
    pages[0, 0] = torch.tensor([-1, 31, -1, 4, 4, 0, -1, 30, 99, 31, -1, 1 << 30], dtype=I32)
    pages[0, 1] = -1
    pages[1, 0] = torch.tensor([31] * 12, dtype=I32)
    pages[2] = pages[2].flip(-1)
    pages[3] = torch.arange(12, dtype=I32)      # a row without a context
    got = _selected_check(dev, 4, 2, case)
    assert (got[0, 128:] == 0).all() and (got[3] == 0).all()
    case[3][0, 4] = -7                          # a page that is not in the cache counts as not there
    case[3][1, 31] = 1 << 30
    q, k, v, tables, ctx, pages, seq = (x.to(dev) for x in case)
    got = longctx.paged_selected(q, k, v, tables, ctx, pages, 4, 2, 0.125)
    pages = case[5].clone()
    pages[0][pages[0] == 4] = -1
    pages[1][pages[1] == 31] = -1
    case[3][0, 4], case[3][1, 31] = 0, 0
    want, tol = _selected_want(4, 2, 0.125, *case[:5], pages, case[6])
    _close(got, want, tol)


def test_selected_places_that_nobody_sees(dev):
    """NaN and infinities behind the context, in other pages, and in no page of the list reach nothing; large scores do not overflow."""
    case = _selected_case(4, 2, 64, 16, [37, 500, 16, 161], 5)
    q, k, v, tables, ctx, pages, seq = case
    used = torch.zeros(k.shape[0], 2, 16, dtype=torch.bool)
    for t in range(4):
        for h in range(2):
            for p in pages[t, h].tolist():
                if 0 <= p * 16 < int(ctx[t]):
                    used[tables[t, p], h, : int(ctx[t]) - 16 * p] = True
    k[~used] = math.nan
    v[~used] = math.inf
    v[~used & (torch.arange(16) % 2 == 0)] = math.nan
    _selected_check(dev, 4, 2, case)
    q.mul_(1e3)
    _selected_check(dev, 4, 2, case)
    _selected_check(dev, 4, 2, case, scale=-0.125)
    _selected_check(dev, 4, 2, case, scale=0.0)


def test_selected_out_and_strides(dev):
    case = _selected_case(8, 2, 64, 16, [300, 50, 1], 8, extra=40)
    out = torch.full((3, 8 * 64 + 16), 5.0, dtype=BF16, device=dev)
    got = _selected_check(dev, 8, 2, case, out=out)
    assert got.data_ptr() == out.data_ptr() and (out[:, 512:] == 5.0).all()
    empty = [x[:0] if i in (0, 4, 5, 6) else x for i, x in enumerate(case)]
    q, k, v, tables, ctx, pages, seq = (x.to(dev) for x in empty)
    assert longctx.paged_selected(q, k, v, tables, ctx, pages, 8, 2, 0.125).shape == (0, 512)


@pytest.mark.parametrize("nh,nkv,hd,page", [(1, 1, 64, 16), (5, 1, 128, 4), (14, 2, 128, 32), (16, 1, 64, 16), (6, 2, 256, 16), (2, 2, 128, 128),
                                            (3, 1, 64, 1)])
def test_selected_prompts(dev, nh, nkv, hd, page):
    """Neighbouring rows of two sequences, whose lists have some pages in common; heads that do not divide a tile; any page."""
    case = _selected_case(nh, nkv, hd, page, [19 * page + 3, 40 * page], 7, rows=19)
    pages = case[5]
    pages[3:9] = pages[3]                                   # all in common, in another order for one
    pages[5] = pages[5].flip(-1)
    _selected_check(dev, nh, nkv, case)


def test_selected_prompts_with_lists_in_any_order(dev):
    """Rows side by side: lists with pages twice, empty entries anywhere, pages behind the context, nothing; rows without a context; rows of
    no sequence; pages that are none."""
    case = _selected_case(4, 2, 64, 16, [500, 300], 9, rows=24)
    q, k, v, tables, ctx, pages, seq = case
    pages[1] = pages[1].flip(-1)
    pages[2, 0] = torch.tensor([3, 3, -1, 30, 30, 99, 1 << 30, -(1 << 31), 0], dtype=I32)
    pages[4] = -1
    pages[9, 1] = torch.tensor([7] * 9, dtype=I32)
    pages[26:29] = torch.tensor([[-1, 2, -1, 5, 18, 17, -1, 4, 0]], dtype=I32)
    ctx[12], ctx[13] = 0, -4
    got = _selected_check(dev, 4, 2, case)
    assert (got[4] == 0).all() and (got[12:14] == 0).all()
    given = [x.clone() for x in case]
    given[3][0, 7], given[3][1, 5], given[6][17], given[6][40] = -1, 1 << 30, 2, -1
    got = longctx.paged_selected(*(x.to(dev) for x in given[:6]), 4, 2, 0.125, row_seq=given[6].to(dev))
    gone = pages.clone()
    gone[(pages == 7) & (seq == 0)[:, None, None]] = -1
    gone[(pages == 5) & (seq == 1)[:, None, None]] = -1
    gone[17], gone[40] = -1, -1
    want, tol = _selected_want(4, 2, 0.125, *case[:5], gone, seq)
    _close(got, want, tol)


@pytest.mark.parametrize("nh,count,lens,rows", [(1, 90, [9000], 33), (2, 300, [8000], 9), (8, 150, [3000, 2500], 18)])
def test_selected_prompts_with_long_lists(dev, nh, count, lens, rows):
    """Rows that go together have more pages between them than a workgroup holds at a time."""
    _selected_check(dev, nh, 1, _selected_case(nh, 1, 64, 16, lens, count, rows=rows))


def test_selected_prompts_and_pages_of_other_rows(dev):
    """A page that one row has in its list, and its neighbour has not, holds NaN and infinities: they reach that row alone.  So do the keys
    of the neighbour's own step that a row does not see."""
    case = _selected_case(4, 2, 64, 16, [320], 4, rows=22)
    q, k, v, tables, ctx, pages, seq = case
    pages[:] = torch.tensor([1, 4, 9, 19], dtype=I32)
    pages[:, :, 3] = ((ctx - 1) // 16)[:, None]
    pages[6, 0, 1], pages[7, 1, 2], pages[11, :, 0] = 5, 12, 2
    k[tables[0, 5], 0, 3] = math.nan
    v[tables[0, 12], 1, :, ::2] = math.inf
    v[tables[0, 2], :, 7] = math.nan
    k[tables[0, 19], :, 15], v[tables[0, 19], :, 15] = math.nan, math.inf      # the last row's own key
    got = longctx.paged_selected(*(x.to(dev) for x in case[:6]), 4, 2, 0.125, row_seq=seq.to(dev)).cpu()
    want, tol = _selected_want(4, 2, 0.125, *case)
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf())
    fin = want.isfinite()
    assert not fin[6, :128].any() and fin[5].all() and fin[8:11].all() and not fin[21].any()
    _close(got[fin], want[fin], tol[fin])


def test_selected_prompts_large_scores_and_strides(dev):
    case = _selected_case(8, 2, 64, 16, [600, 200], 6, rows=20, extra=40)
    case[0].mul_(1e3)
    out = torch.full((40, 8 * 64 + 24), 5.0, dtype=BF16, device=dev)
    for scale in (0.125, -0.125, 0.0):
        got = _selected_check(dev, 8, 2, case, scale=scale, out=out)
        assert got.data_ptr() == out.data_ptr() and (out[:, 512:] == 5.0).all()


@pytest.mark.parametrize("count,lens,nh", [(12, [500], 4), (200, [9000], 4), (700, [13000], 4), (90, [3000] * 8, 16)])
def test_selected_what_is_no_number_stays(dev, count, lens, nh):
    """A query that is no number, such a key among the first of a list that is empty behind it, and an infinite value that hardly counts, where lists
    are cut and where they are not."""
    q, k, v, tables, ctx, pages, seq = case = _selected_case(nh, 1, 64, 16, lens, count)
    scale = 0.125
    tol = _selected_want(nh, 1, scale, *case)[1]
    q[0, 70] = math.nan                                # the second head
    got = longctx.paged_selected(*(x.to(dev) for x in case[:6]), nh, 1, scale)
    want, _ = _selected_want(nh, 1, scale, *case)
    assert want[0, 64:128].isnan().all() and torch.equal(got.isnan().cpu(), want.isnan())
    fin = want.isfinite()
    _close(got.cpu()[fin], want[fin], tol[fin])
    q[0, 70] = 1.0
    full = pages.clone()
    pages[0, 0, 1:] = -1
    k[tables[0, pages[0, 0, 0]], 0, 5] = math.nan
    assert longctx.paged_selected(*(x.to(dev) for x in case[:6]), nh, 1, scale)[0].isnan().all()
    k[tables[0, pages[0, 0, 0]], 0, 5] = 0.0
    pages.copy_(full)
    at = tables[0, pages[0, 0, 0]]                     # keys far below the others: weights of nothing in 32 bits
    q.abs_()
    k[at] = -200.0
    v[at, 0, 3, ::2] = math.inf
    got = longctx.paged_selected(*(x.to(dev) for x in case[:6]), nh, 1, scale)[0].view(nh, 32, 2).cpu()
    assert not got[..., 0].isfinite().any() and got[..., 1].isfinite().all()


def test_selected_lists_that_go_together_are_not_cut():
    """The entry refuses it before any launch, and the rule never asks for it: rows go together from 1024 (row, kv head) pairs on, lists are cut up to
    160 of them."""
    lib, at, n = ctypes.CDLL(dgi.build.build(group="longctx")), ctypes.c_void_p(4096), ctypes.c_longlong
    call = lambda plan, splits: lib.dgi_paged_selected(at, n(512), at, at, at, 4, 4, 1, 4, at, at, at, 4, at, n(512), at, at, splits, plan, plan, plan, 4,  # noqa: E731
                                                       8, 2, 64, 16, ctypes.c_float(0.1), None)
    assert call(at, 2) == -5 and call(at, 0) == -5 and call(None, 0) == -5


# ---- trees ------------------------------------------------------------------------------------------------------------------------------

def _tree_case(nh, nkv, hd, page, ctx, nodes, seed=0, extra=0, behind=0):
    g = _gen(seed)
    need = [-(-c // page) for c in ctx]
    pool = sum(need) + 3
    tables = _tables(g, need, max(max(need), 1) + 1, pool, "cpu")
    k, v = _randn(g, pool, nkv, page, hd), _randn(g, pool, nkv, page, hd)
    cu = torch.tensor([sum(nodes[:i]) for i in range(len(nodes) + 1)], dtype=I32)
    q = _randn(g, int(cu[-1]) + behind, nh * hd + extra)
    par = torch.full((len(nodes), 64), -1, dtype=I32)
    for a in range(1, 64):
        par[:, a] = torch.randint(0, a, (len(nodes),), generator=g)
    mask, _ = ops.tree_mask_ref(par)
    return q, k, v, tables, cu, torch.tensor(ctx, dtype=I32), mask


def _tree_want(nh, nkv, scale, q, k, v, tables, cu, ctx, mask):
    page, hd, G = k.shape[2], k.shape[3], nh // nkv
    o, tol = torch.zeros(q.shape[0], nh, hd, dtype=F64), torch.zeros(q.shape[0], nh, hd, dtype=F64)
    for s in range(len(cu) - 1):
        n, c = int(cu[s + 1] - cu[s]), int(ctx[s])
        ids = tables[s, : -(-c // page)].long()
        for a in range(n):
            row = int(cu[s]) + a
            see = torch.tensor([j < c - n or bool(int(mask[s, a]) >> (j - c + n) & 1) for j in range(c)], dtype=torch.bool)
            for h in range(nkv):
                kk, vv = k[ids, h].reshape(-1, hd)[:c][see], v[ids, h].reshape(-1, hd)[:c][see]
                x = q[row, : nh * hd].view(nkv, G, hd)[h]
                o[row, h * G:(h + 1) * G], tol[row, h * G:(h + 1) * G] = _attention(x, kk, vv, scale)
    return o.view(q.shape[0], -1), tol.view(q.shape[0], -1)


def _tree_check(dev, nh, nkv, case, max_nodes=64, scale=None, **kw):
    scale = scale or case[1].shape[-1] ** -0.5
    got = longctx.paged_tree(*(x.to(dev) for x in case), nh, nkv, scale, max_nodes=max_nodes, **kw)
    want, tol = _tree_want(nh, nkv, scale, *case)
    n = int(case[4][-1])
    _close(got[:n, : want.shape[1]], want[:n], tol[:n])
    return got


@pytest.mark.parametrize("nh,nkv,hd", [(8, 2, 64), (7, 1, 128), (16, 1, 64), (4, 4, 256), (8, 1, 128), (2, 2, 128)])
@pytest.mark.parametrize("nodes", [[1], [5, 9, 2], [64, 33]])
def test_tree(dev, nh, nkv, hd, nodes):
    """Trees of one to 64 nodes over contexts from nothing but the tree to several tiles."""
    ctx = [n + c for n, c in zip(nodes, [0, 1, 130] if len(nodes) == 3 else [47, 0])]
    _tree_check(dev, nh, nkv, _tree_case(nh, nkv, hd, 16, ctx, nodes), max_nodes=max(nodes))


@pytest.mark.parametrize("page", [8, 16, 32, 128])
def test_tree_pages(dev, page):
    _tree_check(dev, 8, 2, _tree_case(8, 2, 64, page, [200, 77, 12, 260], [12, 7, 12, 1], extra=16), max_nodes=12)


def test_tree_long_contexts(dev):
    """Contexts cut between workgroups, beside a short one; a limit of nodes that no tree reaches."""
    _tree_check(dev, 4, 1, _tree_case(4, 1, 64, 16, [5000, 20], [6, 8]), max_nodes=8)
    _tree_check(dev, 4, 1, _tree_case(4, 1, 64, 16, [9001], [3]))


def test_tree_empty_sequences_and_rows_behind(dev):
    """Padded sequences: no nodes, no context; rows of no sequence stay as they are."""
    case = _tree_case(8, 2, 64, 16, [30, 0, 40, 25], [4, 0, 3, 0], behind=5)
    out = torch.full((12, 512), 3.0, dtype=BF16, device=dev)
    _tree_check(dev, 8, 2, case, max_nodes=4, out=out)
    assert (out[7:] == 3.0).all()
    case = _tree_case(8, 2, 64, 16, [30, 40], [4, 3])
    case[5][1] = 0                                     # rows without keys
    got = longctx.paged_tree(*(x.to(dev) for x in case), 8, 2, 0.125, max_nodes=4)
    assert (got[4:] == 0).all() and (got[:4] != 0).any()
    case = _tree_case(8, 2, 64, 16, [30], [4])
    case[6][:] = 0                                     # nodes that see none of the tree, and no prefix
    case[5][0] = 4
    assert (longctx.paged_tree(*(x.to(dev) for x in case), 8, 2, 0.125, max_nodes=4) == 0).all()
    none = [case[0][:0], *case[1:3], case[3][:0], torch.zeros(1, dtype=I32), case[5][:0], case[6][:0]]
    assert longctx.paged_tree(*(x.to(dev) for x in none), 8, 2, 0.125).shape == (0, 512)


@pytest.mark.parametrize("nh,nkv,hd", [(8, 2, 64), (8, 1, 128), (2, 2, 64)])
def test_tree_keys_that_a_row_does_not_see(dev, nh, nkv, hd):
    """NaN and infinities in a drafted key or value reach the rows that see it, and no other; nor do those behind the context."""
    case = _tree_case(nh, nkv, hd, 16, [100, 45], [9, 13])
    q, k, v, tables, cu, ctx, mask = case
    for s, (c, n, bad) in enumerate([(100, 9, 4), (45, 13, 6)]):
        key = c - n + bad
        v[tables[s, key // 16], :, key % 16, ::3] = math.inf
        k[tables[s, (key + 1) // 16], :, (key + 1) % 16] = math.nan
        v[tables[s, (key + 1) // 16], :, (key + 1) % 16] = math.nan
        for j in range(c, -(-c // 16) * 16):
            k[tables[s, j // 16], :, j % 16], v[tables[s, j // 16], :, j % 16] = math.nan, math.nan
    got = longctx.paged_tree(*(x.to(dev) for x in case), nh, nkv, hd ** -0.5, max_nodes=13)
    want, tol = _tree_want(nh, nkv, hd ** -0.5, *case)
    assert torch.equal(got.isnan().cpu(), want.isnan())
    assert torch.equal(got.isinf().cpu(), want.isinf())
    fin = want.isfinite()
    assert fin.any() and not fin.all()
    _close(got.cpu()[fin], want[fin], tol[fin])


def test_tree_unknown_pages(dev):
    case = _tree_case(8, 2, 64, 16, [100], [5])
    case[3][0, 2] = -1
    got = longctx.paged_tree(*(x.to(dev) for x in case), 8, 2, 0.125, max_nodes=5)
    case[3][0, 2] = 1 << 30
    assert torch.equal(got, longctx.paged_tree(*(x.to(dev) for x in case), 8, 2, 0.125, max_nodes=5))
    q, k, v, tables, cu, ctx, mask = case
    keep = [j for j in range(100) if not 32 <= j < 48]      # the same as a context without those keys
    ids = [(int(tables[0, j // 16]), j % 16) for j in keep]
    k2, v2 = torch.zeros_like(k), torch.zeros_like(v)
    t2 = torch.arange(k.shape[0], dtype=I32)[None, : tables.shape[1]].contiguous()
    for i, (p, o) in enumerate(ids):
        k2[i // 16, :, i % 16], v2[i // 16, :, i % 16] = k[p, :, o], v[p, :, o]
    want, tol = _tree_want(8, 2, 0.125, q, k2, v2, t2, cu, torch.tensor([84], dtype=I32), mask)
    _close(got, want, tol)


def _without(case, gone):
    """The same trees over tables whose pages ``gone`` (sequence, place) are not there, and what they see: 64 bits and tolerances."""
    nh, nkv, scale, q, k, v, tables, cu, ctx, mask = case
    page, hd, G = k.shape[2], k.shape[3], nh // nkv
    o, tol = torch.zeros(q.shape[0], nh, hd, dtype=F64), torch.zeros(q.shape[0], nh, hd, dtype=F64)
    for s in range(len(cu) - 1):
        n, c = int(cu[s + 1] - cu[s]), int(ctx[s])
        ids = tables[s, : -(-c // page)].long()
        for a in range(n):
            see = torch.tensor([(s, j // page) not in gone and (j < c - n or bool(int(mask[s, a]) >> (j - c + n) & 1)) for j in range(c)], dtype=torch.bool)
            row = int(cu[s]) + a
            for h in range(nkv):
                kk, vv = k[ids, h].reshape(-1, hd)[:c][see], v[ids, h].reshape(-1, hd)[:c][see]
                heads = slice(h * G, (h + 1) * G)
                o[row, heads], tol[row, heads] = _attention(q[row, : nh * hd].view(nkv, G, hd)[h], kk, vv, scale)
    return o.view(q.shape[0], -1), tol.view(q.shape[0], -1)


@pytest.mark.parametrize("nh,nkv,hd,page", [(8, 2, 64, 16), (16, 1, 128, 16), (8, 2, 64, 4), (8, 2, 64, 128)])
def test_tree_pages_that_are_not_there(dev, nh, nkv, hd, page):
    """Ids outside the cache before the tree, among its own keys, at the end and everywhere, where page 0, which is nobody's, holds no numbers."""
    q, k, v, tables, cu, ctx, mask = _tree_case(nh, nkv, hd, page, [700, 200, 260, 150], [40, 33, 9, 12])
    nobody = torch.full_like(k[:1], math.nan), torch.full_like(v[:1], math.inf)
    nobody[1][:, :, ::2] = math.nan
    k, v, tables = torch.cat([nobody[0], k]), torch.cat([nobody[1], v]), tables + (tables >= 0)
    last = [-(-c // page) - 1 for c in ctx.tolist()]
    gone = {(0, 1), (0, last[0] // 2), (1, 0), (1, last[1]), (2, last[2] - 1)} | {(3, p) for p in range(last[3] + 1)}
    want, tol = _without((nh, nkv, 0.125, q, k, v, tables, cu, ctx, mask), gone)
    for i, (s, p) in enumerate(sorted(gone)):
        tables[s, p] = (-1, k.shape[0], 1 << 30, -(1 << 31))[i % 4]
    got = longctx.paged_tree(*(x.to(dev) for x in (q, k, v, tables, cu, ctx, mask)), nh, nkv, 0.125)
    _close(got, want, tol)
    assert (got[82:] == 0).all()


@pytest.mark.parametrize("nh,nkv,hd", [(32, 8, 128), (16, 1, 64), (8, 8, 64), (5, 1, 128), (16, 4, 256)])
def test_tree_many_sequences(dev, nh, nkv, hd):
    """More trees than a wave has lanes, of none to 20 nodes, contexts of nothing but the tree to some pages: both ways to split the work, with
    padded sequences between."""
    g = _gen(7)
    nodes = torch.randint(0, 21, (70,), generator=g).tolist()
    ctx = [n + int(c) for n, c in zip(nodes, torch.randint(0, 60, (70,), generator=g))]
    nodes[3], ctx[3], nodes[4], ctx[4], nodes[69], ctx[69] = 0, 0, 0, 33, 20, 20
    _tree_check(dev, nh, nkv, _tree_case(nh, nkv, hd, 16, ctx, nodes, behind=2), max_nodes=20)


@pytest.mark.parametrize("nh,nkv,hd,nodes", [(32, 2, 64, [64, 7, 64]), (16, 1, 128, [40, 64]), (3, 1, 64, [64, 64]), (12, 4, 256, [64, 50])])
@pytest.mark.parametrize("page", [4, 16, 256])
def test_tree_many_nodes(dev, nh, nkv, hd, nodes, page):
    """Trees of up to 1024 rows a kv head over contexts cut in parts."""
    _tree_check(dev, nh, nkv, _tree_case(nh, nkv, hd, page, [n + 700 * i + 33 for i, n in enumerate(nodes)], nodes, extra=8))


@pytest.mark.parametrize("nh,nkv,hd,ctx,nodes", [(4, 1, 64, [5000], [6]), (4, 1, 64, [9000, 300], [3, 8]), (8, 2, 64, [200], [6]), (16, 1, 128, [20000], [60])])
def test_tree_what_is_no_number_stays(dev, nh, nkv, hd, ctx, nodes):
    """A query that is no number, an infinite value that hardly counts, a key of the context's beginning that is no number."""
    q, k, v, tables, cu, ctx, mask = case = _tree_case(nh, nkv, hd, 16, ctx, nodes)
    most = max(nodes)
    call = lambda: longctx.paged_tree(*(x.to(dev) for x in case), nh, nkv, 0.125, max_nodes=most).cpu()
    clean = call()
    q[2, hd + 3] = math.nan
    got = call()
    assert got[2, hd: 2 * hd].isnan().all()
    got[2, hd: 2 * hd] = clean[2, hd: 2 * hd]
    assert torch.equal(got, clean)                     # nothing else
    q[2, hd + 3] = 1.0
    q.abs_()
    k[tables[0, 1]] = -200.0                           # keys far below the others: weights of nothing in 32 bits
    v[tables[0, 1], :, 3, ::2] = math.inf
    got = call()[: nodes[0]].view(nodes[0], nh, hd // 2, 2)
    assert not got[..., 0].isfinite().any() and got[..., 1].isfinite().all()
    k[tables[0, 0], :, 2] = math.nan
    got = call()
    assert got[: nodes[0]].isnan().all() and got[nodes[0]:].isfinite().all()


@pytest.mark.parametrize("nh,nkv,hd,nodes", [(4, 1, 64, 6), (8, 2, 128, 33), (4, 2, 256, 5)])
def test_tree_own_values_that_hardly_count(dev, nh, nkv, hd, nodes):
    """An infinite value of a node whose score leaves it a weight of nothing in 32 bits: no row that sees it is finite, all others are."""
    q, k, v, tables, cu, ctx, mask = case = _tree_case(nh, nkv, hd, 16, [200], [nodes])
    q.abs_()
    at = 200 - nodes + 1
    k[tables[0, at // 16], :, at % 16] = -200.0
    v[tables[0, at // 16], :, at % 16, ::2] = math.inf
    got = longctx.paged_tree(*(x.to(dev) for x in case), nh, nkv, 0.125).cpu().view(nodes, nh, hd // 2, 2)
    sees = (mask[0, :nodes] >> 1 & 1).bool()
    assert sees.any() and not sees.all()
    assert not got[sees][..., 0].isfinite().any() and got[~sees].isfinite().all() and got[..., 1].isfinite().all()


@pytest.mark.parametrize("nh,nkv,hd", [(32, 2, 64), (16, 2, 256)])
@pytest.mark.parametrize("scale", [-0.25, 1e-30, 4.0])
def test_tree_scales(dev, nh, nkv, hd, scale):
    _tree_check(dev, nh, nkv, _tree_case(nh, nkv, hd, 16, [300, 40, 64], [24, 40, 64]), scale=scale)


@pytest.mark.parametrize("nh,nkv", [(32, 2), (8, 2)])
def test_tree_scores_without_a_scale(dev, nh, nkv):
    """A scale of zero: every key that a row sees counts the same."""
    case = _tree_case(nh, nkv, 64, 16, [300, 40], [24, 40])
    got = longctx.paged_tree(*(x.to(dev) for x in case), nh, nkv, 0.0)
    want, tol = _tree_want(nh, nkv, 0.0, *case)
    _close(got, want, tol)


@pytest.mark.parametrize("nh,nkv", [(32, 2), (8, 2)])
@pytest.mark.parametrize("scale", [0.0, 2.0 ** -108, -(2.0 ** -110)])
def test_tree_large_scores_and_scales_of_nothing(dev, nh, nkv, scale):
    """Scores up to 2^112 before scales that are zero or bring them to the ordinary."""
    q, k, v, tables, cu, ctx, mask = case = _tree_case(nh, nkv, 64, 16, [300, 40], [24, 40])
    q.mul_(2.0 ** 60)
    k.mul_(2.0 ** 46)
    got = longctx.paged_tree(*(x.to(dev) for x in case), nh, nkv, scale)
    want, tol = _tree_want(nh, nkv, scale, *case)
    _close(got, want, tol)
    clean = got.cpu()
    q[3, 70], q[5, 2] = math.nan, math.inf             # a head of two rows
    got = longctx.paged_tree(*(x.to(dev) for x in case), nh, nkv, scale).cpu()
    assert got[3, 64:128].isnan().all() and got[5, :64].isnan().all()
    got[3, 64:128], got[5, :64] = clean[3, 64:128], clean[5, :64]
    assert torch.equal(got, clean)                     # nothing else


@pytest.mark.parametrize("nh,nkv,ctx,nodes", [(32, 2, [300, 40], [24, 40]), (8, 2, [300, 40], [24, 40]), (4, 1, [5000], [6]), (16, 1, [9000], [64])])
@pytest.mark.parametrize("signs", [1, -1])
@pytest.mark.parametrize("exp", [26, 34, 60, 105])
def test_tree_scores_of_any_size(dev, nh, nkv, ctx, nodes, signs, exp):
    """Scores around 2^exp, or all below -2^exp: a row's weight is its best key's wherever the next one is behind by more than the error of both."""
    q, k, v, tables, cu, ctx, mask = case = _tree_case(nh, nkv, 64, 16, ctx, nodes)
    if signs < 0:
        q.abs_()
        k.copy_(-k.abs())
    q.mul_(2.0 ** (exp // 2))
    k.mul_(2.0 ** (exp - exp // 2))
    got = longctx.paged_tree(*(x.to(dev) for x in case), nh, nkv, 0.125).cpu().view(-1, nkv, nh // nkv, 64)
    told = 0
    for s, (c, n) in enumerate(zip(ctx.tolist(), nodes)):
        ids = tables[s, : -(-c // 16)].long()
        for h in range(nkv):
            kk, vv = (x[ids, h].reshape(-1, 64)[:c].double() for x in (k, v))
            for a in range(n):
                row = int(cu[s]) + a
                see = torch.tensor([j < c - n or bool(int(mask[s, a]) >> (j - c + n) & 1) for j in range(c)])
                x = q[row].double().view(nkv, -1, 64)[h]
                score = (x @ kk.t() * 0.125).masked_fill(~see, -math.inf)
                error = 68 * U24 * 0.125 * (x.abs() @ kk.abs().t()).amax(1)
                best = score.topk(2, 1)
                clear = best.values[:, 0] - best.values[:, 1] > 2 * error + 100
                assert torch.equal(got[row, h][clear].double(), vv[best.indices[clear, 0]])
                told += int(clear.sum())
    assert told > 0.9 * sum(nodes) * nh and got.isfinite().all()


@pytest.mark.parametrize("nh,nkv", [(32, 2), (4, 2)])
def test_tree_rows_without_keys(dev, nh, nkv):
    """A tree whose sequence has no context, one whose nodes see nothing and have no prefix, one with fewer keys than nodes; no page is there."""
    case = _tree_case(nh, nkv, 64, 16, [200, 40, 33, 90], [40, 40, 33, 40])
    q, k, v, tables, cu, ctx, mask = case
    ctx[1] = 0
    mask[2] = 0
    tables[3] = -1
    got = longctx.paged_tree(*(x.to(dev) for x in case), nh, nkv, 0.125)
    assert (got[40:] == 0).all()
    want, tol = _tree_want(nh, nkv, 0.125, q, k, v, tables, cu[:2], ctx[:1], mask)
    _close(got[:40], want[:40], tol[:40])
    ctx[0] = 7                                         # the last 40 of seven keys: nodes 33 .. 39 have keys, and none has a prefix
    got = longctx.paged_tree(*(x.to(dev) for x in case), nh, nkv, 0.125)
    want, tol = _tree_want(nh, nkv, 0.125, q, k, v, tables, cu[:2], ctx[:1], mask)
    _close(got[:40], want[:40], tol[:40])


def test_tree_more_rows_than_sequences_say(dev):
    """More nodes than max_nodes: the first of them; row numbers behind q, and falling ones: nothing beyond."""
    case = _tree_case(4, 2, 64, 16, [90, 70], [30, 20], behind=3)
    out = torch.full((53, 256), 2.0, dtype=BF16, device=dev)
    longctx.paged_tree(*(x.to(dev) for x in case), 4, 2, 0.125, max_nodes=8, out=out)
    assert (out[8:30] == 2.0).all() and (out[38:] == 2.0).all() and (out[:8] != 2.0).any()
    q, k, v, tables, cu, ctx, mask = case
    cu = torch.tensor([0, 30, 99], dtype=I32)          # the second tree is cut at the last row
    got = longctx.paged_tree(*(x.to(dev) for x in (q, k, v, tables, cu, ctx, mask)), 4, 2, 0.125)
    want = longctx.paged_tree_ref(q, k, v, tables, torch.tensor([0, 30, 53], dtype=I32), ctx, mask, 4, 2, 0.125)
    tol = 2 * _tree_want(4, 2, 0.125, q, k, v, tables, torch.tensor([0, 30, 53], dtype=I32), ctx, mask)[1] + 2.0 ** -8 * want.abs().double()
    _close(got, want, tol)


# ---- together ---------------------------------------------------------------------------------------------------------------------------

def _server(dev, nh, nkv, hd, prompts, steps, page=16, seed=0):
    """State of a small server: caches, bounds, tables, and the rows of a prompt step and some decode steps."""
    g = _gen(seed)
    need = [-(-(n + steps) // page) for n in prompts]
    pool = sum(need) + 2
    tables = _tables(g, need, max(need), pool, dev)
    k, v = torch.full((pool, nkv, page, hd), math.nan, dtype=BF16, device=dev), torch.full((pool, nkv, page, hd), math.nan, dtype=BF16, device=dev)
    return dict(tables=tables, k=k, v=v, bounds=longctx.empty_bounds(k), cs=ops.rope_cos_sin(hd, max(prompts) + steps + 1, 10000.0, device=dev), g=g)


def _step(s, nh, nkv, hd, spans, count, page=16, qkv=None):
    """One step: positions ``spans`` = [(first, rows)] of each sequence; append, select, attend."""
    dev = s["k"].device
    pos = torch.cat([torch.arange(p, p + n) for p, n in spans]).to(I32).to(dev)
    seq = torch.tensor([i for i, (_, n) in enumerate(spans) for _ in range(n)], dtype=I32, device=dev)
    slots = s["tables"][seq.long(), pos.long() // page] * page + pos % page
    qkv = _randn(s["g"], len(pos), (nh + 2 * nkv) * hd, dev=dev) if qkv is None else qkv
    q = longctx.rope_cache_bounds(qkv, pos, s["cs"], nh, nkv, hd, slots, s["k"], s["v"], s["bounds"])
    pages = longctx.select_pages(q, s["bounds"], s["tables"], pos + 1, nh, nkv, page, count, 1, 2, row_seq=seq)
    return q, pos + 1, seq, pages, longctx.paged_selected(q, s["k"], s["v"], s["tables"], pos + 1, pages, nh, nkv, hd ** -0.5, row_seq=seq)


@pytest.mark.parametrize("nh,nkv,hd", [(8, 2, 64), (4, 1, 128)])
def test_steps_of_a_server(dev, nh, nkv, hd):
    """A prompt step, the rest of a prompt beside decode rows, decode steps: bounds as rebuilt, selections and outputs as in 64 bits, and where a
    context has no more pages than are kept, full attention."""
    prompts = [50, 7, 130]
    s = _server(dev, nh, nkv, hd, prompts, 20)
    count = 5
    plan = [[(0, 50), (0, 7), (0, 90)], [(50, 1), (7, 1), (90, 40)]] + [[(51 + i, 1), (8 + i, 1), (130 + i, 1)] for i in range(12)]
    for spans in plan:
        q, ctx, seq, pages, got = _step(s, nh, nkv, hd, spans, count)
        ends = [p + n for p, n in spans]
        rebuilt = longctx.empty_bounds(s["k"])
        held = [(int(s["tables"][i, j]), min(16, e - 16 * j)) for i, e in enumerate(ends) for j in range(-(-e // 16))]
        longctx.page_bounds(s["k"], rebuilt, torch.tensor([p for p, _ in held], dtype=I32, device=dev),
                            torch.tensor([n for _, n in held], dtype=I32, device=dev))
        assert torch.equal(rebuilt, s["bounds"])
        cpu = [x.cpu() for x in (q, s["k"], s["v"], s["tables"], ctx, pages, seq)]
        assert torch.equal(cpu[5], _selection64(cpu[0], s["bounds"].cpu(), cpu[3], cpu[4], nh, nkv, 16, count, 1, 2, cpu[6]))
        want, tol = _selected_want(nh, nkv, hd ** -0.5, *cpu)
        _close(got, want, tol)
        short = (ctx <= count * 16).cpu()
        full = ops.paged_decode_ref(q.cpu(), s["k"].cpu(), s["v"].cpu(), s["tables"].cpu()[seq.cpu().long()], ctx.cpu(), nh, nkv, hd ** -0.5)
        _close(got.cpu()[short], full[short], 2 * tol[short])
    # a draft of four nodes behind the last step, then its rejection: bounds stay wide, and the next step starts its page anew if it begins one
    pos = [p + 1 for (p, _) in plan[-1]]
    spans = [(p, 4) for p in pos]
    q, ctx, seq, _, _ = _step(s, nh, nkv, hd, spans, count)
    par = torch.tensor([[-1, 0, 0, 1]] * 3, dtype=I32)
    mask, _ = ops.tree_mask_ref(par)
    cu = torch.tensor([0, 4, 8, 12], dtype=I32)
    ends = torch.tensor([p + 4 for p in pos], dtype=I32)
    got = longctx.paged_tree(q, s["k"], s["v"], s["tables"], cu.to(dev), ends.to(dev), mask.to(dev), nh, nkv, hd ** -0.5, max_nodes=4)
    want, tol = _tree_want(nh, nkv, hd ** -0.5, q.cpu(), s["k"].cpu(), s["v"].cpu(), s["tables"].cpu(), cu, ends, mask)
    _close(got, want, tol)


# ---- refusals ---------------------------------------------------------------------------------------------------------------------------

def test_refusals(dev):
    def refused(f, *a, **kw):
        with pytest.raises(ValueError):
            f(*a, **kw)

    def change(args, i, x):
        return [*args[:i], x, *args[i + 1:]]

    qkv, pos, cs, slots, k, v, b = _append_case(dev, 8, 2, 64, 64, 0, 16, [(3, 5)])
    good = [qkv, pos, cs, 8, 2, 64, slots, k, v, b]
    longctx.rope_cache_bounds(*good)
    f = longctx.rope_cache_bounds
    refused(f, *change(good, 0, qkv[:, :500]))
    refused(f, *change(good, 1, pos[:4]))
    refused(f, *change(good, 1, pos.long()))
    refused(f, *change(good, 2, cs[:, :24].contiguous()))
    refused(f, *change(good, 3, 9))
    refused(f, *change(good, 3, 64))
    refused(f, *change(good, 6, slots[:-1]))
    refused(f, *change(good, 7, k[:, :1]))
    refused(f, *change(good, 8, v[1:]))
    refused(f, *change(good, 9, b[:, :, :1]))
    refused(f, *good, mode=2)
    refused(f, *good, out=torch.empty(5, 500, dtype=BF16, device=dev))

    f = longctx.page_bounds
    pages, lens = torch.zeros(2, dtype=I32, device=dev), torch.ones(2, dtype=I32, device=dev)
    refused(f, k[0], b, pages, lens)
    refused(f, k, b[1:], pages, lens)
    refused(f, k, b, pages.long(), lens)
    refused(f, k, b, pages, lens[:1])

    q, bb, tables, ctx, seq = (x.to(dev) for x in _select_case(8, 2, 64, 16, [300, 900], 3))
    f = longctx.select_pages
    good = [q, bb, tables, ctx, 8, 2, 16, 6]
    f(*good, row_seq=seq)
    refused(f, *good)      # a table for each row, or row_seq
    refused(f, *good, row_seq=seq[1:])
    refused(f, *good, row_seq=seq.long())
    refused(f, *good, first=5, recent=2, row_seq=seq)
    refused(f, *good, recent=0, row_seq=seq)
    refused(f, *good, first=-1, row_seq=seq)
    refused(f, *change(good, 0, q[:, :500]), row_seq=seq)
    refused(f, *change(good, 1, bb[:, :, 0]), row_seq=seq)
    refused(f, *change(good, 2, tables.long()), row_seq=seq)
    refused(f, *change(good, 3, ctx[1:]), row_seq=seq)
    refused(f, *change(good, 4, 64), row_seq=seq)
    refused(f, *change(good, 6, 0), row_seq=seq)
    refused(f, *good, row_seq=seq, out=torch.empty(6, 2, 5, dtype=I32, device=dev))
    refused(f, *change(good, 0, q.clone().requires_grad_()), row_seq=seq)

    q, k, v, tables, ctx, pages, seq = (x.to(dev) for x in _selected_case(8, 2, 64, 16, [300, 90], 6))
    f = longctx.paged_selected
    good = [q, k, v, tables, ctx, pages, 8, 2, 0.125]
    f(*good)
    refused(f, *change(good, 1, k[:, :, :12]))
    refused(f, *change(good, 2, v[1:]))
    refused(f, *change(good, 3, tables[:1]))
    refused(f, *change(good, 4, ctx[:1]))
    refused(f, *change(good, 5, pages[:, :1].contiguous()))
    refused(f, *change(good, 5, pages.long()))
    refused(f, *change(good, 5, pages[:, :, :0]))
    refused(f, *change(good, 6, 7))
    refused(f, *good, out=torch.empty(1, 512, dtype=BF16, device=dev))
    refused(f, *change(good, 0, q.clone().requires_grad_()))
    k12 = torch.zeros(4, 2, 12, 64, dtype=BF16, device=dev)
    refused(f, *change(change(good, 1, k12), 2, k12))      # pages of a power of two

    case = [x.to(dev) for x in _tree_case(8, 2, 64, 16, [300, 90], [6, 4])]
    f = longctx.paged_tree
    f(*case, 8, 2, 0.125, max_nodes=6)
    refused(f, *case, 8, 2, 0.125, max_nodes=65)
    refused(f, *case, 8, 2, 0.125, max_nodes=0)
    refused(f, *change(case, 4, case[4][:2]), 8, 2, 0.125)
    refused(f, *change(case, 6, case[6][:, :3].contiguous()), 8, 2, 0.125)
    refused(f, *change(case, 6, case[6].int()), 8, 2, 0.125)
    refused(f, *change(case, 3, case[3][:1]), 8, 2, 0.125)
    refused(f, *case, 8, 3, 0.125)


def test_refusals_of_dimensions(dev):
    """Tensors of fewer dimensions than an argument has, and caches without pages or tokens."""
    qkv, pos, cs, slots, k, v, b = _append_case(dev, 8, 2, 64, 64, 0, 16, [(3, 5)])
    one = torch.zeros(1, dtype=I32, device=dev)
    none = torch.zeros(0, 2, 16, 64, dtype=BF16, device=dev), torch.zeros(4, 2, 0, 64, dtype=BF16, device=dev)
    calls = [lambda: longctx.rope_cache_bounds(qkv, pos, cs[0].contiguous(), 8, 2, 64, slots, k, v, b),
             lambda: longctx.rope_cache_bounds(qkv, pos, cs[:0], 8, 2, 64, slots, k, v, b),
             lambda: longctx.rope_cache_bounds(qkv[0], pos, cs, 8, 2, 64, slots, k, v, b)]
    for q in (qkv[0, 0], qkv[0]):
        calls += [lambda q=q: longctx.select_pages(q, b, one[None], one, 8, 2, 16, 4),
                  lambda q=q: longctx.select_pages(q, b, one[None], one, 8, 2, 16, 4, out=torch.zeros(1, 2, 4, dtype=I32, device=dev)),
                  lambda q=q: longctx.paged_selected(q, k, v, one[None], one, one[None, None], 8, 2, 0.125),
                  lambda q=q: longctx.paged_tree(q, k, v, one[None], torch.cat([one, one]), one, one[None].long(), 8, 2, 0.125, max_nodes=1)]
    for c in none:
        calls += [lambda c=c: longctx.paged_selected(qkv[:1], c, c, one[None], one, one[None, None].expand(1, 2, 1).contiguous(), 8, 2, 0.125),
                  lambda c=c: longctx.paged_tree(qkv[:1], c, c, one[None], torch.cat([one, one + 1]), one, one[None].long(), 8, 2, 0.125, max_nodes=1)]
    for call in calls:
        with pytest.raises(ValueError):
            call()


@gpu
def test_refusals_of_the_kernels():
    """What only the kernels cannot take: other types and head sizes, starts off 16 bytes, tensors of other devices."""
    dev = "cuda"
    longctx.load_native(required=True)
    q, k, v, tables, ctx, pages, seq = (x.to(dev) for x in _selected_case(8, 2, 64, 16, [300, 90], 6))
    f = longctx.paged_selected
    good = [q, k, v, tables, ctx, pages, 8, 2, 0.125]
    with pytest.raises(ValueError):
        f(q.float(), *good[1:])
    with pytest.raises(ValueError):
        f(q, k.half(), v.half(), *good[3:])
    with pytest.raises(ValueError):
        f(torch.zeros(2, 8 * 64 + 1, dtype=BF16, device=dev)[:, 1:], *good[1:])
    with pytest.raises(ValueError):
        f(q, k.cpu(), v.cpu(), *good[3:])
    k32 = torch.zeros(4, 2, 16, 32, dtype=BF16, device=dev)
    with pytest.raises(ValueError):
        f(q, k32, k32, *good[3:])
    with pytest.raises(ValueError):
        f(*good, out=torch.empty(2, 512, dtype=torch.float32, device=dev))


# ---- on the device ----------------------------------------------------------------------------------------------------------------------

@gpu
def test_captured_steps():
    """Append, selection, attention and a tree in one graph, replayed with other inputs between the program's own work: as eagerly."""
    dev, nh, nkv, hd = "cuda", 8, 2, 64
    longctx.load_native(required=True)
    g = _gen(4)
    R, cols, nodes = 3, 60, 8
    tables = torch.randperm(R * cols, generator=g).to(I32).view(R, cols).to(dev)
    cs = ops.rope_cos_sin(hd, cols * 16 + 1, 10000.0, device=dev)
    k0, v0 = _randn(g, R * cols, nkv, 16, hd, dev=dev), _randn(g, R * cols, nkv, 16, hd, dev=dev)
    b0 = torch.stack([k0.amin(2), k0.amax(2)], 2)
    mask, _ = ops.tree_mask_ref(torch.tensor([[-1, 0, 0, 1, 1, 2, 3, 3]] * R, dtype=I32))
    st = dict(k=k0.clone(), v=v0.clone(), b=b0.clone(), qkv=torch.zeros(R * nodes, (nh + 2 * nkv) * hd, dtype=BF16, device=dev),
              pos=torch.zeros(R * nodes, dtype=I32, device=dev), slots=torch.zeros(R * nodes, dtype=I32, device=dev),
              ends=torch.zeros(R, dtype=I32, device=dev), seq=torch.arange(R, dtype=I32, device=dev).repeat_interleave(nodes),
              cu=torch.arange(0, R * nodes + 1, nodes, dtype=I32, device=dev), mask=mask.to(dev))

    def step(s):
        q = longctx.rope_cache_bounds(s["qkv"], s["pos"], cs, nh, nkv, hd, s["slots"], s["k"], s["v"], s["b"])
        ctx = s["pos"] + 1
        pages = longctx.select_pages(q, s["b"], tables, ctx, nh, nkv, 16, 7, 1, 2, row_seq=s["seq"])
        o = longctx.paged_selected(q, s["k"], s["v"], tables, ctx, pages, nh, nkv, hd ** -0.5, row_seq=s["seq"])
        t = longctx.paged_tree(q, s["k"], s["v"], tables, s["cu"], s["ends"], s["mask"], nh, nkv, hd ** -0.5, max_nodes=nodes)
        return q, pages, o, t

    def load(s, seed):
        g = _gen(seed)
        starts = torch.randint(1, cols * 16 - nodes, (R,), generator=g)
        pos = (starts[:, None] + torch.arange(nodes)).view(-1)
        s["pos"].copy_(pos.to(I32))
        s["slots"].copy_((tables.cpu()[torch.arange(R).repeat_interleave(nodes), pos // 16] * 16 + pos % 16).to(I32))
        s["ends"].copy_((starts + nodes).to(I32))
        s["qkv"].copy_(_randn(g, *s["qkv"].shape))
        for name, x in (("k", k0), ("v", v0), ("b", b0)):
            s[name].copy_(x)

    with torch.inference_mode():
        load(st, 0)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(st)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step(st)
        for seed in range(1, 6):
            load(st, seed)
            want = [x.clone() for x in (*step(st), st["k"], st["v"], st["b"])]
            load(st, seed)
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip((*outs, st["k"], st["v"], st["b"]), want):
                assert torch.equal(a, b)


@gpu
def test_two_streams_at_once():
    """Calls on two streams, unlike in size, do not share scratch memory."""
    longctx.load_native(required=True)
    cases = [[x.cuda() for x in _selected_case(4, 1, 64, 16, [9000], 300, seed=1)], [x.cuda() for x in _selected_case(4, 1, 64, 16, [5000, 100], 200, seed=2)]]
    trees = [[x.cuda() for x in _tree_case(4, 1, 64, 16, [5000], [6], seed=3)], [x.cuda() for x in _tree_case(4, 1, 64, 16, [900, 4000], [9, 2], seed=4)]]

    def both(i):
        q, k, v, tables, ctx, pages, seq = cases[i]
        return longctx.paged_selected(q, k, v, tables, ctx, pages, 4, 1, 0.125, row_seq=seq), longctx.paged_tree(*trees[i], 4, 1, 0.125, max_nodes=9)

    want = [both(0), both(1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(both(i))
    torch.cuda.synchronize()
    for i in range(2):
        for a, b in got[i]:
            assert torch.equal(a, want[i][0]) and torch.equal(b, want[i][1])


@gpu
def test_offsets_past_32_bits():
    """A cache of more than 2^31 values: pages at its end are read and written where they lie."""
    longctx.load_native(required=True)
    dev, nh, nkv, hd, page = "cuda", 16, 8, 128, 16
    nb = (1 << 31) // (nkv * page * hd) + 70
    k = torch.zeros(nb, nkv, page, hd, dtype=BF16, device=dev)
    v = torch.zeros_like(k)
    g = _gen(9)
    last = torch.arange(nb - 64, nb, dtype=I32)
    small_k, small_v = _randn(g, 64, nkv, page, hd, dev=dev), _randn(g, 64, nkv, page, hd, dev=dev)
    k[last.long()], v[last.long()] = small_k, small_v
    perm = torch.randperm(64, generator=g).to(I32)
    tables, small_tables = last[perm.long()][None].contiguous().to(dev), perm[None].contiguous().to(dev)
    bounds, small_bounds = longctx.empty_bounds(k), longctx.empty_bounds(small_k)
    lens = torch.full((64,), 16, dtype=I32, device=dev)
    longctx.page_bounds(k, bounds, last.to(dev), lens)
    longctx.page_bounds(small_k, small_bounds, torch.arange(64, dtype=I32, device=dev), lens)
    assert torch.equal(bounds[last.long()], small_bounds)
    qkv = _randn(g, 3, (nh + 2 * nkv) * hd, dev=dev)
    pos = torch.tensor([1000, 1001, 1002], dtype=I32, device=dev)
    cs = ops.rope_cos_sin(hd, 1024, 10000.0, device=dev)
    outs = []
    for kk, vv, tt, bb in ((k, v, tables, bounds), (small_k, small_v, small_tables, small_bounds)):
        # 2^31 values are 2^27 slots of 16: slots stay within 32 bits where offsets do not
        slots = tt[0, pos.long() // 16] * 16 + pos % 16
        q = longctx.rope_cache_bounds(qkv, pos, cs, nh, nkv, hd, slots, kk, vv, bb)
        seq = torch.zeros(3, dtype=I32, device=dev)
        pages = longctx.select_pages(q, bb, tt, pos + 1, nh, nkv, 16, 20, 1, 1, row_seq=seq)
        o = longctx.paged_selected(q, kk, vv, tt, pos + 1, pages, nh, nkv, hd ** -0.5, row_seq=seq)
        mask, _ = ops.tree_mask_ref(torch.tensor([[-1, 0, 0]], dtype=I32))
        t = longctx.paged_tree(q, kk, vv, tt, torch.tensor([0, 3], dtype=I32, device=dev), torch.tensor([1003], dtype=I32, device=dev),
                               mask.to(dev), nh, nkv, hd ** -0.5, max_nodes=3)
        outs.append((q, pages, o, t, kk[tt[0].long()], vv[tt[0].long()], bb[tt[0].long()]))
    for a, b in zip(*outs):
        assert torch.equal(a, b)


@gpu
def test_prompts_and_large_trees_on_streams_and_in_graphs():
    """The forms for many rows: two streams at once, and two graphs that share their memory, replayed in turn between eager calls."""
    longctx.load_native(required=True)
    select = [[x.cuda() for x in _select_case(8, 2, 128, 16, lens, 40, seed=s)] for s, lens in ((1, [3000, 900]), (2, [1200]))]
    selected = [[x.cuda() for x in _selected_case(8, 2, 128, 16, lens, 9, rows=40, seed=s)] for s, lens in ((3, [700, 2000]), (4, [1500]))]
    trees = [[x.cuda() for x in _tree_case(32, 2, 128, 16, ctx, n, seed=s)] for s, ctx, n in ((5, [3000, 200, 640], [60, 33, 64]), (6, [900, 4000], [64, 40]))]

    def both(i):
        q, b, tables, ctx, seq = select[i]
        pages = longctx.select_pages(q, b, tables, ctx, 8, 2, 16, 12, 1, 2, row_seq=seq)
        q, k, v, tables, ctx, some, seq = selected[i]
        return (pages, longctx.paged_selected(q, k, v, tables, ctx, some, 8, 2, 0.1, row_seq=seq), longctx.paged_tree(*trees[i], 32, 2, 0.1))

    want = [both(0), both(1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(6):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(both(i))
    torch.cuda.synchronize()
    with torch.inference_mode():
        graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
        pool = torch.cuda.graph_pool_handle()
        for i in range(2):
            with torch.cuda.graph(graphs[i], pool=pool):
                outs.append(both(i))
        for turn in range(5):
            for i in (0, 1) if turn % 2 else (1, 0):
                graphs[i].replay()
                got[i].append([x.clone() for x in outs[i]])
            got[turn % 2].append(both(turn % 2))
            torch.cuda.synchronize()
    for i in range(2):
        for x in got[i]:
            for a, b in zip(x, want[i]):
                assert torch.equal(a, b)


@gpu
def test_many_rows_past_32_bits():
    """The forms for many rows over a cache of more than 2^31 values."""
    longctx.load_native(required=True)
    nkv, page, hd = 8, 16, 128
    nb = (1 << 31) // (nkv * page * hd) + 300
    k = torch.zeros(nb, nkv, page, hd, dtype=BF16, device="cuda")
    v, bounds = torch.zeros_like(k), torch.zeros(nb, nkv, 2, hd, dtype=BF16, device="cuda")
    q, k0, v0, tables, ctx, pages, seq = (x.cuda() for x in _selected_case(16, nkv, hd, page, [3000], 9, rows=40))
    far = nb - k0.shape[0]
    b0 = torch.stack([k0.amin(2), k0.amax(2)], 2)
    k[far:], v[far:], bounds[far:] = k0, v0, b0
    tree = [x.cuda() for x in _tree_case(16, nkv, hd, page, [300], [64])]
    outs = []
    for kk, vv, bb, at in ((k, v, bounds, far), (k0, v0, b0, 0)):
        outs.append((longctx.select_pages(q, bb, tables + at, ctx, 16, nkv, page, 12, 1, 1, row_seq=seq),
                     longctx.paged_selected(q, kk, vv, tables + at, ctx, pages, 16, nkv, 0.1, row_seq=seq),
                     longctx.paged_tree(tree[0], kk, vv, tables[:, :20].contiguous() + at, *tree[4:], 16, nkv, 0.1)))
    for a, b in zip(*outs):
        assert torch.equal(a, b) and (a != 0).any()


# ---- the forms for many rows, at the sizes of the tests above -----------------------------------------------------------------------------

@pytest.fixture
def crowd(monkeypatch):
    """Behind the rows of every call as many that see nothing as make the kernels take neighbouring rows together."""
    longctx.load_native(required=True)
    select, selected, more = longctx.select_pages, longctx.paged_selected, 20000

    def grown(x, value):
        return torch.cat([x, x.new_full((more, *x.shape[1:]), value)])

    def select_many(q, bounds, tables, ctx, *args, row_seq):
        assert q.is_cuda
        return select(grown(q, 1.0), bounds, tables, grown(ctx, 0), *args, row_seq=grown(row_seq, 0))[: q.shape[0]]

    def selected_many(q, k, v, tables, ctx, pages, *args, row_seq, out=None):
        assert q.is_cuda
        big = None if out is None else grown(out, 7.0)
        r = selected(grown(q, 1.0), k, v, tables, grown(ctx, 0), grown(pages, 3), *args, row_seq=grown(row_seq, 0), out=big)
        assert (r[q.shape[0]:, : args[0] * k.shape[3]] == 0).all()
        return r[: q.shape[0]] if out is None else out.copy_(r[: q.shape[0]])

    monkeypatch.setattr(longctx, "select_pages", select_many)
    monkeypatch.setattr(longctx, "paged_selected", selected_many)


@gpu
@pytest.mark.parametrize("rows,page,extra", [(37, 16, 0), (5, 64, 64), (64, 16, 8), (130, 32, 0)])
def test_crowd_select_rows_of_prompts(crowd, rows, page, extra):
    test_select_rows_of_prompts("cuda", rows, page, extra)


@gpu
@pytest.mark.parametrize("what", ["alike", "zeros", "close", "huge", "tiny", "no numbers", "a hundred alike", "two of a kind"])
@pytest.mark.parametrize("hd,pages", [(64, 300), (128, 200), (128, 1300), (256, 250)])
def test_crowd_select_every_bit(crowd, what, hd, pages):
    test_select_prompts_that_need_every_bit("cuda", what, hd, pages)


@gpu
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("q_exp,b_exp", [(-122, 40), (-127, 60), (-112, 0), (60, -130), (100, -128)])
def test_crowd_select_the_least_numbers(crowd, hd, q_exp, b_exp):
    test_select_prompts_of_the_least_numbers("cuda", hd, q_exp, b_exp)


@gpu
@pytest.mark.parametrize("hd,pages", [(64, 200), (256, 1000), (128, 1090), (64, 5000), (128, 8300), (256, 9000)])
def test_crowd_select_long_prompts(crowd, hd, pages):
    test_select_rows_of_long_prompts("cuda", hd, pages)


@gpu
@pytest.mark.parametrize("nh,nkv,hd", [(8, 2, 64), (18, 2, 128), (4, 4, 256)])
def test_crowd_select_beside_single_rows(crowd, nh, nkv, hd):
    test_select_prompts_beside_single_rows("cuda", nh, nkv, hd)


@gpu
@pytest.mark.parametrize("nh,nkv,hd,page", [(1, 1, 64, 16), (5, 1, 128, 4), (14, 2, 128, 32), (16, 1, 64, 16), (6, 2, 256, 16), (2, 2, 128, 128),
                                            (3, 1, 64, 1)])
def test_crowd_selected(crowd, nh, nkv, hd, page):
    test_selected_prompts("cuda", nh, nkv, hd, page)


@gpu
@pytest.mark.parametrize("nh,count,lens,rows", [(1, 90, [9000], 33), (2, 300, [8000], 9), (8, 150, [3000, 2500], 18)])
def test_crowd_selected_long_lists(crowd, nh, count, lens, rows):
    test_selected_prompts_with_long_lists("cuda", nh, count, lens, rows)


@gpu
@pytest.mark.parametrize("test", ["test_selected_prompts_with_lists_in_any_order", "test_selected_prompts_and_pages_of_other_rows",
                                  "test_selected_prompts_large_scores_and_strides", "test_selected_places_that_nobody_sees"])
def test_crowd_selected_places(crowd, test):
    globals()[test]("cuda")


@gpu
@pytest.mark.parametrize("nh,nkv,hd", [(8, 2, 64), (4, 1, 128)])
def test_crowd_steps_of_a_server(crowd, nh, nkv, hd):
    test_steps_of_a_server("cuda", nh, nkv, hd)


@gpu
@pytest.mark.parametrize("nh,nkv,hd,T,pages", [(28, 4, 128, 600, 90), (16, 8, 64, 700, 300), (4, 4, 256, 520, 60)])
def test_many_rows_as_one_by_one(nh, nkv, hd, T, pages):
    """A long portion beside decode rows: as on the CPU, and in the same step as row by row."""
    longctx.load_native(required=True)
    lens = [16 * pages, 16 * pages - 200, 300, 77]
    q, b, tables, ctx, seq = _select_case(nh, nkv, hd, 16, lens, T)
    rows = torch.cat([torch.arange(T), torch.arange(2 * T - 40, 2 * T), torch.tensor([3 * T - 1, 4 * T - 1])])
    q, ctx, seq = q[rows].contiguous(), ctx[rows].clamp(min=1), seq[rows].contiguous()
    want = longctx.select_pages(q, b, tables, ctx, nh, nkv, 16, 20, 1, 2, row_seq=seq)
    q, b, tables, ctx, seq = (x.cuda() for x in (q, b, tables, ctx, seq))
    pages_ = longctx.select_pages(q, b, tables, ctx, nh, nkv, 16, 20, 1, 2, row_seq=seq)
    assert torch.equal(pages_.cpu(), want)
    g = _gen(8)
    k, v = _randn(g, b.shape[0], nkv, 16, hd, dev="cuda"), _randn(g, b.shape[0], nkv, 16, hd, dev="cuda")
    got = longctx.paged_selected(q, k, v, tables, ctx, pages_, nh, nkv, hd ** -0.5, row_seq=seq)
    some = torch.randperm(len(rows), generator=g)[:60].tolist() + [T - 1, T, len(rows) - 2, len(rows) - 1]
    one = [x[some].cpu() for x in (q, ctx, pages_, seq)]
    want, tol = _selected_want(nh, nkv, hd ** -0.5, one[0], k.cpu(), v.cpu(), tables.cpu(), one[1], one[2], one[3])
    _close(got[some], want, tol)


@gpu
def test_selected_long_lists_of_many_rows():
    """Unions of so many rows that they are made for some of them at a time: no more memory than that, and rows on both sides of the border."""
    longctx.load_native(required=True)
    g, T, count = _gen(12), 5000, 512
    q, k, v, tables, _, _, _ = _selected_case(16, 8, 64, 16, [16 * 600], 1)
    q = _randn(g, T, 16 * 64)
    ctx = 16 * 600 - torch.randint(0, 200, (T,), generator=g).to(I32)
    pages = torch.full((T, 8, count), -1, dtype=I32)
    pages[:, :, 100:140] = torch.stack([torch.randperm(600, generator=g)[:40] for _ in range(T)]).to(I32)[:, None]
    seq = torch.zeros(T, dtype=I32)
    dev = [x.cuda() for x in (q, k, v, tables, ctx, pages)]
    seq_dev, out = seq.cuda(), torch.empty(T, 16 * 64, dtype=BF16, device="cuda")
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    longctx.paged_selected(*dev, 16, 8, 0.125, row_seq=seq_dev, out=out)
    assert torch.cuda.max_memory_allocated() - before <= 260 << 20
    some = [0, 1, 7, 8, 4080, 4095, 4096, 4097, 4103, 4111, 4999]
    want, tol = _selected_want(16, 8, 0.125, q[some], k, v, tables, ctx[some], pages[some], seq[some])
    _close(out[some], want, tol)


@pytest.fixture
def woods(monkeypatch):
    """Before and behind the sequences of every call as many without nodes as make the kernels take a sequence's pairs as tiles."""
    longctx.load_native(required=True)
    tree, more = longctx.paged_tree, 600

    def many(q, k, v, tables, cu, ctx, mask, nh, nkv, scale, max_nodes=64, out=None):
        assert q.is_cuda and k.shape[3] <= 128
        S = ctx.numel()
        around = lambda x, value: torch.cat([x.new_full((more, *x.shape[1:]), value), x, x.new_full((more, *x.shape[1:]), value)])
        cu = torch.cat([cu[:1].expand(more), cu, cu[-1:].expand(more)])
        max_nodes = max_nodes if max_nodes * (nh // nkv) > 32 else min(64, mask.shape[1])
        return tree(q, k, v, around(tables[:S], -1), cu, around(ctx, 33), around(mask[:S], -1), nh, nkv, scale, max_nodes=max_nodes, out=out)

    monkeypatch.setattr(longctx, "paged_tree", many)


@gpu
@pytest.mark.parametrize("nh,nkv,hd", [(8, 2, 64), (7, 1, 128), (16, 1, 64), (8, 1, 128), (2, 2, 128)])
@pytest.mark.parametrize("nodes", [[1], [5, 9, 2], [64, 33]])
def test_woods(woods, nh, nkv, hd, nodes):
    test_tree("cuda", nh, nkv, hd, nodes)


@gpu
@pytest.mark.parametrize("nh,nkv,hd,nodes", [(32, 2, 64, [64, 7, 64]), (16, 1, 128, [40, 64]), (3, 1, 64, [64, 64])])
@pytest.mark.parametrize("page", [4, 16, 256])
def test_woods_many_nodes(woods, nh, nkv, hd, nodes, page):
    test_tree_many_nodes("cuda", nh, nkv, hd, nodes, page)


@gpu
@pytest.mark.parametrize("nh,nkv,hd", [(8, 2, 64), (8, 1, 128), (2, 2, 64)])
def test_woods_keys_that_a_row_does_not_see(woods, nh, nkv, hd):
    test_tree_keys_that_a_row_does_not_see("cuda", nh, nkv, hd)


@gpu
@pytest.mark.parametrize("page", [8, 16, 32, 128])
def test_woods_pages(woods, page):
    test_tree_pages("cuda", page)


@gpu
@pytest.mark.parametrize("scale", [-0.25, 1e-30, 4.0])
def test_woods_scales(woods, scale):
    test_tree_scales("cuda", 32, 2, 64, scale)


@gpu
@pytest.mark.parametrize("test,args", [("test_tree_long_contexts", ()), ("test_tree_empty_sequences_and_rows_behind", ()), ("test_tree_unknown_pages", ()),
                                       ("test_tree_scores_without_a_scale", (32, 2)), ("test_tree_scores_without_a_scale", (8, 2)),
                                       ("test_tree_rows_without_keys", (32, 2)), ("test_tree_rows_without_keys", (4, 2))])
def test_woods_places(woods, test, args):
    globals()[test]("cuda", *args)


@gpu
@pytest.mark.parametrize("nh,nkv,hd,page", [(8, 2, 64, 16), (16, 1, 128, 16), (8, 2, 64, 4), (8, 2, 64, 128)])
def test_woods_pages_that_are_not_there(woods, nh, nkv, hd, page):
    test_tree_pages_that_are_not_there("cuda", nh, nkv, hd, page)


@gpu
@pytest.mark.parametrize("nh,nkv,hd,ctx,nodes", [(4, 1, 64, [5000], [6]), (8, 2, 64, [200], [6]), (16, 1, 128, [900, 9000], [60, 7])])
def test_woods_what_is_no_number_stays(woods, nh, nkv, hd, ctx, nodes):
    test_tree_what_is_no_number_stays("cuda", nh, nkv, hd, ctx, nodes)


@gpu
@pytest.mark.parametrize("nh,nkv,hd,nodes", [(4, 1, 64, 6), (8, 2, 128, 33)])
def test_woods_own_values_that_hardly_count(woods, nh, nkv, hd, nodes):
    test_tree_own_values_that_hardly_count("cuda", nh, nkv, hd, nodes)


@gpu
@pytest.mark.parametrize("scale", [0.0, 2.0 ** -108, -(2.0 ** -110)])
def test_woods_large_scores_and_scales_of_nothing(woods, scale):
    test_tree_large_scores_and_scales_of_nothing("cuda", 32, 2, scale)


@gpu
@pytest.mark.parametrize("signs", [1, -1])
@pytest.mark.parametrize("exp", [26, 34, 60, 105])
def test_woods_scores_of_any_size(woods, signs, exp):
    test_tree_scores_of_any_size("cuda", 32, 2, [300, 40], [24, 40], signs, exp)
    test_tree_scores_of_any_size("cuda", 16, 1, [3000], [64], signs, exp)


@gpu
@pytest.mark.parametrize("nh,nkv,hd,nodes,ctx", [(32, 8, 128, [64], [9000]), (64, 8, 128, [60, 33, 64, 50] * 3, [900, 300, 2000, 64] * 3),
                                                 (16, 1, 128, [64, 64], [20000, 64]), (64, 8, 64, [30] * 40, [1000] * 40)])
def test_trees_in_shares(nh, nkv, hd, nodes, ctx):
    """Whole row tiles, cut ones, and many parts of one: rows in random places against 64 bits."""
    longctx.load_native(required=True)
    g = _gen(11)
    case = _tree_case(nh, nkv, hd, 16, ctx, nodes)
    got = longctx.paged_tree(*(x.cuda() for x in case), nh, nkv, 0.1)
    q, k, v, tables, cu, ctx, mask = case
    for s in torch.randperm(len(nodes), generator=g)[:4].tolist():
        n, c = nodes[s], int(ctx[s])
        ids = tables[s, : -(-c // 16)].long()
        for a in {0, n - 1, int(torch.randint(0, n, (1,), generator=g))}:
            see = (torch.arange(c) < c - n) | torch.tensor([bool(int(mask[s, a]) >> max(j - c + n, 0) & 1) and j >= c - n for j in range(c)])
            row = int(cu[s]) + a
            for h in range(nkv):
                kk, vv = k[ids, h].reshape(-1, hd)[:c][see], v[ids, h].reshape(-1, hd)[:c][see]
                heads = slice(h * nh // nkv, (h + 1) * nh // nkv)
                want, tol = _attention(q[row, : nh * hd].view(nh, hd)[heads], kk, vv, 0.1)
                _close(got[row].view(nh, hd)[heads], want, tol, f"sequence {s} node {a} head {h}")


@gpu
@pytest.mark.parametrize("nkv,hd", [(1, 64), (3, 128)])
def test_select_rows_in_turn(nkv, hd):
    """Thousands of rows whose sequences take turns, a long portion among them, and more: groups that go together and groups that do not."""
    longctx.load_native(required=True)
    g = _gen(21)
    lens = torch.randint(600, 1000, (30,), generator=g).tolist()
    q, b, tables, _, _ = _select_case(2 * nkv, nkv, hd, 16, lens, 1)
    seq = torch.cat([torch.arange(300) % 30, torch.full((700,), 3), torch.arange(3500) % 29, torch.arange(64) // 4, torch.full((437,), 7)]).to(I32)
    ctx = (torch.tensor(lens)[seq.long()] - torch.randint(0, 300, (len(seq),), generator=g)).to(I32)
    q = _randn(g, len(seq), 2 * nkv * hd)
    want = longctx.select_pages(q, b, tables, ctx, 2 * nkv, nkv, 16, 20, 1, 2, row_seq=seq)
    got = longctx.select_pages(*(x.cuda() for x in (q, b, tables, ctx)), 2 * nkv, nkv, 16, 20, 1, 2, row_seq=seq.cuda())
    assert torch.equal(got.cpu(), want)
