"""Chosen pages (ops.page_bounds, plan_selected, select_pages, attention_selected): refusals and the
plan on the CPU; bounds bit for bit, choices and attention against plain evaluations on the GPU.

Bounds are values of the cache, and chosen pages whole numbers: equal, not near.  A score's products
have 8 or 11 bits times 11 and are exact in 64 bits, and with the tests' rows (exponents within
2^20 of each other) the sums of 256 of them as well, so that the order of a sum changes nothing.
Attention: the tolerances of the decode kernel's other tests (test_scored_attention.py)."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from oracle import cases
from oracle.attention import read_history
from oscar_amd import _lib, ops
from test_scored_attention import LSE_TOL, REL_TOL, reference

SHAPES = [dict(hk=1, group=6, d=256), dict(hk=2, group=8, d=128), dict(hk=2, group=5, d=256)]
KINDS = {"bf16": torch.bfloat16, "f16": torch.float16}


# ------------------------------------------------------------------ refusals (no launch)
def bounds_args(**changes):
    a = _lib.BoundsArgs(block_table=4096, block_table_stride=4, block_table_rows=2, block_table_cols=4, lengths=4096, seq_lens=4096,
                        num_reqs=2, max_new=5, bounds=4096)
    a.cache = _lib.Cache(k=4096, v=4096, num_blocks=4, block_size=128, num_kv_heads=1, head_dim=256)
    a.cache.k_stride[:] = [128 * 256, 256, 256]
    for name, value in changes.items():
        if name == "stride":
            a.cache.k_stride[1] = value
        else:
            setattr(a.cache if name.startswith("cache_") else a, name.removeprefix("cache_"), value)
    return a


@pytest.mark.parametrize("changes,message", [
    (dict(cache_head_dim=64), "head_dim 64"), (dict(num_reqs=-1), "out of range"), (dict(num_reqs=65536), "out of range"),
    (dict(cache_num_kv_heads=0), "out of range"), (dict(cache_num_kv_heads=65536), "out of range"), (dict(cache_block_size=0), "block_size"),
    (dict(max_new=-1), "max_new"), (dict(max_new=2 ** 31), "max_new"), (dict(bounds=None), "missing pointer"), (dict(lengths=None), "missing pointer"),
    (dict(block_table_rows=1), "rows"), (dict(block_table_cols=0), "rows"), (dict(block_table_stride=3), "rows"), (dict(bounds=4104), "aligned"),
    (dict(cache_k=4100), "aligned"), (dict(stride=250), "aligned"),
])
def test_bounds_refusals(changes, message):
    lib = _lib.load()
    assert lib.oscarop_page_bounds_v1(C.byref(bounds_args(**changes)), None) == -22
    assert message in lib.oscar_last_error().decode()
    assert lib.oscarop_page_bounds_v1(None, None) == -22
    assert lib.oscarop_page_bounds_v1(C.byref(bounds_args(num_reqs=0)), None) == 0
    assert lib.oscarop_page_bounds_v1(C.byref(bounds_args(max_new=0)), None) == 0


def select_args(**changes):
    fixed = dict(q=4096, num_tokens=4, num_q_heads=6, q_stride_token=1536, q_dtype=_lib.OSCAR_BF16, has_new=1, bounds=4096, num_blocks=9,
                 num_kv_heads=1, head_dim=256, block_size=128, block_table=4096, block_table_stride=50, block_table_rows=2,
                 block_table_cols=50, query_start_loc=4096, seq_lens=4096, num_reqs=2, max_pages=50, budget=9, first_pages=1,
                 last_pages=3, table=4096, pages=4096, workspace=4096, workspace_bytes=10 ** 6, arrivals=4096)
    return _lib.SelectArgs(**{**fixed, **changes})


@pytest.mark.parametrize("changes,message", [
    (dict(head_dim=64), "head_dim 64"), (dict(q_dtype=0), "q_dtype"), (dict(num_reqs=-1), "out of range"), (dict(num_kv_heads=0), "out of range"),
    (dict(max_pages=2 ** 25), "out of range"), (dict(num_q_heads=0), "multiple"), (dict(num_kv_heads=4), "multiple"), (dict(block_size=0), "block_size"),
    (dict(budget=4), "budget"), (dict(last_pages=0), "budget"), (dict(first_pages=-1), "budget"), (dict(table=None), "missing pointer"),
    (dict(seq_lens=None), "missing pointer"), (dict(block_table_rows=1), "rows"), (dict(block_table_stride=40), "rows"), (dict(q=None), "missing pointer"),
    (dict(bounds=None), "missing pointer"), (dict(num_blocks=0), "missing pointer"), (dict(arrivals=None), "missing pointer"), (dict(q=4100), "aligned"),
    (dict(q_stride_token=1500), "aligned"),
])
def test_select_refusals(changes, message):
    lib = _lib.load()
    assert lib.oscarop_select_v1(C.byref(select_args(**changes)), None) == -22
    assert message in lib.oscar_last_error().decode()


def test_select_workspace():
    lib = _lib.load()
    size = lambda **changes: lib.oscarop_select_workspace_bytes_v1(C.byref(select_args(**changes)))  # noqa: E731
    assert size() == 2 * 50 * 8 and size(max_pages=9) == 0 and size(num_reqs=65536) == -22
    assert lib.oscarop_select_v1(None, None) == lib.oscarop_select_workspace_bytes_v1(None) == -22
    assert lib.oscarop_select_v1(C.byref(select_args(workspace_bytes=799)), None) == -28
    assert lib.oscarop_select_v1(C.byref(select_args(workspace=4104)), None) == -28
    assert lib.oscarop_select_v1(C.byref(select_args(num_reqs=0)), None) == 0


@pytest.mark.parametrize("stride,message", [(49, "each KV head"), (0, "each KV head"), (51, "each KV head")])
def test_attention_refusals(stride, message):
    lib = _lib.load()
    a = _lib.AttnArgs(num_items=1, num_groups=1, block_table_cols=50, block_table_stride=101)
    a.cache.num_kv_heads, a.cache.head_dim = 2, 256
    assert lib.oscarop_attn_selected_v1(C.byref(a), None, stride, None) == -22 and message in lib.oscar_last_error().decode()
    a.cache.num_kv_heads = 0
    assert lib.oscarop_attn_selected_v1(C.byref(a), None, 50, None) == -22
    assert lib.oscarop_attn_selected_v1(C.byref(a), C.byref(_lib.Score(0.0, 4096)), 50, None) == -22
    assert lib.oscarop_attn_selected_v1(None, None, 50, None) == -22


def test_plan_refusals():
    plan = lambda **changes: ops.plan_selected([0, 1], [900], has_new=True, **{**dict(block_size=128, budget=5, num_kv_heads=1, group=6, head_dim=256,  # noqa: E731
                                                                                     device="cpu"), **changes})
    for bad in (dict(budget=2), dict(last_pages=0), dict(first_pages=-1), dict(block_size=0), dict(budget=4, first_pages=2, last_pages=2)):
        with pytest.raises(ValueError, match="budget"):
            plan(**bad)


@pytest.mark.parametrize("seq,n,last,fits", [(1280, 128, 1, True), (1280, 129, 1, False), (1281, 1, 1, True), (1281, 2, 1, False),
                                             (1281, 129, 2, True), (1281, 130, 2, False), (512, 500, 1, True)])
def test_cached_queries_in_the_last_pages(monkeypatch, seq, n, last, fits):
    """A query in a page that may be left out would not know what it sees (512 tokens: all pages are
    read); new keys stand behind the chosen pages, and any number of queries is served."""
    monkeypatch.setattr(ops, "cu_count", lambda device: 256)
    sizes = dict(block_size=128, budget=4, last_pages=last, num_kv_heads=1, group=6, head_dim=256, device="cpu")
    plan = lambda seq, has_new: ops.plan_selected([0, n], [seq], has_new=has_new, **sizes)  # noqa: E731
    monkeypatch.setattr(ops, "upload", lambda parts, device: [torch.from_numpy(np.array(p)) for p in parts])
    if fits:
        assert plan(seq, False).max_pages == -(-seq // 128)
    else:
        with pytest.raises(ValueError, match="cached queries"):
            plan(seq, False)
    assert plan(seq + n, True).max_pages == -(-seq // 128)


# ------------------------------------------------------------------ bounds
def plain_keys(k8, d):
    """The keys of every slot, fp16 [blocks, bs, hk, d]: mul, then add, in fp32, as the cache's reader."""
    k = torch.as_tensor(k8).view(torch.uint8)
    consts = k[..., :4].contiguous().view(torch.float16).float()
    codes = torch.stack([k[..., 32:32 + d // 4] >> s & 3 for s in (0, 2, 4, 6)], -1).flatten(-2).float()
    return (codes * consts[..., :1] + consts[..., 1:]).half()


def plain_bounds(bounds, k8, table, old, new, bs, d):
    out, keys = bounds.clone(), plain_keys(k8, d)
    for r, (a, b) in enumerate(zip(old, new)):
        if a < 0 or b <= a or (b - 1) // bs >= table.shape[1]:
            continue
        for col in range(a // bs, -(-b // bs)):
            page = int(table[r, col])
            if not 0 <= page < keys.shape[0]:
                continue
            x = keys[page, :min(bs, b - col * bs)]
            out[page] = torch.stack([x.amin(0), x.amax(0)], 1)
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("bs", [128, 32, 200])
def test_bounds(cuda, bs, shape):
    """Steps of one token and of many pages, from the border of a page and from within, requests that
    did not grow; the pages that were not touched keep what they had."""
    hk, d = shape["hk"], shape["d"]
    old = [0, 0, bs - 1, bs, 3 * bs + 7, 5, 250, 17]
    new = [1, 6 * bs + 1, bs, bs + 3, 9 * bs, 5, 251, 3]
    c = cases.make_case(new, [1] * len(new), hk=hk, group=1, d=d, bs=bs, window=False)
    cache, table = torch.from_numpy(c["k8"]).view(torch.int8), torch.from_numpy(c["bt"])
    before = torch.randn(cache.shape[0], hk, 2, d).half()
    want = plain_bounds(before, c["k8"], table, old, new, bs, d)
    got = before.to(cuda)
    out = ops.page_bounds(cache.to(cuda), got, table.to(cuda), torch.tensor(old, dtype=torch.int32, device=cuda),
                          torch.tensor(new, dtype=torch.int32, device=cuda), max_new=6 * bs + 1, head_dim=d)
    assert out is got and torch.equal(got.cpu(), want)
    assert not torch.equal(want, before)


@pytest.mark.gpu
def test_bounds_of_odd_constants(cuda):
    """NaN and infinite constants go through; pages outside the cache and lengths that do not fit touch
    nothing."""
    g = torch.Generator().manual_seed(1)
    cache = torch.randint(-128, 128, (6, 128, 1, 256), generator=g, dtype=torch.int8)
    consts = (torch.randn(6, 128, 1, 4, generator=g) * 3).half()
    consts[1, 5, 0, 0] = math.inf
    consts[2, 7, 0, 1] = math.nan
    consts[3, 9, 0, 1] = -math.inf
    cache[..., :8] = consts.view(torch.int8)
    table = torch.tensor([[0, 1, 2, 3], [4, -3, 2 ** 31 - 1, 5], [4, 5, 4, 5], [4, 5, 4, 5]], dtype=torch.int32)
    old, new = [0, 0, -1, 0], [512, 512, 500, 513]
    before = torch.randn(6, 1, 2, 256, generator=g).half()
    want = plain_bounds(before, cache, table, old, new, 128, 256)
    got = ops.page_bounds(cache.to(cuda), before.to(cuda), table.to(cuda), torch.tensor(old, dtype=torch.int32, device=cuda),
                          torch.tensor(new, dtype=torch.int32, device=cuda), max_new=513, head_dim=256)
    assert torch.equal(torch.isnan(got).cpu(), torch.isnan(want)) and torch.isnan(want).any() and torch.isinf(want).any()
    assert torch.equal(got.cpu().nan_to_num(7.0), want.nan_to_num(7.0))
    with pytest.raises(ValueError, match="bounds"):
        ops.page_bounds(cache.to(cuda), before.float().to(cuda), table.to(cuda), got[:0, 0, 0, 0].int(), got[:0, 0, 0, 0].int(), max_new=1, head_dim=256)
    with pytest.raises(ValueError, match="rows"):
        x = torch.zeros(9, dtype=torch.int32, device=cuda)
        ops.page_bounds(cache.to(cuda), got, table.to(cuda), x, x, max_new=1, head_dim=256)


@pytest.mark.gpu
def test_pages_past_four_gigabytes(cuda):
    """Bounds and attention of pages at both ends of a cache of 5.2 GB: what the same pages give in a
    small one."""
    hk, d, blocks = 4, 256, 40000
    g = torch.Generator().manual_seed(9)
    small = [torch.randint(-128, 128, (8, 128, hk, d), generator=g, dtype=torch.int8) for _ in range(2)]
    for c in small:
        c[..., :8] = (torch.randn(8, 128, hk, 4, generator=g) * 0.5).half().view(torch.int8)
    large = [torch.empty(blocks, 128, hk, d, dtype=torch.int8, device=cuda) for _ in range(2)]
    where = torch.tensor([0, blocks - 1, 3, blocks - 2, 16383, 16384, 32768, blocks - 3])
    q, k, v = (torch.randn(1, n * hk, d, generator=g).bfloat16().to(cuda) for n in (2, 1, 1))
    ends = torch.tensor([1000], dtype=torch.int32, device=cuda)
    got = []
    for caches, at in (([c.to(cuda) for c in small], torch.arange(8)), (large, where)):
        for c, s in zip(caches, small):
            c[at.to(cuda)] = s.to(cuda)
        table = at.to(torch.int32)[None].to(cuda)
        bounds = torch.zeros(caches[0].shape[0], hk, 2, d, dtype=torch.float16, device=cuda)
        ops.page_bounds(caches[0], bounds, table, ends * 0, ends, max_new=1000, head_dim=d)
        plan = ops.plan_selected([0, 1], [1001], has_new=True, block_size=128, budget=5, num_kv_heads=hk, group=2, head_dim=d, device=cuda)
        chosen, pages = ops.select_pages(q, bounds, table, plan)
        got.append((bounds[at.to(cuda)], pages, *ops.attention_selected(q, k, v, *caches, chosen, plan, d ** -0.5, head_dim=d)))
    assert all(torch.equal(a, b) for a, b in zip(got[0][:2], got[1][:2])) and got[0][0].any()
    assert (got[0][2] - got[1][2]).abs().max() <= 1e-3 and (got[0][3] - got[1][3]).abs().max() <= 1e-5


# ------------------------------------------------------------------ the choice
def plain_choice(q, bounds, table, qsl, seqs, has_new, bs, budget, first, last, hk):
    """Scores in 64 bits from the definition, then the pages one by one."""
    group, chosen = q.shape[1] // hk, []
    for r, seq in enumerate(seqs):
        a, b = qsl[r], qsl[r + 1]
        pages = -(-(seq - (b - a if has_new else 0)) // bs)
        for h in range(hk):
            cols = list(range(pages))
            if pages > budget:
                mid = cols[first:pages - last]
                x = bounds[table[r, mid].long().clamp(0, len(bounds) - 1), h].double()
                rows = q[a:b, h * group:(h + 1) * group].double().reshape(-1, q.shape[2])
                # max(q low, q high) as both bounds' parts, exact as they are
                parts = rows[:, None] * ((x[:, 1] + x[:, 0]) / 2)[None] + rows.abs()[:, None] * ((x[:, 1] - x[:, 0]) / 2)[None]
                sums = parts.sum(-1)
                sums = torch.where(sums.isfinite(), sums, math.inf)
                s = sums.amax(0) if b > a else torch.zeros(len(mid)).double()
                order = sorted(range(len(mid)), key=lambda i: (-s[i].item(), i))
                cols = sorted(cols[:first] + [mid[i] for i in order[:budget - first - last]] + cols[pages - last:])
            chosen.append(cols + [-1] * (budget - len(cols)))
    return torch.tensor(chosen, dtype=torch.int32).view(len(seqs), hk, budget)


def choose(cuda, q, bounds, table, qsl, seqs, *, hk, d, budget, first=1, last=1, has_new=True, bs=128):
    plan = ops.plan_selected(qsl, seqs, has_new=has_new, block_size=bs, budget=budget, first_pages=first, last_pages=last, num_kv_heads=hk,
                             group=q.shape[1] // hk, head_dim=d, device=cuda)
    got, pages = ops.select_pages(q.to(cuda), bounds.to(cuda), table.to(cuda), plan)
    want = plain_choice(q, bounds, table, qsl, seqs, has_new, bs, budget, first, last, hk)
    assert torch.equal(pages.cpu(), want)
    rows = table[:len(seqs), None].expand(-1, hk, -1)
    assert torch.equal(got.cpu(), torch.where(want >= 0, torch.gather(rows, 2, want.long().clamp(min=0)), -1))
    return plan, got, pages


def random_bounds(g, blocks, hk, d):
    x = torch.randn(blocks, hk, 2, d, generator=g) + torch.randn(blocks, hk, 1, 1, generator=g) * 0.3
    x = x.half()
    x[x.abs() < 2.0 ** -10] = 0.0  # exponents within the exact sums' range
    return torch.stack([x.amin(2), x.amax(2)], 2)


def random_queries(g, *shape, dtype):
    x = (torch.randn(*shape, generator=g) * 2).to(dtype)
    x[x.abs() < 2.0 ** -9] = 0.0
    return x


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("seqs,counts,budget,first,last", [
    ([5000], [1], 8, 1, 3), ([300, 128 * 9, 128 * 9 + 1, 128 * 9 + 2, 20000], [1, 1, 1, 1, 1], 9, 1, 1), ([9000, 70000, 4000], [4, 1, 5], 33, 0, 2),
    ([30000], [40], 64, 2, 3), ([6000] * 40, [2] * 40, 7, 1, 1), ([40000, 3], [0, 3], 12, 1, 4)])
def test_choice(cuda, seqs, counts, budget, first, last, shape, dtype):
    """Histories within the budget, at it and above, one query and more than LDS holds at a time,
    requests without queries, few lists and many."""
    g = torch.Generator().manual_seed(sum(seqs))
    hk, d = shape["hk"], shape["d"]
    qsl = [0] + np.cumsum(counts).tolist()
    cols = max(-(-s // 128) for s in seqs) + 1
    table = torch.randperm(cols * len(seqs), generator=g).to(torch.int32).view(len(seqs), cols)
    choose(cuda, random_queries(g, qsl[-1], hk * shape["group"], d, dtype=KINDS[dtype]), random_bounds(g, cols * len(seqs), hk, d), table, qsl, seqs,
           hk=hk, d=d, budget=budget, first=first, last=last)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [40, 700, 5000])
@pytest.mark.parametrize("budget", [6, 30, 39])
def test_ties(cuda, n, budget):
    """Scores of few values (the earlier page first), all the same, and from both signs; more pages than
    LDS holds."""
    g = torch.Generator().manual_seed(n)
    table = torch.randperm(n, generator=g).to(torch.int32)[None]
    q = random_queries(g, 1, 6, 256, dtype=torch.bfloat16)
    few = random_bounds(g, 5, 1, 256)
    for bounds in (few[torch.randint(0, 5, (n,), generator=g)], few[:1].expand(n, -1, -1, -1).contiguous(),
                   torch.zeros(n, 1, 2, 256).half(), -few[torch.randint(0, 2, (n,), generator=g)].flip(2),
                   torch.where(torch.rand(n, 1, 1, 1, generator=g) < 0.5, 0.0, -0.0).half().expand(-1, 1, 2, 256).contiguous()):
        choose(cuda, q, bounds, table, [0, 1], [n * 128 + 1], hk=1, d=256, budget=budget)


@pytest.mark.gpu
def test_scores_that_are_not_finite(cuda):
    """A bound that is not finite makes a page the largest, whatever its sign and the query's; a
    query, all pages alike."""
    g = torch.Generator().manual_seed(3)
    n = 60
    bounds, table = random_bounds(g, n, 1, 128), torch.arange(n, dtype=torch.int32)[None]
    bounds[11, 0, 1, 3] = math.nan
    bounds[31, 0, 1, 3] = math.inf
    bounds[32, 0, :, 5] = -math.inf
    q = random_queries(g, 2, 8, 128, dtype=torch.float16)
    q[..., 3] = 1.0
    q[..., 5] = 2.0
    _, _, pages = choose(cuda, q, bounds, table, [0, 2], [n * 128 + 2], hk=1, d=128, budget=5, last=2)
    assert pages[0, 0].tolist() == [0, 11, 31, 58, 59]
    q[1, 2, 7] = math.nan  # a query that is not a number: every page's score
    _, _, pages = choose(cuda, q, bounds, table, [0, 2], [n * 128 + 2], hk=1, d=128, budget=5, last=2)
    assert pages[0, 0].tolist() == [0, 1, 2, 58, 59]


@pytest.mark.gpu
def test_scores_near_each_other(cuda):
    """Scores that differ in their last bits of 64 are told apart, where 32 bits would take the earlier."""
    n, d = 50, 256
    g = torch.Generator().manual_seed(5)
    bounds = random_bounds(g, 1, 1, d).expand(n, -1, -1, -1).contiguous()
    q = random_queries(g, 1, 1, d, dtype=torch.bfloat16)
    q[0, 0, :2] = torch.tensor([1.0, 2.0 ** -9])
    bounds[:, 0, :, 0] = 60000.0
    bounds[:, 0, :, 1] = (torch.arange(n)[:, None] * 2.0 ** -12).half()
    _, _, pages = choose(cuda, q, bounds, torch.arange(n, dtype=torch.int32)[None], [0, 1], [n * 128 + 1], hk=1, d=d, budget=6)
    assert pages[0, 0].tolist() == [0, 45, 46, 47, 48, 49]


@pytest.mark.gpu
def test_requests_that_do_not_fit(cuda):
    """Lists on the device that are not the plan's: -1 throughout, and nothing is read."""
    g = torch.Generator().manual_seed(7)
    bounds, table = random_bounds(g, 60, 1, 256), torch.randperm(60, generator=g).to(torch.int32).view(2, 30)
    q = random_queries(g, 2, 6, 256, dtype=torch.bfloat16)
    plan, want, _ = choose(cuda, q, bounds, table, [0, 1, 2], [3700, 3000], hk=1, d=256, budget=9)
    for qsl, seqs in (([0, 1, 3], [3700, 3000]), ([0, 1, 2], [3700, 0]), ([0, 1, 2], [3700, 31 * 128]), ([0, 1, -5], [3700, 3000])):
        plan.qsl.copy_(torch.tensor(qsl, dtype=torch.int32))
        plan.seqs.copy_(torch.tensor(seqs, dtype=torch.int32))
        got, pages = ops.select_pages(q.to(cuda), bounds.to(cuda), table.to(cuda), plan)
        assert torch.equal(got[0], want[0]) and (got[1] == -1).all() and (pages[1] == -1).all()


# ------------------------------------------------------------------ attention
def sparse_case(cuda, hists, chunks, *, hk, group, d, dtype, budget, first, last, window=True, has_new=True):
    c = cases.make_case(hists, chunks, hk=hk, group=group, d=d, window=window, fresh=has_new)
    x = {name: torch.from_numpy(c[name]).to(KINDS[dtype]) for name in ("qkv" if has_new else "q")}
    k_cache, v_cache = (torch.from_numpy(c[name]).view(torch.int8).to(cuda) for name in ("k8", "v8"))
    stage = None if c["stage"] is None else tuple(torch.from_numpy(a).to(cuda) for a in c["stage"])
    table = torch.from_numpy(c["bt"])
    bounds = torch.zeros(k_cache.shape[0], hk, 2, d, dtype=torch.float16, device=cuda)
    ends = torch.tensor(hists, dtype=torch.int32, device=cuda)
    ops.page_bounds(k_cache, bounds, table.to(cuda), ends * 0, ends, max_new=max(hists), head_dim=d)
    plan = ops.plan_selected(c["qsl"], c["seqs"], has_new=has_new, block_size=128, budget=budget, first_pages=first, last_pages=last,
                             num_kv_heads=hk, group=group, head_dim=d, device=cuda, window=(0, 256) if window else (0, 0))
    return c, x, k_cache, v_cache, stage, table, bounds, plan


@pytest.mark.gpu
@pytest.mark.parametrize("cap", [0.0, 20.0])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("hists,chunks,has_new", [([6000], [1], True), ([2000, 130, 128 * 12, 0], [4, 2, 9, 3], True), ([3000, 500], [2, 3], False),
                                                  ([2700, 1500], [260, 300], False), ([1400], [200], True)])
def test_attention(cuda, hists, chunks, has_new, shape, dtype, cap):
    """Chosen pages with their window copies and the current chunk, against the formula over those
    tokens alone; the pages that the kernel chose are the plain choice."""
    hk, group, d, budget = shape["hk"], shape["group"], shape["d"], 7
    c, x, k_cache, v_cache, stage, table, bounds, plan = sparse_case(cuda, hists, chunks, dtype=dtype, budget=budget, first=1, last=3, has_new=has_new, **shape)
    got_table, pages = ops.select_pages(x["q"].to(cuda), bounds, table.to(cuda), plan)
    assert torch.equal(pages.cpu(), plain_choice(x["q"], bounds.cpu(), table, c["qsl"], c["seqs"], has_new, 128, budget, 1, 3, hk))
    new = [x[name].to(cuda) for name in "kv"] if has_new else [None, None]
    out, lse = ops.attention_selected(x["q"].to(cuda), *new, k_cache, v_cache, got_table, plan, c["scale"], stage, head_dim=d, soft_cap=cap)
    out, lse = out.double().cpu(), lse.double().cpu()
    for r, h in enumerate(hists):
        a, b = c["qsl"][r], c["qsl"][r + 1]
        cached = h if has_new else c["seqs"][r]
        old = read_history(c["k8"], c["v8"], c["bt"][r], 0, cached, hk, d, c["stage"], "bf16" if dtype == "bf16" else "f16")
        for kv in range(hk):
            cols = [p for p in pages[r, kv].tolist() if p >= 0]
            at = np.concatenate([np.arange(p * 128, min(p * 128 + 128, cached)) for p in cols] or [np.arange(0)])
            k, v = (y[at][:, kv:kv + 1] for y in old)
            if has_new:
                k, v = (np.concatenate([y, x[n][a:b, kv:kv + 1].float().numpy()]) for y, n in ((k, "k"), (v, "v")))
            heads = slice(kv * group, (kv + 1) * group)
            want, want_lse, size = reference(x["q"][a:b, heads].float(), k, v, 0, c["scale"], cap, None,
                                             len(at) + 1 if has_new else len(at) - (b - a) + 1)
            assert (lse[a:b, heads] - want_lse).abs().max() <= LSE_TOL
            assert ((out[a:b, heads] - want).abs() - REL_TOL * size - 2.0 ** -17).max() <= 0


@pytest.mark.gpu
def test_all_pages_chosen_is_the_plain_decode(cuda):
    """A budget that every history fits in: the whole table for each KV head, and the decode's result
    to the roundings of a probability (2^-10 of sum p |v|: both round theirs, at half a step 2^-11)."""
    hists, chunks = [700, 3000], [2, 4]
    c, x, k_cache, v_cache, stage, table, bounds, plan = sparse_case(cuda, hists, chunks, hk=2, group=8, d=128, dtype="bf16", budget=30, first=1, last=1)
    q, k, v = (x[n].to(cuda) for n in "qkv")
    got_table, pages = ops.select_pages(q, bounds, table.to(cuda), plan)
    assert pages[0, :, :6].tolist() == [list(range(6))] * 2 and (pages[0, :, 6:] == -1).all()
    out, lse = ops.attention_selected(q, k, v, k_cache, v_cache, got_table, plan, c["scale"], stage, head_dim=128)
    dense = ops.plan_decode(c["qsl"], c["seqs"], has_new=True, num_kv_heads=2, group=8, head_dim=128, device=cuda, window=(0, 256))
    want, want_lse = ops.attention_decode(q, k, v, k_cache, v_cache, table.to(cuda), dense, c["scale"], stage, head_dim=128)
    assert (lse - want_lse).abs().max() <= 1e-5
    most = max(torch.as_tensor(read_history(c["k8"], c["v8"], c["bt"][r], 0, h, 2, 128, c["stage"], "f16")[1]).abs().max().item() for r, h in enumerate(hists))
    assert (out - want).abs().max() <= 2.0 ** -10 * max(most, v.abs().max().item())


@pytest.mark.gpu
def test_captured_streams_and_refusals(cuda):
    """Two graphs of choice and attention replayed in turn on two streams, with eager calls of another
    size and changed queries between; then what is refused."""
    hists, chunks = [5000, 2500], [2, 2]
    c, x, k_cache, v_cache, stage, table, bounds, plan = sparse_case(cuda, hists, chunks, hk=2, group=8, d=128, dtype="bf16", budget=9, first=1, last=3)
    q, k, v = (x[n].to(cuda) for n in "qkv")
    dev_table = table.to(cuda)

    def call(q):
        t, pages = ops.select_pages(q, bounds, dev_table, plan)
        return (*ops.attention_selected(q, k, v, k_cache, v_cache, t, plan, c["scale"], stage, head_dim=128), t, pages)

    inputs = [torch.randn_like(q) for _ in range(2)]
    call(q)
    torch.cuda.synchronize()
    graphs = []
    for y in inputs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = call(y)
        graphs.append((g, out))
    streams = [torch.cuda.Stream() for _ in graphs]
    small = ops.plan_selected([0, 2], [5002], has_new=True, block_size=128, budget=5, num_kv_heads=2, group=8, head_dim=128, device=cuda)
    for turn in range(4):
        for y in inputs:
            y.copy_(torch.randn_like(y))
        ops.select_pages(q, bounds, dev_table, small)
        want = [tuple(t.clone() for t in call(y)) for y in inputs]
        torch.cuda.synchronize()
        for s, (g, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for (_, out), w in zip(graphs, want):
            assert torch.equal(out[2], w[2]) and torch.equal(out[3], w[3])
            # (the decode's waves take tiles as they get to them: its last bits are not fixed)
            assert (out[0] - w[0]).abs().max() <= 1e-3 and (out[1] - w[1]).abs().max() <= 1e-5, turn

    t, _ = ops.select_pages(q, bounds, dev_table, plan)
    for bad, message in ((lambda: ops.select_pages(q.float(), bounds, dev_table, plan), "bf16 or fp16"),
                         (lambda: ops.select_pages(q[:, :9], bounds, dev_table, plan), "multiple"),
                         (lambda: ops.select_pages(q[:3], bounds, dev_table, plan), "more queries"),
                         (lambda: ops.select_pages(q, bounds[:, :1], dev_table, plan), "bounds"),
                         (lambda: ops.select_pages(q, bounds, dev_table[:, :20], plan), "cover"),
                         (lambda: ops.select_pages(q, bounds, dev_table[:1], plan), "rows"),
                         (lambda: ops.attention_selected(q, None, None, k_cache, v_cache, t, plan, 0.1, head_dim=128), "disagree"),
                         (lambda: ops.attention_selected(q, k, v, k_cache, v_cache, t[:, :, :5], plan, 0.1, head_dim=128), "budget"),
                         (lambda: ops.attention_selected(q, k, v, k_cache, v_cache, t[:1], plan, 0.1, head_dim=128), "rows"),
                         (lambda: ops.attention_selected(q, k, v, k_cache, v_cache, t.long(), plan, 0.1, head_dim=128), "table"),
                         (lambda: ops.attention_selected(q, k, v, k_cache[:, :64].contiguous(), v_cache[:, :64].contiguous(), t, plan, 0.1, head_dim=128), "pages of 128")):
        with pytest.raises(ValueError, match=message):
            bad()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_values_that_are_not_finite(cuda, bad, shape, dtype):
    """A value of the chunk that is not finite reaches the queries that see it, in its channel, and a
    key the queries that see it: the others and the other channels stay what they were."""
    hists, chunks = [1500, 40], [4, 3]
    c, x, k_cache, v_cache, stage, table, bounds, plan = sparse_case(cuda, hists, chunks, dtype=dtype, budget=6, first=1, last=3, **shape)
    q, k, v = (x[n].to(cuda) for n in "qkv")
    got_table, _ = ops.select_pages(q, bounds, table.to(cuda), plan)
    call = lambda k, v: ops.attention_selected(q, k, v, k_cache, v_cache, got_table, plan, c["scale"], stage, head_dim=shape["d"])[0].cpu()  # noqa: E731
    clean = call(k, v)
    for row, head, channel in ((2, 0, 5), (3, shape["hk"] - 1, shape["d"] - 1), (5, 0, 64)):
        sees = torch.zeros(7, dtype=torch.bool)
        sees[row:4 if row < 4 else 7] = True
        heads = slice(head * shape["group"], (head + 1) * shape["group"])
        hit = torch.zeros_like(clean, dtype=torch.bool)
        hit[:, heads, channel] = sees[:, None]
        worse = v.clone()
        worse[row, head, channel] = bad
        out = call(k, worse)
        assert torch.equal(~out.isfinite(), hit)
        assert math.isnan(bad) or (out[hit] == bad).all()
        # (the decode's waves take tiles as they get to them: its last bits are not fixed)
        assert (out - clean)[~hit].abs().max() <= 1e-3
        worse = k.clone()
        worse[row, head, channel] = math.nan
        out = call(worse, v)
        hit[:, heads] = sees[:, None, None]
        assert torch.equal(~out.isfinite(), hit) and (out - clean)[~hit].abs().max() <= 1e-3
