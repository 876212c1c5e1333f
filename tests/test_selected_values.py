"""Values in attention over chosen pages: the history's are fp16(x), wherever a tile of keys is read
from, and those that are not finite reach the queries that see them alone.

Queries of zero give every key the same score exactly, so that outputs are means of values and no
score's error hides a value's: the fp32 sums of at most 900 terms of either sign err by 900 2^-24 of
the mean |v| at most (5.4e-5) and in the order of the root of their number (2e-6); a bf16 value errs by
up to 2^-9 of itself, 1.1e-3 in the root mean square, and a mean of 900 by 4e-5.  The largest error allowed is
the bound, the root mean square 1e-5."""
import math

import numpy as np
import pytest
import torch

from oracle.attention import read_history
from oscar_amd import ops
from test_page_select import KINDS, SHAPES, sparse_case

MOST, MEAN = 900 * 2.0 ** -24, 1e-5


def stage_everything(stage, seed):
    """Window copies of all tokens of pages 0 to 63, their values fp32 beside any 16-bit grid."""
    stage_k, stage_v, owner = stage
    owner.copy_(torch.arange(owner.shape[0], device=owner.device)[:, None].expand_as(owner))
    stage_v.copy_(torch.randn(stage_v.shape, generator=torch.Generator().manual_seed(seed)))


def attend(cuda, c, x, caches, stage, table, bounds, plan, d, has_new):
    q = x["q"].to(cuda)
    new = [x[n].to(cuda) for n in "kv"] if has_new else [None, None]
    chosen, pages = ops.select_pages(q, bounds, table.to(cuda), plan)
    out, lse = ops.attention_selected(q, *new, *caches, chosen, plan, c["scale"], stage, head_dim=d)
    return out.double().cpu(), lse.double().cpu(), pages.cpu()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("window", [True, False])
def test_one_cached_token(cuda, window, shape, dtype):
    """A query that sees one token gets its value, fp16(x), to the last bit: from the FP32 window or
    from the packed slot."""
    hk, d, reqs = shape["hk"], shape["d"], 4
    c, x, k_cache, v_cache, stage, table, bounds, plan = sparse_case(cuda, [1] * reqs, [1] * reqs, dtype=dtype, budget=6, first=1, last=3,
                                                                     window=window, has_new=False, **shape)
    if window:
        stage_everything(stage, 5)
    out, lse, _ = attend(cuda, c, x, (k_cache, v_cache), stage, table, bounds, plan, d, False)
    copies = None if stage is None else tuple(t.cpu().numpy() for t in stage)
    v = torch.cat([torch.from_numpy(np.asarray(read_history(c["k8"], c["v8"], c["bt"][r], 0, 1, hk, d, copies, "f16")[1])) for r in range(reqs)])
    assert torch.equal(out, v.double().repeat_interleave(shape["group"], 1))
    assert v.bfloat16().ne(v).any() and lse.isfinite().all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("hists,chunks,has_new", [([1900], [4], True), ([5, 33, 700], [1, 40, 3], True), ([130, 1500], [3, 9], False), ([0, 64], [5, 1], True)])
def test_means_of_window_copies(cuda, hists, chunks, has_new, shape, dtype):
    """Chosen pages that the FP32 window holds, with and without a chunk in the same tile: means of
    fp16(x) and of the chunk's values."""
    hk, group, d = shape["hk"], shape["group"], shape["d"]
    c, x, k_cache, v_cache, stage, table, bounds, plan = sparse_case(cuda, hists, chunks, dtype=dtype, budget=6, first=1, last=3, has_new=has_new, **shape)
    stage_everything(stage, 6)
    x["q"].zero_()
    out, lse, pages = attend(cuda, c, x, (k_cache, v_cache), stage, table, bounds, plan, d, has_new)
    copies, off = tuple(t.cpu().numpy() for t in stage), []
    for r, h in enumerate(hists):
        a, b = c["qsl"][r], c["qsl"][r + 1]
        cached = h if has_new else c["seqs"][r]
        old = np.asarray(read_history(c["k8"], c["v8"], c["bt"][r], 0, cached, hk, d, copies, "f16")[1])
        for kv in range(hk):
            at = [t for p in pages[r, kv].tolist() if p >= 0 for t in range(p * 128, min(p * 128 + 128, cached))]
            v = torch.from_numpy(old[at, kv]).double()
            if has_new:
                v = torch.cat([v, x["v"][a:b, kv].double()])
            for i in range(b - a):
                seen = len(v) - (b - a) + i + 1
                got = out[a + i, kv * group:(kv + 1) * group]
                assert (lse[a + i, kv * group:(kv + 1) * group] - math.log(seen)).abs().max() <= 1e-5
                error = (got - v[:seen].mean(0)).abs()
                assert (error - MOST * v[:seen].abs().mean(0)).max() <= 0
                off.append(error)
    assert torch.cat([e.flatten() for e in off]).square().mean().sqrt() <= MEAN


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf, 1e6])
def test_cached_values_that_are_not_finite(cuda, bad, shape, dtype):
    """Cached queries: a later token's value reaches none of the earlier queries, whether its copy in the
    FP32 window is not finite (or past fp16, 1e6) in a channel or its slot's constants are in all of them."""
    hk, group, d = shape["hk"], shape["group"], shape["d"]
    c, x, k_cache, v_cache, stage, table, bounds, plan = sparse_case(cuda, [1500, 40], [4, 5], dtype=dtype, budget=6, first=1, last=3, has_new=False, **shape)
    call = lambda stage: attend(cuda, c, x, (k_cache, v_cache), stage, table, bounds, plan, d, False)[0]  # noqa: E731
    clean, packed = call(stage), call(None)
    for r, at, sees in ((0, 1498, [2, 3]), (0, 1499, [3]), (1, 38, [7, 8])):
        page, off, head = int(table[r, at // 128]), at % 128, (at + r) % hk
        heads = slice(head * group, (head + 1) * group)
        seat = (page % stage[0].shape[0], off, head)
        assert stage[2][seat[0], off] == page
        hit = torch.zeros_like(clean, dtype=torch.bool)
        hit[sees, heads, 7] = True
        was = stage[1][seat].clone()
        stage[1][seat][7] = bad
        out = call(stage)
        assert torch.equal(~out.isfinite(), hit) and (math.isnan(bad) or (out[hit] == math.copysign(math.inf, bad)).all())
        assert (out - clean)[~hit].abs().max() <= 1e-3
        stage[1][seat] = was
        if abs(bad) == 1e6:
            continue
        hit[sees, heads] = True
        constants = k_cache[page, off, head, 6:8].view(torch.float16)
        was = constants.clone()
        constants[0] = bad  # the values' zero
        out = call(None)
        assert torch.equal(~out.isfinite(), hit) and (math.isnan(bad) or (out[hit] == bad).all())
        assert (out - packed)[~hit].abs().max() <= 1e-3
        constants.copy_(was)


@pytest.mark.gpu
def test_captured_again(cuda):
    """Tiles of window copies and a chunk in a graph: every replay gives what the eager call does, to
    the last bits of tiles taken in another order."""
    c, x, k_cache, v_cache, stage, table, bounds, plan = sparse_case(cuda, [2000], [4], hk=2, group=8, d=128, dtype="bf16", budget=6, first=1, last=3)
    stage_everything(stage, 7)
    q, k, v = (x[n].to(cuda) for n in "qkv")
    chosen, _ = ops.select_pages(q, bounds, table.to(cuda), plan)
    call = lambda: ops.attention_selected(q, k, v, k_cache, v_cache, chosen, plan, c["scale"], stage, head_dim=128)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = call()
    for _ in range(4):
        v.copy_(torch.randn_like(v))
        want, want_lse = (t.clone() for t in call())
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert (out - want).abs().max() <= 1e-3 and (lse - want_lse).abs().max() <= 1e-5
