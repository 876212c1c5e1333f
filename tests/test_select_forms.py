"""select_pages in more than 512 workgroups of 8 pages, where one scores 32 pages with all rows of the
queries: every shape and type, several lists, lists whose last workgroups have nothing to score, more
rows than LDS holds, calls one after the other.  And what attention over chosen pages leaves out when it
rounds a probability times a value's scale, where the scales change along a history."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from oscar_amd import _lib, ops
from test_page_select import KINDS, SHAPES, choose, random_bounds, random_queries, sparse_case
from test_tree_attention import attn_args

MOST_BY_ROWS = 512  # workgroups


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("seqs,count,budget,first,last", [
    ([6000] * 100, 2, 7, 1, 1), ([70000, 300, 30000, 128 * 12 + 1] * 8, 1, 9, 1, 3), ([9000, 5000, 20000] * 16, 7, 16, 0, 2), ([100000], 1, 5, 1, 1)])
def test_many_workgroups(cuda, seqs, count, budget, first, last, shape, dtype):
    hk, d, group = shape["hk"], shape["d"], shape["group"]
    g = torch.Generator().manual_seed(len(seqs))
    qsl = [count * i for i in range(len(seqs) + 1)]
    cols = max(-(-s // 128) for s in seqs) + 1
    if len(seqs) > 1:
        assert -(-(cols - 1 - first - last) // 8) * hk * len(seqs) > MOST_BY_ROWS
    table = torch.randperm(cols * len(seqs), generator=g).to(torch.int32).view(len(seqs), cols)
    bounds = random_bounds(g, cols * len(seqs), hk, d)
    q = random_queries(g, qsl[-1], hk * group, d, dtype=KINDS[dtype])
    plan, table1, pages1 = choose(cuda, q, bounds, table, qsl, seqs, hk=hk, d=d, budget=budget, first=first, last=last)
    # the same again, one call behind the other on the stream, after one of other lists: the counters are at zero
    other = ops.plan_selected([0, 2], [3000], has_new=True, block_size=128, budget=4, num_kv_heads=hk, group=group, head_dim=d, device=cuda)
    dev = [q.to(cuda), bounds.to(cuda), table.to(cuda)]
    got = [ops.select_pages(*dev, plan) for _ in range(2)]
    ops.select_pages(dev[0][:2].repeat(1 + (len(q) < 2), 1, 1), *dev[1:], other)
    got += [ops.select_pages(*dev, plan)]
    assert all(torch.equal(t, table1) and torch.equal(p, pages1) for t, p in got)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("steps", [0, 12])
def test_scales_that_change_along_a_history(cuda, steps, shape, dtype):
    """Values' scales of 1, or of 1 to 4096 from page to page (past 255 the kernel lowers its factor in the
    middle of an item), probabilities of about 1 and 1/3 in each tile.

    A code's part c s of a value c s + z meets P' = fp16(p s) and a correction of 1.5 times what that
    rounding leaves out, d = p s - P', |d| <= 2^-11 p s.  Left is sum d (c - 1.5), where d is the same share
    of p s for all tokens of one p (scales are powers of two): at most 2^-11 |sum s (c - 1.5)| p over those of
    each p, for a row.  Beside it the fp32 sums of 16 terms of a tile, and of its waves' tiles: fewer than
    40 of 1.5 p s + p |v| each in a lane, 2^-24 of the partial sums at most, and scores' errors of 1e-6."""
    hk, group, d = shape["hk"], shape["group"], shape["d"]
    hists, chunks = [2300, 1500], [1, 2]
    c, x, k_cache, v_cache, _, table, bounds, plan = sparse_case(cuda, hists, chunks, dtype=dtype, budget=9, first=1, last=3, window=False, **shape)
    near = math.log(3.0) / (c["scale"] * 16.0)
    meta = c["k8"][..., :8].view(np.float16)  # K scale, K zero, V scale, V zero
    meta[..., 0] = 0.0
    meta[..., 1] = np.where(np.arange(128) % 32 == 7, near, 0.0)[None, :, None]  # one key of a tile three times the others
    for r in range(2):
        for col in range(c["bt"].shape[1]):
            s = 2.0 ** (col * 5 % (steps + 1))
            meta[c["bt"][r, col], :, :, 2], meta[c["bt"][r, col], :, :, 3] = s, -1.5 * s
    k_cache.copy_(torch.from_numpy(c["k8"]).view(torch.int8))
    for name in "qkv":
        x[name].zero_()
    x["q"][:, :, 0] = 16.0
    q, k, v = (x[n].to(cuda) for n in "qkv")
    chosen, pages = ops.select_pages(q, bounds, table.to(cuda), plan)
    out, lse = ops.attention_selected(q, k, v, k_cache, v_cache, chosen, plan, c["scale"], None, head_dim=d)
    out, pages = out.double().cpu(), pages.cpu()
    codes = np.stack([c["v8"][..., :d // 4] >> s & 3 for s in (0, 2, 4, 6)], -1).reshape(*c["v8"].shape[:3], d)
    for r, h in enumerate(hists):
        a, b = c["qsl"][r], c["qsl"][r + 1]
        for kv in range(hk):
            at = np.array([t for p in pages[r, kv].tolist() if p >= 0 for t in range(p * 128, min(p * 128 + 128, h))])
            page, off = c["bt"][r, at // 128], at % 128
            s, code = meta[page, off, kv, 2].astype(np.float64), codes[page, off, kv].astype(np.float64)
            key = x["k"].new_tensor(meta[page, off, kv, 1].astype(np.float32)).to(KINDS[dtype]).double().numpy()
            w = np.exp(16.0 * key * c["scale"])
            for i in range(b - a):
                total = w.sum() + i + 1  # the chunk's keys: scores of zero, values of zero
                want = (w * s) @ (code - 1.5) / total
                part = sum(np.abs((s * w * (key == z)) @ (code - 1.5)) for z in np.unique(key)) / total
                sizes = (w * s) @ (3.0 + np.abs(code - 1.5)) / total
                error = np.abs(out[a + i, kv * group:(kv + 1) * group].numpy() - want)
                assert (error - 2.0 ** -11 * part - (40 * 2.0 ** -24 + 1e-6) * sizes).max() <= 0
    assert lse.isfinite().all()


@pytest.mark.gpu
def test_a_step_without_queries(cuda):
    """A list of requests none of which has a row: every page scores alike, the earlier ones are chosen, and
    there is nothing to attend to."""
    g = torch.Generator().manual_seed(3)
    table = torch.randperm(80, generator=g).to(torch.int32).view(2, 40)
    q = torch.zeros(0, 6, 256, dtype=torch.bfloat16)
    plan, chosen, _ = choose(cuda, q, random_bounds(g, 80, 1, 256), table, [0, 0, 0], [5000, 300], hk=1, d=256, budget=6)
    k_cache = torch.zeros(80, 128, 1, 256, dtype=torch.int8, device=cuda)
    none = torch.zeros(0, 1, 256, dtype=torch.bfloat16, device=cuda)
    out, lse = ops.attention_selected(q.to(cuda), none, none, k_cache, k_cache, chosen, plan, 0.1, head_dim=256)
    assert out.shape == (0, 6, 256) and lse.shape == (0, 6)


def test_slopes_are_refused_by_name():
    """Arguments that pass every other check."""
    lib, a = _lib.load(), attn_args().attn
    a.block_table_stride = 4 * a.cache.num_kv_heads
    score = _lib.Score(0.0, 4096)
    assert lib.oscarop_attn_selected_v1(C.byref(a), C.byref(score), 4, None) == -22
    assert "alibi_slopes" in lib.oscar_last_error().decode()
    for scale in (0.0, -1.0, math.inf, math.nan):
        a.scale = scale
        assert lib.oscarop_attn_selected_v1(C.byref(a), None, 4, None) == -22
        assert "scale" in lib.oscar_last_error().decode()
    a.scale = 0.1
    a.workspace = None
    assert lib.oscarop_attn_selected_v1(C.byref(a), None, 4, None) == -22
    assert "workspace" in lib.oscar_last_error().decode()
    assert lib.oscarop_attn_selected_v1(None, None, 4, None) == -22
    assert "null args" in lib.oscar_last_error().decode()
