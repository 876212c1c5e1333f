"""Drafted trees (ops.tree_mask, plan_tree, attention_tree): refusals and the plan on the CPU,
masks and attention against plain evaluations on the GPU, the latter in 64 bits.

Tolerances.  Scores: products of 16-bit values are exact, their fp32 sum over d <= 256 terms
errs by at most d 2^-24 sum|q k| scale, below 3e-4 for standard normal rows (a key that the test makes
larger makes it larger: the tests that do so say by how much), a cap's tanh by cap 2^-22.  LSE: the
largest score error and the logarithm's rounding, 4e-4.  Outputs, of sum p |v|: a probability errs by
twice a score's error (numerator and sum), 8e-4, and by its rounding to fp16, half a step 2^-11; the values
of the history are fp16 as they are, the chunk's 16 bits as well, and probabilities against a bf16 chunk
have two bf16 parts (2^-16).  A probability is stored up to 2^15 with the row's largest at 2^7 at least,
so that an fp16 subnormal's rounding, 2^-25, is 2^-32 of it: for t keys t 2^-32 max|v|."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from oracle import cases
from oracle.attention import read_history
from oscar_amd import _lib, ops

LSE_TOL, REL_TOL = 4e-4, 2.0 ** -11 + 8e-4


# ------------------------------------------------------------------ the plan (host)
def c_plan(qsl, seqs, hk, group, d, target=256):
    lib, sizes, i32p = _lib.load(), _lib.TreeSizes(), C.POINTER(C.c_int32)
    qa, sa = (C.c_int32 * len(qsl))(*qsl), (C.c_int32 * max(len(seqs), 1))(*seqs)
    call = lambda items, n, groups, m: lib.oscarop_tree_plan_v1(qa, sa, len(seqs), hk, group, d, target, items, n, groups, m,  # noqa: E731
                                                                C.byref(sizes))
    rc = call(None, 0, None, 0)
    if rc < 0:
        return rc, None, None, sizes
    items = np.zeros((max(sizes.num_items, 1), _lib.TREE_ITEM_INTS), np.int32)
    groups = np.zeros((max(sizes.num_groups, 1), _lib.GROUP_INTS), np.int32)
    ip, gp = items.ctypes.data_as(i32p), groups.ctypes.data_as(i32p)
    if sizes.num_items:
        assert call(ip, sizes.num_items - 1, gp, sizes.num_groups) == -28
        assert call(ip, sizes.num_items, gp, sizes.num_groups - 1) == -28
    assert call(ip, sizes.num_items, gp, sizes.num_groups) == rc == sizes.num_items
    return rc, items[:sizes.num_items], groups[:sizes.num_groups], sizes


@pytest.mark.parametrize("d", [128, 256])
@pytest.mark.parametrize("target", [1, 256, 10000])
@pytest.mark.parametrize("hists,nodes,hk,group", [
    ([500], [16], 1, 6), ([24576] * 8, [32] * 8, 1, 6), ([0, 1, 31, 32, 33, 64, 700], [1, 64, 3, 0, 150, 2, 7], 2, 8),
    ([0], [1], 1, 1), ([40000, 5], [1000, 1], 1, 7), ([100], [3], 1, 100), ([], [], 1, 6),
])
def test_plan_deals_every_tile_once(hists, nodes, hk, group, target, d):
    """Each KV head's rows in blocks of at most 256, the tiles of each block (its history, and the
    chunk up to its last node) in one item each, the partials apart."""
    qsl = [0] + np.cumsum(nodes).tolist()
    rc, items, groups, sizes = c_plan(qsl, [h + n for h, n in zip(hists, nodes)], hk, group, d, target)
    assert rc == len(items)
    kt = 8192 // d
    taken = np.zeros(max(sizes.partial_rows, 1), int)
    by_block, rows = {}, {}
    for it in items:
        req, kvh, qa, n, hist, row0, count_rows, first, stride, count, part = it[:11].tolist()
        assert qa == qsl[req] and n == nodes[req] and hist == hists[req] and 0 < count_rows <= 256 and count >= 1
        taken[part:part + count_rows] += 1
        tiles = [first + stride * j for j in range(count)]
        assert all(t < hist // kt for t in tiles) or all(t >= hist // kt for t in tiles)
        by_block.setdefault((req, kvh, row0, count_rows), []).append((part, tiles))
        rows.setdefault((req, kvh), set()).add((row0, count_rows))
    assert taken[:sizes.partial_rows].max(initial=1) == 1 and taken.sum() == sizes.partial_rows
    for r, n in enumerate(nodes):
        for h in range(hk if n else 0):
            spans = sorted(rows[r, h])
            assert [a for a, _ in spans] == [sum(c for _, c in spans[:i]) for i in range(len(spans))]
            assert sum(c for _, c in spans) == n * group
            for a, c in spans:
                last = (a + c - 1) // group
                want = list(range(-(-hists[r] // kt) + last // kt + 1))
                assert sorted(sum((t for _, t in by_block[r, h, a, c]), [])) == want
    for kvh, qa, row0, count_rows, part, many, step, _ in groups.tolist():
        r = qsl.index(qa) if nodes[qsl.index(qa)] else max(i for i, a in enumerate(qsl[:-1]) if a == qa and nodes[i])
        assert sorted(p for p, _ in by_block[r, kvh, row0, count_rows]) == [part + i * step for i in range(many)]
    assert sizes.partial_bytes == sizes.partial_rows * (d + 1) * 4 and len(groups) == len(by_block)


@pytest.mark.parametrize("qsl,seqs,hk,group,d,message", [
    ([0, 4], [3], 1, 6, 256, "must cover"), ([0, 4], [9], 0, 6, 256, "invalid"), ([0, 4], [9], 1, 0, 256, "invalid"),
    ([0, 4], [9], 1, 6, 64, "head_dim"), ([0, 2 ** 24], [2 ** 24], 1, 6, 256, "too long"), ([-1, 3], [9], 1, 6, 256, "must cover"),
])
def test_plan_refusals(qsl, seqs, hk, group, d, message):
    assert c_plan(qsl, seqs, hk, group, d)[0] == -22
    assert message in _lib.load().oscar_last_error().decode()


# ------------------------------------------------------------------ refusals (no launch)
def attn_args(**changes):
    """Arguments that pass every check; the addresses are never read."""
    a = _lib.TreeAttnArgs(mask=4096, mask_words=1, partial_rows=64)
    x = a.attn
    for name in ("q", "k_new", "v_new", "block_table", "query_start_loc", "seq_lens", "items", "groups", "workspace", "out_rot", "lse"):
        setattr(x, name, 4096)
    x.num_tokens, x.num_q_heads, x.q_stride_token, x.kv_new_stride_token = 4, 6, 1536, 256
    x.cache = _lib.Cache(k=4096, v=4096, num_blocks=4, block_size=128, num_kv_heads=1, head_dim=256)
    x.cache.k_stride[:] = x.cache.v_stride[:] = [128 * 256, 256, 256]
    x.block_table_stride = x.block_table_cols = 4
    x.block_table_rows = x.num_reqs = 1
    x.num_items = x.num_groups = 1
    x.workspace_bytes, x.q_dtype, x.scale = 64 * 257 * 4, _lib.OSCAR_BF16, 0.1
    for name, value in changes.items():
        if name.startswith("cache_"):
            setattr(x.cache, name[6:], value)
        else:
            setattr(x if hasattr(x, name) else a, name, value)
    return a


@pytest.mark.parametrize("changes,message", [
    (dict(cache_head_dim=64), "head_dim 64"), (dict(q=None), "missing pointer"), (dict(k_new=None), "together"),
    (dict(k_new=None, v_new=None), "nodes' K and V"), (dict(mask=None), "mask"), (dict(mask=4100), "mask"), (dict(mask_words=0), "mask"),
    (dict(partial_rows=0), "workspace"), (dict(partial_rows=65), "workspace"), (dict(workspace=None), "workspace"),
    (dict(workspace=4104), "workspace"), (dict(phases=1), "phases"), (dict(q_dtype=0), "q_dtype"), (dict(block_table_rows=0), "rows"),
    (dict(cache_block_size=48), "block_size"), (dict(q=4098), "16-byte aligned"), (dict(num_q_heads=0x20000 * 3), "too many"),
])
def test_attention_refusals(changes, message):
    lib = _lib.load()
    a = attn_args(**changes)
    assert lib.oscarop_attn_tree_v1(C.byref(a), None, None) == -22
    assert message in lib.oscar_last_error().decode()


def test_attention_scores_refused():
    lib = _lib.load()
    for score, message in ((_lib.Score(0.0, 4096), "alibi_slopes"), (_lib.Score(1e9, None), "soft_cap")):
        assert lib.oscarop_attn_tree_v1(C.byref(attn_args()), C.byref(score), None) == -22
        assert message in lib.oscar_last_error().decode()
    assert lib.oscarop_attn_tree_v1(None, None, None) == -22
    assert lib.oscarop_attn_tree_v1(C.byref(attn_args(num_items=0)), None, None) == 0


@pytest.mark.parametrize("changes,message", [
    (dict(num_reqs=-1), "out of range"), (dict(num_reqs=65536), "out of range"), (dict(num_tokens=-1), "out of range"),
    (dict(max_nodes=0), "max_nodes"), (dict(max_nodes=1025, mask_words=17), "max_nodes"), (dict(mask_words=2), "max_nodes"),
    (dict(parents=None), "missing pointer"), (dict(query_start_loc=None), "missing pointer"), (dict(depths=None), "missing pointer"),
])
def test_mask_refusals(changes, message):
    lib = _lib.load()
    fixed = dict(parents=4096, query_start_loc=4096, num_reqs=1, max_nodes=64, num_tokens=4, mask=4096, mask_words=1, depths=4096)
    assert lib.oscarop_tree_mask_v1(C.byref(_lib.TreeArgs(**{**fixed, **changes})), None) == -22
    assert message in lib.oscar_last_error().decode()


# ------------------------------------------------------------------ masks
def plain_masks(parents, qsl, max_nodes, rows):
    words = -(-max_nodes // 64)
    mask, depths = np.zeros((rows, words), np.uint64), np.full(rows, -1, np.int32)
    for a, b in zip(qsl, qsl[1:]):
        if b - a > max_nodes:
            continue
        seen = []
        for i in range(b - a):
            p = parents[a + i]
            bad = p < -1 or p >= i or (p >= 0 and seen[p] is None)
            seen.append(None if bad else (set() if p < 0 else seen[p]) | {i})
            if not bad:
                for j in seen[i]:
                    mask[a + i, j // 64] |= np.uint64(1 << j % 64)
                depths[a + i] = len(seen[i]) - 1
    return mask.view(np.int64), depths


def random_parents(g, n, kind):
    if kind == "chain":
        return list(range(-1, n - 1))
    if kind == "star":
        return [-1] + [0] * (n - 1)
    p = [-1 if i == 0 or g.random() < 0.05 else int(i * g.random() ** 2) for i in range(n)]
    if kind == "broken":
        for i in g.integers(0, n, 3) if n else ():
            p[i] = int(g.choice([i, i + 3, -2, 2 ** 31 - 1, -2 ** 31]))
    return p


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["chain", "star", "random", "broken"])
@pytest.mark.parametrize("nodes,max_nodes", [([1], 1), ([16], 16), ([64, 1, 0, 63, 33], 64), ([65, 7, 128, 129], 128), ([1000, 1024, 3], 1024),
                                             ([200, 64], 150)])
def test_masks(cuda, nodes, max_nodes, kind):
    """Trees up to 1024 nodes deep, nodes without a proper parent, a request of too many nodes, rows
    of no request in front and behind."""
    g = np.random.default_rng(sum(nodes))
    qsl = [2] + (2 + np.cumsum(nodes)).tolist()
    parents = [5, 5] + sum((random_parents(g, n, kind) for n in nodes), []) + [0] * 70
    want, want_depths = plain_masks(parents, qsl, max_nodes, len(parents))
    mask, depths = ops.tree_mask(torch.tensor(parents, dtype=torch.int32, device=cuda),
                                 torch.tensor(qsl, dtype=torch.int32, device=cuda), max_nodes=max_nodes)
    assert np.array_equal(mask.cpu().numpy(), want) and np.array_equal(depths.cpu().numpy(), want_depths)


@pytest.mark.gpu
def test_mask_wrapper(cuda):
    qsl, p = torch.tensor([0, 3], dtype=torch.int32, device=cuda), torch.zeros(3, dtype=torch.int32, device=cuda)
    for bad in (dict(max_nodes=0), dict(max_nodes=1025)):
        with pytest.raises(ValueError, match="max_nodes"):
            ops.tree_mask(p, qsl, **bad)
    for a, b in ((p.long(), qsl), (p, qsl.long()), (p.view(1, 3), qsl), (p, qsl[:0])):
        with pytest.raises(ValueError, match="int32"):
            ops.tree_mask(a, b, max_nodes=4)
    mask, depths = ops.tree_mask(p[:0], qsl[:1], max_nodes=4)
    assert mask.shape == (0, 1) and depths.shape == (0,)
    # query starts past the rows: their rows have no bit
    mask, depths = ops.tree_mask(torch.tensor([-1, 0], dtype=torch.int32, device=cuda), qsl, max_nodes=4)
    assert mask.tolist() == [[0], [0]] and depths.tolist() == [-1, -1]


# ------------------------------------------------------------------ attention
def bits(mask, n):
    """[rows, n] truth values of mask words."""
    m = np.asarray(mask).view(np.uint64)
    return ((m[:, np.arange(n) // 64] >> (np.arange(n) % 64).astype(np.uint64)) & np.uint64(1)).astype(bool)


def reference(q, k, v, see, scale, cap):
    """64-bit attention of one request: q [n, hq, d], keys and values [t, hk, d], see [n, t].
    Returns out, lse, sum p |v|."""
    n, hq, d = q.shape
    hk = k.shape[1]
    q, k, v = (torch.as_tensor(np.asarray(x)).double() for x in (q, k, v))
    out, size = torch.zeros(n, hq, d, dtype=torch.float64), torch.zeros(n, hq, d, dtype=torch.float64)
    lse = torch.full((n, hq), -math.inf, dtype=torch.float64)
    see = torch.from_numpy(see)
    for h in range(hq):
        s = q[:, h] @ k[:, h * hk // hq].t() * scale
        if cap:
            s = cap * torch.tanh(s / cap)
        s = s.masked_fill(~see, -math.inf)
        lse[:, h] = torch.logsumexp(s, -1)
        p = torch.softmax(s, -1).nan_to_num(0.0)
        out[:, h], size[:, h] = p @ v[:, h * hk // hq], p @ v[:, h * hk // hq].abs()
    return out, lse, size


def make(cuda, hists, nodes, *, hk=1, group=6, d=256, dtype="bf16", bs=128, window=True, seed=1, **other):
    c = cases.make_case(hists, nodes, hk=hk, group=group, d=d, bs=bs, window=window, seed=seed, **other)
    t = torch.bfloat16 if dtype == "bf16" else torch.float16
    x = {name: torch.from_numpy(c[name]).to(t).to(cuda) for name in "qkv"}
    x["caches"] = [torch.from_numpy(c[name]).view(torch.int8).to(cuda) for name in ("k8", "v8")]
    x["stage"] = None if c["stage"] is None else tuple(torch.from_numpy(a).to(cuda) for a in c["stage"])
    x["table"] = torch.from_numpy(c["bt"]).to(cuda)
    return c, x


def expected(c, x, hists, nodes, mask, hk, d, dtype, cap):
    n, hq = x["q"].shape[:2]
    out, size = torch.zeros(n, hq, d, dtype=torch.float64), torch.zeros(n, hq, d, dtype=torch.float64)
    lse = torch.full((n, hq), -math.inf, dtype=torch.float64)
    most = 0.0
    for r, (h, m) in enumerate(zip(hists, nodes)):
        a, b = c["qsl"][r], c["qsl"][r + 1]
        if a == b:
            continue
        rounding = "bf16" if dtype == "bf16" else "f16"
        old_k = read_history(c["k8"], c["v8"], c["bt"][r], 0, h, hk, d, c["stage"], rounding)[0]
        old_v = read_history(c["k8"], c["v8"], c["bt"][r], 0, h, hk, d, c["stage"], "f16")[1]
        k = np.concatenate([old_k, x["k"][a:b].float().cpu().numpy()])
        v = np.concatenate([old_v, x["v"][a:b].float().cpu().numpy()])
        see = np.concatenate([np.ones((m, h), bool), bits(mask[a:b], m) & np.tri(m, dtype=bool)], 1)
        out[a:b], lse[a:b], size[a:b] = reference(x["q"][a:b].float().cpu().numpy(), k, v, see, c["scale"], cap)
        most = max(most, (h + m) * np.abs(v).max(initial=0))
    return out, lse, size, most * 2.0 ** -32


def check(got, want, scores=1.0):
    out, lse = (t.double().cpu() for t in got)
    want_out, want_lse, size, least = want
    seen = want_lse.isfinite()
    assert torch.equal(lse.isfinite(), seen) and (lse[~seen] == -math.inf).all() and (out[~seen] == 0).all()
    assert (lse - want_lse)[seen].abs().le(LSE_TOL * scores).all()
    excess = (out - want_out).abs() - ((2.0 ** -11 + 8e-4 * scores) * size + least)
    assert excess.max() <= 0, excess.max()


def run(x, c, mask, hists, nodes, cap=0.0, d=256, hk=1, group=6, **other):
    plan = ops.plan_tree(c["qsl"], c["seqs"], num_kv_heads=hk, group=group, head_dim=d, device=x["q"].device)
    return ops.attention_tree(x["q"], x["k"], x["v"], *x["caches"], x["table"], plan, mask, c["scale"], x["stage"], head_dim=d,
                              soft_cap=cap, **other)


def tree_bits(g, nodes, kind="random"):
    qsl = [0] + np.cumsum(nodes).tolist()
    parents = sum((random_parents(g, n, kind) for n in nodes), [])
    return plain_masks(parents, qsl, max(max(nodes), 1), qsl[-1])[0]


SHAPES = [dict(hk=1, group=6, d=256, dtype="bf16"), dict(hk=2, group=8, d=128, dtype="f16"), dict(hk=2, group=5, d=256, dtype="f16"),
          dict(hk=1, group=8, d=128, dtype="bf16"), dict(hk=3, group=1, d=128, dtype="bf16")]


@pytest.mark.gpu
@pytest.mark.parametrize("cap", [0.0, 20.0])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(str(v) for v in s.values()))
@pytest.mark.parametrize("hists,nodes,bs", [([500], [16], 128), ([0, 1, 31, 32], [1, 9, 64, 33], 32), ([63, 64, 65, 700], [7, 65, 0, 2], 64),
                                            ([3000, 129], [40, 150], 128), ([257], [1], 96)])
def test_attention(cuda, hists, nodes, bs, shape, cap):
    """Fresh requests, histories at the borders of tiles and pages, one node and more than a
    workgroup's rows, a request without nodes; the FP32 window in all."""
    c, x = make(cuda, hists, nodes, bs=bs, **shape)
    mask = tree_bits(np.random.default_rng(3), nodes)
    got = run(x, c, torch.from_numpy(mask).to(cuda), hists, nodes, cap, shape["d"], shape["hk"], shape["group"])
    check(got, expected(c, x, hists, nodes, mask, shape["hk"], shape["d"], shape["dtype"], cap))


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES[:2], ids=["bf16", "f16"])
@pytest.mark.parametrize("window", [False, True])
def test_any_mask(cuda, shape, window):
    """Bits at random, a row's own among them or not, rows without a bit (with no history: zeros and
    -inf), bits of later rows, which count for nothing, and words to spare."""
    hists, nodes = [0, 300, 0, 40], [70, 33, 5, 1]
    c, x = make(cuda, hists, nodes, window=window, **shape)
    g = np.random.default_rng(8)
    mask = g.integers(-2 ** 63, 2 ** 63 - 1, (sum(nodes), 3))
    mask[[0, 4, 70, 80, 103, 107]] = 0
    got = run(x, c, torch.from_numpy(mask).to(cuda), hists, nodes, 0.0, shape["d"], shape["hk"], shape["group"])
    want = expected(c, x, hists, nodes, mask, shape["hk"], shape["d"], shape["dtype"], 0.0)
    assert not want[1][0].isfinite().any() and not want[1][103].isfinite().any()
    check(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES[:2], ids=["bf16", "f16"])
def test_rising_scores_and_large_values(cuda, shape):
    """The reference moves many times along a history whose keys grow up to 30 times (and their scores'
    sums with them); values up to 2e4."""
    hists, nodes = [9000], [24]
    c, x = make(cuda, hists, nodes, key_ramp=3.0, v_gain=3e3, **shape)
    mask = tree_bits(np.random.default_rng(5), nodes)
    got = run(x, c, torch.from_numpy(mask).to(cuda), hists, nodes, 0.0, shape["d"], shape["hk"], shape["group"])
    check(got, expected(c, x, hists, nodes, mask, shape["hk"], shape["d"], shape["dtype"], 0.0), scores=30.0)


@pytest.mark.gpu
def test_a_long_tail(cuda):
    """A first node far above 6000 keys of equal score, whose probabilities are 2^-19 of its own and
    a fiftieth of the sum: they keep their 11 bits."""
    hists, nodes, d = [6016], [2], 256
    c, x = make(cuda, hists, nodes, window=False)
    x["q"].zero_()
    x["k"].zero_()
    x["q"][:, :, 0] = 16.0
    x["k"][0, :, 0] = 13.125  # a score of 13.125 = 18.9 in log2; the history's: k[..., 0] = 0
    k8 = c["k8"].reshape(-1, c["k8"].shape[-1])
    k8[:, :4] = 0  # scale and zero of K: all keys zero
    x["caches"][0].view(torch.uint8).view(-1, c["k8"].shape[-1])[:, :4] = 0
    mask = np.array([[1], [3]], np.int64)
    got = run(x, c, torch.from_numpy(mask).to(cuda), hists, nodes)
    check(got, expected(c, x, hists, nodes, mask, 1, d, "bf16", 0.0))


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES[:2], ids=["bf16", "f16"])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_values_that_are_not_finite(cuda, shape, bad):
    """Keys and values of nodes that a row does not see may hold anything; the rows that see them
    get what the formula gives."""
    hists, nodes, d = [130, 0], [40, 70], shape["d"]
    c, x = make(cuda, hists, nodes, **shape)
    mask = tree_bits(np.random.default_rng(5), nodes)
    clean = expected(c, x, hists, nodes, mask, shape["hk"], d, shape["dtype"], 0.0)
    see = np.concatenate([bits(mask[:40], 110), np.zeros((70, 110), bool)])
    see[40:, 40:] = bits(mask[40:], 70)
    odd_v, odd_k = [7, 39, 40 + 33, 40 + 66], [11, 40 + 35]
    for i in odd_v:
        x["v"][i, :, 3::5] = bad
    for i in odd_k:
        x["k"][i, :, 5] = bad
    out, lse = run(x, c, torch.from_numpy(mask).to(cuda), hists, nodes, 0.0, d, shape["hk"], shape["group"])
    hit_k, hit_v = torch.from_numpy(see[:, odd_k].any(1)), torch.from_numpy(see[:, odd_v].any(1))
    assert hit_k.any() and hit_v.any() and (~hit_k & ~hit_v).any()
    keep = (~hit_k & ~hit_v).nonzero().flatten()
    check((out.cpu()[keep], lse.cpu()[keep]), (*(t[keep] for t in clean[:3]), clean[3]))
    # a value's channels alone in the rows that see it, and nothing else of them
    rows = (~hit_k & hit_v).nonzero().flatten()
    got, channels = out.double().cpu()[rows], torch.zeros(d, dtype=torch.bool)
    channels[3::5] = True
    assert not got[:, :, channels].isfinite().any()
    check((got[:, :, ~channels], lse.cpu()[rows]), (clean[0][rows][:, :, ~channels], clean[1][rows], clean[2][rows][:, :, ~channels], clean[3]))
    # a key's score is NaN or infinite: with infinity other rows may still be finite (-inf: the key drops out)
    assert torch.isnan(lse.cpu()[hit_k]).any() or not math.isnan(bad)


@pytest.mark.gpu
def test_strides_outputs_streams_and_padding(cuda):
    """Rows of a fused projection, a wider table and mask, outputs given, another stream, rows of no
    request in front and behind: the same bits as the plain call."""
    hists, nodes = [300, 800], [9, 20]
    c, x = make(cuda, hists, nodes)
    mask = torch.from_numpy(tree_bits(np.random.default_rng(5), nodes)).to(cuda)
    want = run(x, c, mask, hists, nodes)
    n = 29
    fused = torch.randn(n, 8 * 256, device=cuda).bfloat16()
    fused[:, :6 * 256] = x["q"].view(n, -1)
    fused[:, 6 * 256:7 * 256] = x["k"].view(n, -1)
    fused[:, 7 * 256:] = x["v"].view(n, -1)
    y = dict(x, q=fused[:, :6 * 256].view(n, 6, 256), k=fused[:, 6 * 256:7 * 256].view(n, 1, 256), v=fused[:, 7 * 256:].view(n, 1, 256))
    wide = torch.zeros(2, 40, dtype=torch.int32, device=cuda)
    wide[:, 3:3 + x["table"].shape[1]] = x["table"]
    y["table"] = wide[:, 3:3 + x["table"].shape[1]]
    more = torch.cat([mask, torch.full_like(mask, -1)], 1)[:, :1]
    given = dict(out_rot=torch.full((n, 6, 256), 7.0, device=cuda), lse=torch.full((n, 6), 7.0, device=cuda))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = run(y, c, more, hists, nodes, **given)
    stream.synchronize()
    assert got[0] is given["out_rot"] and all(torch.equal(a, b) for a, b in zip(got, want))
    # padding: two rows in front, five behind
    pad = lambda t: torch.cat([t.new_zeros(2, *t.shape[1:]), t, t.new_zeros(5, *t.shape[1:])])  # noqa: E731
    z = dict(x, q=pad(x["q"]), k=pad(x["k"]), v=pad(x["v"]))
    padded = dict(c, qsl=[a + 2 for a in c["qsl"]])
    out, lse = run(z, padded, pad(mask), hists, nodes)
    assert torch.equal(out[2:31], want[0]) and torch.equal(lse[2:31], want[1])
    assert not out[:2].any() and not out[31:].any() and (lse[:2] == -math.inf).all() and (lse[31:] == -math.inf).all()


@pytest.mark.gpu
def test_wrapper_refusals(cuda):
    hists, nodes = [300, 800], [9, 70]
    c, x = make(cuda, hists, nodes)
    mask = torch.from_numpy(tree_bits(np.random.default_rng(5), nodes)).to(cuda)
    plan = ops.plan_tree(c["qsl"], c["seqs"], num_kv_heads=1, group=6, head_dim=256, device=cuda)

    def call(q=x["q"], k=x["k"], v=x["v"], caches=x["caches"], table=x["table"], plan=plan, mask=mask, d=256, **other):
        return ops.attention_tree(q, k, v, *caches, table, plan, mask, c["scale"], x["stage"], head_dim=d, **other)

    narrow = ops.plan_tree(c["qsl"], c["seqs"], num_kv_heads=1, group=3, head_dim=256, device=cuda)
    for bad, message in ((dict(q=x["q"].float()), "bf16 or fp16"), (dict(k=x["k"].half()), "Current K/V"), (dict(k=None), "nodes' K and V"),
                         (dict(v=x["v"][:5]), "Current K/V"), (dict(mask=mask.int()), "mask"), (dict(mask=mask[:5]), "mask"),
                         (dict(mask=mask[:, :1]), "words"), (dict(table=x["table"][:1]), "rows"), (dict(table=x["table"][:, :3]), "cover"),
                         (dict(plan=narrow), "plan is for"), (dict(q=x["q"][:70], k=x["k"][:70], v=x["v"][:70], mask=mask[:70]), "more queries"),
                         (dict(soft_cap=-1.0), "soft_cap"), (dict(out_rot=torch.zeros(79, 6, 256, device=cuda).half()), "out_rot"),
                         (dict(lse=torch.zeros(79, 5, device=cuda)), "lse"), (dict(d=128), "head_dim"),
                         (dict(caches=[x["caches"][0], x["caches"][1][:1]]), "same blocks")):
        with pytest.raises(ValueError, match=message):
            call(**bad)
    with pytest.raises(RuntimeError, match="device tensors"):
        call(mask=mask.cpu())
    with pytest.raises(ValueError, match="cover its query chunk"):
        ops.plan_tree([0, 5], [4], num_kv_heads=1, group=6, head_dim=256, device=cuda)


@pytest.mark.gpu
def test_captured_calls(cuda):
    """Two graphs of the same plan replayed in turn on two streams, with eager calls and changed inputs
    between: every replay gives the eager call's bits."""
    hists, nodes = [2500, 300], [30, 12]
    c, x = make(cuda, hists, nodes)
    parents = torch.tensor(sum((random_parents(np.random.default_rng(4), n, "random") for n in nodes), []), dtype=torch.int32, device=cuda)
    plan = ops.plan_tree(c["qsl"], c["seqs"], num_kv_heads=1, group=6, head_dim=256, device=cuda)

    def call(y):
        mask, _ = ops.tree_mask(parents, plan.qsl, max_nodes=30)
        return ops.attention_tree(y["q"], y["k"], y["v"], *x["caches"], x["table"], plan, mask, c["scale"], x["stage"], head_dim=256)

    inputs = [{k: torch.randn_like(x[k]) for k in "qkv"} for _ in range(2)]
    call(inputs[0])
    torch.cuda.synchronize()
    graphs = []
    for y in inputs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = call(y)
        graphs.append((g, out))
    streams = [torch.cuda.Stream() for _ in graphs]
    for turn in range(4):
        for y in inputs:
            for t in y.values():
                t.copy_(torch.randn_like(t))
        want = [tuple(t.clone() for t in call(y)) for y in inputs]
        torch.cuda.synchronize()
        for s, (g, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for (_, out), w in zip(graphs, want):
            assert all(torch.equal(a, b) for a, b in zip(out, w)), turn


@pytest.mark.gpu
def test_pages_past_four_gigabytes(cuda):
    """The same pages at the front of a small cache and at the end of one of 4.3 GB a side: the same
    bits."""
    hists, nodes = [1500, 700], [20, 5]
    c, x = make(cuda, hists, nodes, window=False)
    mask = torch.from_numpy(tree_bits(np.random.default_rng(5), nodes)).to(cuda)
    want = run(x, c, mask, hists, nodes)
    small = x["caches"]
    pages, blocks = small[0].shape[0], (1 << 32) // small[0][0].numel() + 1000
    large = [torch.empty(blocks, *t.shape[1:], dtype=torch.int8, device=cuda) for t in small]
    for a, b in zip(large, small):
        a[blocks - pages:] = b
    got = run(dict(x, caches=large, table=x["table"] + (blocks - pages)), c, mask, hists, nodes)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_bad_tables_and_records(cuda):
    """Page ids outside the cache read page 0 (no fault); a record that breaks the plan's rules makes
    its rows NaN and leaves the others."""
    hists, nodes = [600, 600], [5, 5]
    c, x = make(cuda, hists, nodes)
    mask = torch.from_numpy(tree_bits(np.random.default_rng(5), nodes)).to(cuda)
    want = run(x, c, mask, hists, nodes)
    bad = x["table"].clone()
    bad[1, :2] = torch.tensor([-7, 2 ** 31 - 1], device=cuda)
    out, _ = run(dict(x, table=bad), c, mask, hists, nodes)
    assert torch.equal(out[:5], want[0][:5]) and out.isfinite().all()
    plan = ops.plan_tree(c["qsl"], c["seqs"], num_kv_heads=1, group=6, head_dim=256, device=cuda)
    items = plan.items.view(-1, _lib.TREE_ITEM_INTS)
    second = (items[:, 0] == 1).nonzero().flatten()[0]
    for field, value in ((0, 99), (1, 3), (2, 1 << 20), (4, -5), (7, 1 << 28), (9, 100000)):
        saved = items[second, field].clone()
        items[second, field] = value
        out, lse = ops.attention_tree(x["q"], x["k"], x["v"], *x["caches"], x["table"], plan, mask, c["scale"], x["stage"], head_dim=256)
        assert torch.equal(out[:5], want[0][:5]) and torch.isnan(out[5:]).all() and torch.isnan(lse[5:]).all(), field
        items[second, field] = saved
