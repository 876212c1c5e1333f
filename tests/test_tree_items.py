"""Long items of a tree's attention: plans made for few workgroups, so that one item walks up to 120 full
tiles of a history, or its ragged end and several tiles of the chunk.  With a workgroup for each compute unit
small tests get one or two tiles an item.

Tolerances: test_tree_attention.py's; where scores are exact (test_a_tail_in_one_item) what is left is a
probability's rounding to fp16, 2^-11, and the fp32 sums of 16 terms of each of 188 tiles in numerator and
denominator, 2 * 3008 * 2^-24 = 3.6e-4."""
import math

import numpy as np
import pytest
import torch

from oscar_amd import _lib, ops
from test_tree_attention import bits, c_plan, check, expected, make, plain_masks, random_parents, tree_bits

KINDS = [(256, "bf16"), (256, "f16"), (128, "bf16"), (128, "f16")]


def plan_for(c, cuda, *, hk, group, d, target):
    """plan_tree's plan, but for `target` workgroups."""
    count, items, groups, sizes = c_plan(c["qsl"], c["seqs"], hk, group, d, target)
    assert count > 0
    nodes = np.diff(c["qsl"])
    parts = [torch.from_numpy(np.ascontiguousarray(x, np.int32).reshape(-1)).to(cuda) for x in (items, groups, c["qsl"], c["seqs"])]
    return items, ops.TreePlan(tuple(c["qsl"]), tuple(c["seqs"]), hk, group, d, sizes.num_items, sizes.num_groups, sizes.partial_rows,
                               sizes.partial_bytes, int(max(np.array(c["seqs"]) - nodes)), int(max(nodes)), c["qsl"][-1], *parts)


def attend(x, c, plan, mask, d, cap=0.0):
    return ops.attention_tree(x["q"], x["k"], x["v"], *x["caches"], x["table"], plan, mask, c["scale"], x["stage"], head_dim=d, soft_cap=cap)


@pytest.mark.gpu
@pytest.mark.parametrize("d,dtype", KINDS)
@pytest.mark.parametrize("busy", range(1, 9))
def test_long_items(cuda, busy, d, dtype):
    """1 to 120 full tiles in one item (the double buffers refilled, two tiles on their way, odd and even
    counts) with 1 to 8 waves that have rows, keys that grow along the history, so that the reference moves
    again and again, and window copies at both ends."""
    kt, nodes = 8192 // d, 4 * busy - 1
    counts = [1, 2, 3, 4, 5, 25, 120]
    hists = [kt * n + (7 * n) % kt for n in counts]
    shape = dict(hk=1, group=8, d=d, dtype=dtype)
    c, x = make(cuda, hists, [nodes] * len(hists), key_ramp=3.0, bs=96, **shape)
    items, plan = plan_for(c, cuda, hk=1, group=8, d=d, target=1)
    full = items[items[:, 7] < items[:, 4] // kt]
    assert sorted(full[:, 9].tolist()) == counts and (-(-items[:, 6] // 32) == busy).all()
    mask = tree_bits(np.random.default_rng(busy), [nodes] * len(hists))
    got = attend(x, c, plan, torch.from_numpy(mask).to(cuda), d)
    check(got, expected(c, x, hists, [nodes] * len(hists), mask, 1, d, dtype, 0.0), scores=30.0)


@pytest.mark.gpu
@pytest.mark.parametrize("d,dtype", KINDS)
@pytest.mark.parametrize("target", [1, 6, 8])
def test_few_workgroups(cuda, target, d, dtype):
    """Blocks of several requests and two KV heads dealt to few items, capped scores, ordinary keys."""
    hists, nodes = [3000, 70, 1025, 0], [40, 100, 1, 70]
    c, x = make(cuda, hists, nodes, hk=2, group=5, d=d, dtype=dtype)
    _, plan = plan_for(c, cuda, hk=2, group=5, d=d, target=target)
    mask = tree_bits(np.random.default_rng(target), nodes)
    got = attend(x, c, plan, torch.from_numpy(mask).to(cuda), d, 20.0)
    check(got, expected(c, x, hists, nodes, mask, 2, d, dtype, 20.0))


@pytest.mark.gpu
@pytest.mark.parametrize("d,dtype", KINDS)
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_slow_items_of_many_tiles(cuda, bad, d, dtype):
    """An item that holds a ragged end and all tiles of the chunk, with values that are not finite in tiles
    next to each other, in one tile twice, and in the last: the rows that see them alone, in their channels."""
    hists, nodes = [70 + 8192 // d, 0], [200, 130]
    shape = dict(hk=1, group=1, d=d, dtype=dtype)
    c, x = make(cuda, hists, nodes, **shape)
    items, plan = plan_for(c, cuda, hk=1, group=1, d=d, target=1)
    kt = 8192 // d
    slow = items[items[:, 7] >= items[:, 4] // kt]
    assert slow[:, 9].max() >= 1 + 200 // kt
    mask = tree_bits(np.random.default_rng(9), nodes)
    clean = expected(c, x, hists, nodes, mask, 1, d, dtype, 0.0)
    odd = [kt - 1, kt, kt + 3, 2 * kt, 3 * kt - 2, 199, 200 + 5, 200 + kt, 329]
    see = np.zeros((330, 330), bool)
    see[:200, :200], see[200:, 200:] = bits(mask[:200], 200), bits(mask[200:], 130)
    for i in odd:
        x["v"][i, :, 3::5] = bad
    out, lse = (t.cpu() for t in attend(x, c, plan, torch.from_numpy(mask).to(cuda), d))
    hit = torch.from_numpy(see[:, odd].any(1))
    assert hit.any() and (~hit).any()
    keep, rows = (~hit).nonzero().flatten(), hit.nonzero().flatten()
    check((out[keep], lse[keep]), (*(t[keep] for t in clean[:3]), clean[3]))
    channels = torch.zeros(d, dtype=torch.bool)
    channels[3::5] = True
    assert not out[rows][:, :, channels].isfinite().any()
    check((out[rows][:, :, ~channels], lse[rows]), (clean[0][rows][:, :, ~channels], clean[1][rows], clean[2][rows][:, :, ~channels], clean[3]))


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [dict(hk=1, group=6, d=256, dtype="bf16"), dict(hk=2, group=8, d=128, dtype="f16")], ids=["bf16", "f16"])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_keys_that_are_not_finite(cuda, bad, shape):
    """What a head of a row that sees such a key gets is what the formula gives: nothing finite where its
    score is +inf or NaN, the result without the key where it is -inf."""
    hists, nodes, d = [130, 0], [40, 70], shape["d"]
    c, x = make(cuda, hists, nodes, **shape)
    mask = tree_bits(np.random.default_rng(5), nodes)
    for i in (0, 11, 39, 40 + 35):
        x["k"][i, :, 5] = bad
    plan = ops.plan_tree(c["qsl"], c["seqs"], num_kv_heads=shape["hk"], group=shape["group"], head_dim=d, device=cuda)
    out, lse = (t.double().cpu() for t in attend(x, c, plan, torch.from_numpy(mask).to(cuda), d))
    # (the reference has a -inf score's p as exp(-inf) = 0, and a row with +inf or NaN as NaN, made zero there)
    want, want_lse, size, least = expected(c, x, hists, nodes, mask, shape["hk"], d, shape["dtype"], 0.0)
    lost = torch.isnan(want_lse) | (want_lse == math.inf)
    assert lost.any() and not lost.all()
    assert not out[lost].isfinite().any() and not lse[lost].isfinite().any()
    check((out[~lost], lse[~lost]), (want[~lost], want_lse[~lost], size[~lost], least))


@pytest.mark.gpu
@pytest.mark.parametrize("at", [0, 3001, 6015])
@pytest.mark.parametrize("d,dtype", KINDS)
def test_a_tail_in_one_item(cuda, d, dtype, at):
    """6015 keys whose probabilities are 2^-19 of one key's in the same item, first, in the middle or last,
    whose own value is zero: the output is the tail's, and keeps its bits."""
    hists, nodes = [6016], [2]
    c, x = make(cuda, hists, nodes, window=False, hk=1, group=6, d=d, dtype=dtype)
    g = np.random.default_rng(3)
    for name in "qkv":
        x[name].zero_()
    x["q"][:, :, 0] = d ** 0.5 if d == 256 else 8.0
    top = 13.125 / (c["scale"] * float(x["q"][0, 0, 0]))  # a score of 13.125 = 18.9 in log2
    # a slot's constants (K scale, K zero, V scale, V zero): every channel of a key 0 or `top`, of a value one number
    consts = c["k8"].reshape(-1, c["k8"].shape[-1])
    slot = np.asarray(c["bt"])[0, np.arange(6016) // 128].astype(np.int64) * 128 + np.arange(6016) % 128
    meta = np.zeros((6016, 4), np.float16)
    meta[at, 1] = top
    meta[:, 3] = 1 + g.random(6016)
    meta[at, 3] = 0
    consts[slot, :8] = meta.view(np.uint8)
    x["caches"][0].copy_(torch.from_numpy(c["k8"]).view(torch.int8))
    # the chunk's keys: a score of 0 and a value of 0, as far from the largest as the tail
    mask = np.array([[1], [3]], np.int64)
    items, plan = plan_for(c, cuda, hk=1, group=6, d=d, target=1)
    assert items[:, 9].max() == 6016 * d // 8192
    out, lse = (t.double().cpu() for t in attend(x, c, plan, torch.from_numpy(mask).to(cuda), d))
    want, want_lse, size, least = expected(c, x, hists, nodes, mask, 1, d, dtype, 0.0)
    assert (size > 0.01).all() and (lse - want_lse).abs().max() <= 4e-4
    assert ((out - want).abs() - (2.0 ** -11 + 2 * 3008 * 2.0 ** -24) * size - least).max() <= 0


@pytest.mark.gpu
def test_the_same_plan_gives_the_same_bits(cuda):
    """Repeated calls, whatever order workgroups run in."""
    hists, nodes = [9000, 300, 0], [40, 12, 64]
    c, x = make(cuda, hists, nodes)
    mask = torch.from_numpy(plain_masks(sum((random_parents(np.random.default_rng(4), n, "random") for n in nodes), []), c["qsl"], 64, c["qsl"][-1])[0]).to(cuda)
    for target in (3, 256):
        _, plan = plan_for(c, cuda, hk=1, group=6, d=256, target=target)
        want = [t.clone() for t in attend(x, c, plan, mask, 256)]
        for _ in range(5):
            assert all(torch.equal(a, b) for a, b in zip(attend(x, c, plan, mask, 256), want))


def test_records_are_plan_trees(monkeypatch):
    """The plans made here have what plan_tree makes for as many compute units."""
    c = dict(qsl=[0, 40, 41], seqs=[3040, 71])
    monkeypatch.setattr(ops, "cu_count", lambda device: 8)
    monkeypatch.setattr(ops, "upload", lambda parts, device: [torch.from_numpy(np.array(p)) for p in parts])
    plan = ops.plan_tree(c["qsl"], c["seqs"], num_kv_heads=2, group=5, head_dim=256, device="cpu")
    mine = plan_for(c, "cpu", hk=2, group=5, d=256, target=8)[1]
    assert plan.items.numel() == plan.num_items * _lib.TREE_ITEM_INTS
    for name in ("items", "groups", "qsl", "seqs"):
        assert torch.equal(getattr(plan, name), getattr(mine, name))
    for name in ("host_qsl", "host_seqs", "num_items", "num_groups", "partial_rows", "partial_bytes", "max_history", "max_nodes", "rows"):
        assert getattr(plan, name) == getattr(mine, name), name
