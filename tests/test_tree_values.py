"""Values of a tree's nodes at the ends of their type's range: outputs are means of them, and as finite.
Tolerances: test_tree_attention.py's."""
import numpy as np
import pytest
import torch

from test_tree_attention import SHAPES, check, expected, make, run, tree_bits

LARGEST = {"bf16": torch.finfo(torch.bfloat16).max, "f16": torch.finfo(torch.float16).max}


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(str(v) for v in s.values()))
@pytest.mark.parametrize("scores", ["equal", "random", "rising"])
@pytest.mark.parametrize("signs", ["one", "both"])
def test_largest_values(cuda, signs, scores, shape):
    """Chunks of one node and of several items, without a history, behind a ragged end, and behind full
    tiles: every value the largest of its type, of one sign (the sums' worst case) or of both."""
    hists, nodes, d, dtype = [0, 0, 45, 2000, 64], [1, 300, 70, 33, 9], shape["d"], shape["dtype"]
    c, x = make(cuda, hists, nodes, **shape)
    g = np.random.default_rng(12)
    mask = tree_bits(g, nodes, "chain")
    x["v"].fill_(LARGEST[dtype])
    if signs == "both":
        x["v"][torch.from_numpy(g.random(x["v"].shape) < 0.5).to(cuda)] *= -1
    if scores == "equal":
        x["q"].zero_()
    elif scores == "rising":  # up to 2 times as large: with them the scores' sums
        x["k"].mul_(torch.linspace(0.1, 2.0, len(x["k"]), device=cuda)[:, None, None].to(x["k"].dtype))
    got = run(x, c, torch.from_numpy(mask).to(cuda), hists, nodes, 0.0, d, shape["hk"], shape["group"])
    assert got[0].isfinite().all()
    with np.errstate(over="ignore"):
        *want, least = expected(c, x, hists, nodes, mask, shape["hk"], d, dtype, 0.0)
    # (a subnormal probability's rounding is nothing beside a row's own bf16 value)
    check(got, (*want, least if dtype == "f16" else 0.0), scores=2.0)


@pytest.mark.gpu
@pytest.mark.parametrize("factor", [2.0 ** -100, 2.0 ** 100])
def test_small_and_large_values(cuda, factor):
    """bf16 values of a chunk without a history, times a power of two: the outputs times that power, to
    fp32's last bits."""
    hists, nodes, d = [0, 0], [90, 7], 256
    c, x = make(cuda, hists, nodes)
    mask = torch.from_numpy(tree_bits(np.random.default_rng(4), nodes)).to(cuda)
    want, want_lse = run(x, c, mask, hists, nodes)
    out, lse = run(dict(x, v=x["v"] * factor), c, mask, hists, nodes)
    assert torch.equal(lse, want_lse)
    assert ((out.double() / factor - want.double()).abs() <= 2.0 ** -20 * want.double().abs()).all()
