"""The order of pages' scores where 64 bits do not hold their sums exactly: bounds and queries over the
whole range of their types.

A score is off by the rounding of at most 21 additions (D 256: 8 terms of a lane in each of 4 sums,
two products a term, 2 additions of the sums and 3 of the lanes), each 2^-53 of a partial sum, which
the sum of the terms' sizes bounds: 21 2^-53 sum_d (|q m| + |q| w).  The reference's sums are exact (math.fsum
rounds once: one more).  A page may be chosen before another if its exact score is no less than the
other's by more than both errors."""
import math

import pytest
import torch

from oscar_amd import ops
from test_page_select import KINDS, SHAPES

STEPS = 22 * 2.0 ** -53


def wide(g, *shape, low, high):
    """Either sign, magnitudes from 2^low to 2^high."""
    x = torch.exp2(torch.rand(*shape, generator=g, dtype=torch.float64) * (high - low) + low)
    return torch.where(torch.rand(*shape, generator=g) < 0.5, -x, x)


def exact_scores(q, bounds):
    """Scores [pages] and their errors' bound; q [rows, d], bounds [pages, 2, d]."""
    q, b = q.double(), bounds.double()
    m, w = (b[:, 1] + b[:, 0]) / 2, (b[:, 1] - b[:, 0]) / 2
    scores, errors = [], []
    for p in range(len(b)):
        sums = [(math.fsum((row * m[p]).tolist() + (row.abs() * w[p]).tolist()),
                 STEPS * float((row * m[p]).abs().sum() + (row.abs() * w[p]).sum())) for row in q]
        scores.append(max(s for s, _ in sums))
        errors.append(max(e for _, e in sums))
    return scores, errors


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("near", [False, True])
def test_values_of_any_range(cuda, near, shape, dtype):
    """Terms up to 2^60 apart; near: every page's bounds those of one page but for one small channel, so that
    the scores differ in their last bits or not at all."""
    g = torch.Generator().manual_seed(11)
    hk, group, d, n, budget = shape["hk"], shape["group"], shape["d"], 70, 20
    x = wide(g, n, hk, 2, d, low=-24, high=15).half()
    if near:
        x = x[:1].repeat(n, 1, 1, 1)
        x[:, :, :, 9] = (torch.randint(0, 6, (n, 1, 1), generator=g) * 2.0 ** -24).half()
    bounds = torch.stack([x.amin(2), x.amax(2)], 2)
    q = wide(g, 1, hk * group, d, low=-20, high=10).to(KINDS[dtype])
    table = torch.randperm(n, generator=g).to(torch.int32)[None]
    plan = ops.plan_selected([0, 1], [n * 128 + 1], has_new=True, block_size=128, budget=budget, num_kv_heads=hk, group=group, head_dim=d, device=cuda)
    _, pages = ops.select_pages(q.to(cuda), bounds.to(cuda), table.to(cuda), plan)
    apart = 0
    for h in range(hk):
        scores, errors = exact_scores(q[0, h * group:(h + 1) * group], bounds[table[0].long(), h])
        chosen = pages[0, h].tolist()
        assert chosen[0] == 0 and chosen[-1] == n - 1 and chosen == sorted(set(chosen)) and len(chosen) == budget
        left = [p for p in range(1, n - 1) if p not in chosen]
        for p in chosen[1:-1]:
            for o in left:
                assert scores[p] >= scores[o] - errors[p] - errors[o], (p, o)
                apart += abs(scores[p] - scores[o]) > errors[p] + errors[o]
    assert near or apart > 0


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("n", [60, 9000])
def test_equal_bounds_tie(cuda, n, shape):
    """Pages of equal bounds have equal scores to the last bit, in a few workgroups and in many: the
    earlier ones are chosen."""
    g = torch.Generator().manual_seed(12)
    hk, group, d, budget = shape["hk"], shape["group"], shape["d"], 12
    x = wide(g, 1, hk, 2, d, low=-24, high=15).half().expand(n, -1, -1, -1)
    bounds = torch.stack([x.amin(2), x.amax(2)], 2)
    q = wide(g, 3, hk * group, d, low=-20, high=10).bfloat16()
    table = torch.randperm(n, generator=g).to(torch.int32)[None]
    plan = ops.plan_selected([0, 3], [n * 128 + 3], has_new=True, block_size=128, budget=budget, last_pages=2, num_kv_heads=hk, group=group,
                             head_dim=d, device=cuda)
    _, pages = ops.select_pages(q.to(cuda), bounds.to(cuda), table.to(cuda), plan)
    assert pages[0].tolist() == [list(range(budget - 2)) + [n - 2, n - 1]] * hk
