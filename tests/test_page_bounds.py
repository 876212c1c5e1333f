"""Bounds of pages (ops.page_bounds) where a request grew by more than the call was told: none of its
pages keeps what it held."""
import numpy as np
import pytest
import torch

from oracle import cases
from oscar_amd import ops
from test_page_select import SHAPES, plain_bounds


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("bs", [128, 32, 200])
@pytest.mark.parametrize("max_new", [0, 1, 300])
def test_growth_past_the_launch(cuda, max_new, bs, shape):
    hk, d = shape["hk"], shape["d"]
    old, new = [0, 3 * bs + 7, 0, bs, 5], [9 * bs + 1, 12 * bs, 1, bs, 7 * bs]
    c = cases.make_case(new, [1] * len(new), hk=hk, group=1, d=d, bs=bs, window=False)
    cache, table = torch.from_numpy(c["k8"]).view(torch.int8), torch.from_numpy(c["bt"].copy())
    table[1, 5] = -1  # a page that is passed over between others of the same workgroup
    before = torch.from_numpy(np.random.default_rng(2).standard_normal((cache.shape[0], hk, 2, d))).half()
    want = plain_bounds(before, c["k8"], table, old, new, bs, d)
    lengths, seq_lens = (torch.tensor(x, dtype=torch.int32, device=cuda) for x in (old, new))
    got = ops.page_bounds(cache.to(cuda), before.to(cuda), table.to(cuda), lengths, seq_lens, max_new=max_new, head_dim=d)
    assert torch.equal(got.cpu(), want) and not torch.equal(want, before)


@pytest.mark.gpu
def test_a_captured_call_replayed_with_longer_steps(cuda):
    """A step of one token captured, replayed for prompts: lengths are the device's."""
    c = cases.make_case([2000, 900], [1, 1], hk=2, group=1, d=128, window=False)
    cache, table = torch.from_numpy(c["k8"]).view(torch.int8).to(cuda), torch.from_numpy(c["bt"]).to(cuda)
    bounds = torch.zeros(cache.shape[0], 2, 2, 128, dtype=torch.float16, device=cuda)
    old, new = (torch.tensor(x, dtype=torch.int32, device=cuda) for x in ([1999, 899], [2000, 900]))
    call = lambda: ops.page_bounds(cache, bounds, table, old, new, max_new=1, head_dim=128)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for starts in ([0, 0], [1999, 450], [128, 127], [0, 899]):
        bounds.fill_(3.0)
        old.copy_(torch.tensor(starts, dtype=torch.int32))
        want = plain_bounds(bounds.cpu(), c["k8"], table.cpu(), starts, [2000, 900], 128, 128)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(bounds.cpu(), want), starts
