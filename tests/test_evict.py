"""Eviction by accumulated weight (ops.plan_evict, ops.evict): refusals and the plan on the
CPU, every byte against a plain evaluation on the GPU.  Nothing is computed, so nothing is
within a tolerance: slot bytes, weights and tags are equal."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from oscar_amd import _lib


# ------------------------------------------------------------------ refusals (no launch)
def args(**changes):
    """Arguments that pass every check; the addresses are never read."""
    a = _lib.EvictArgs()
    cache = _lib.Cache(k=1 << 20, v=1 << 20, num_blocks=4, block_size=128, num_kv_heads=2, head_dim=256)
    cache.k_stride[:] = cache.v_stride[:] = [128 * 512, 512, 256]
    fixed = dict(weights=1 << 12, weights_stride_request=600, weights_stride_head=300, weights_cols=300, weights_out=1 << 16,
                 out_stride_request=600, out_stride_head=300, cache=cache, block_table=1 << 20, block_table_stride=4,
                 block_table_rows=2, block_table_cols=4, requests=1 << 20, num_reqs=2, max_drop=128, workspace=1 << 20,
                 workspace_bytes=1 << 20)
    for name, value in {**fixed, **changes}.items():
        if name.startswith("cache_"):
            setattr(a.cache, name[6:], value)
        else:
            setattr(a, name, value)
    return a


@pytest.mark.parametrize("changes,message", [
    (dict(cache_head_dim=64), "head_dim 64 unsupported"),
    (dict(num_reqs=-1), "negative size"),
    (dict(max_drop=-128), "negative size"),
    (dict(weights=None), "missing pointer"),
    (dict(requests=None), "missing pointer"),
    (dict(cache_v=None), "missing pointer"),
    (dict(weights_cols=0), "out of range"),
    (dict(cache_num_kv_heads=0), "out of range"),
    (dict(max_drop=100), "whole pages"),
    (dict(block_table_rows=1), "block-table rows"),
    (dict(cache_k=(1 << 20) + 2), "16-byte aligned"),
    (dict(weights_stride_head=200), "overlap"),
    (dict(out_stride_request=500), "overlap"),
    (dict(weights_out=(1 << 12) + 4796), "weights_out overlaps"),
    (dict(weights_out=1 << 12), "weights_out overlaps"),
    (dict(workspace=None), "workspace"),
    (dict(workspace_bytes=100), "workspace"),
    (dict(workspace=(1 << 20) + 8), "workspace"),
])
def test_refusals(changes, message):
    lib = _lib.load()
    assert lib.oscarop_evict_v1(C.byref(args(**changes)), None) == -22
    assert message in lib.oscar_last_error().decode()


def test_workspace_and_empty_calls():
    lib = _lib.load()
    assert lib.oscarop_evict_v1(None, None) == -22
    assert lib.oscarop_evict_v1(C.byref(args(num_reqs=0)), None) == 0
    assert lib.oscarop_evict_workspace_bytes_v1(-1, 1, 1) == lib.oscarop_evict_workspace_bytes_v1(1, 0, 1) == -22
    assert lib.oscarop_evict_workspace_bytes_v1(2, 2, 128) >= 2 * 2 * 2 * 128 * 4
    stage = _lib.Staging(owner=None, rows=3)
    assert lib.oscarop_evict_v1(C.byref(args(staging=C.pointer(stage))), None) == -22


@pytest.mark.parametrize("seed", range(20))
def test_overlaps_are_told_from_strides(seed):
    """Small layouts against an enumeration of their elements: rows that share one are refused,
    rows of either axis within the other are not, and two lists of the same such layout overlap
    where they share one and nowhere else (the call then stops at the missing workspace)."""
    g, lib, said = np.random.default_rng(seed), _lib.load(), {"heads or requests overlap": 0, "weights_out overlaps": 0, "workspace": 0}
    for _ in range(200):
        cols, reqs, hk = (int(g.integers(1, n)) for n in (6, 4, 4))
        request, head = (int(x) for x in g.integers(0, 24, 2))
        if g.random() < 0.8:  # one axis within the other
            inner = cols + int(g.integers(0, 9))
            count, outermost = (hk, "request") if g.random() < 0.5 else (reqs, "head")
            outer = (count - 1) * inner + cols + int(g.integers(0, 9))
            request, head = (outer, inner) if outermost == "request" else (inner, outer)
            nested = True
        else:
            nested = False
        by = int(g.integers(-60, 60))
        elements = [r * request + h * head + c for r in range(reqs) for h in range(hk) for c in range(cols)]
        x = args(weights=1 << 12, weights_out=(1 << 12) + 4 * by, weights_stride_request=request, weights_stride_head=head,
                 out_stride_request=request, out_stride_head=head, weights_cols=cols, num_reqs=reqs, cache_num_kv_heads=hk,
                 block_table_rows=reqs, workspace=None)
        assert lib.oscarop_evict_v1(C.byref(x), None) == -22
        got = [m for m in said if m in lib.oscar_last_error().decode()]
        if len(set(elements)) < len(elements):
            want = "heads or requests overlap"
        elif {e + by for e in elements} & set(elements):
            want = "weights_out overlaps"
        else:
            want = "workspace"
        assert got == [want] or not nested and got == ["heads or requests overlap"], (cols, reqs, hk, request, head, by, got, want)
        said[got[0]] += 1
    assert min(said.values()) > 0, said


@pytest.mark.parametrize("sizes", [(1, 1, 1 << 61), (1, 1, 1 << 62), (1, 1, 1 << 30), (0xffff, 0xffff, 1 << 29), (1 << 40, 1, 128),
                                   (1, 1 << 40, 128)])
def test_sizes_that_overflow_are_refused(sizes):
    """2 max_drop + 1 entries a list wrapped around to a few bytes, which a workspace then had."""
    lib = _lib.load()
    assert lib.oscarop_evict_workspace_bytes_v1(*sizes) == -22
    reqs, heads, drop = sizes
    if reqs < 1 << 31:
        a = args(num_reqs=reqs, cache_num_kv_heads=heads, max_drop=drop, block_table_rows=reqs, workspace_bytes=1 << 62,
                 weights_stride_head=1 << 9, weights_stride_request=1 << 26, out_stride_head=1 << 9, out_stride_request=1 << 26,
                 weights_out=1 << 56)
        assert lib.oscarop_evict_v1(C.byref(a), None) == -22
        assert "sizes out of range" in lib.oscar_last_error().decode()


def test_the_largest_sizes_have_a_workspace():
    drop = (1 << 30) - 128
    assert _lib.load().oscarop_evict_workspace_bytes_v1(1, 8, drop) == 8 * 4 * (2 * drop + 1)


def plan_on_the_cpu(monkeypatch, *a, **kw):
    from oscar_amd import ops

    monkeypatch.setattr(ops, "upload", lambda parts, device: [torch.from_numpy(np.ascontiguousarray(p)) for p in parts])
    return ops.plan_evict(*a, device="cpu", **kw)


def test_plan(monkeypatch):
    plan = plan_on_the_cpu(monkeypatch, [1500, 10, 0, 1000], [4, 0, 0, 6], block_size=128, sink_tokens=100, recent_tokens=0)
    assert plan.seq_lens == [1500 - 512, 10, 0, 1000 - 768] and plan.max_drop == 768
    assert plan.requests.tolist() == [[1500, 100, 1408, 512], [10, 0, 0, 0], [0, 0, 0, 0], [1000, 100, 896, 768]]
    table = torch.arange(48, dtype=torch.int32).view(4, 12)
    new = plan.table(table)
    assert new[0].tolist() == list(range(7)) + [11] + [7, 8, 9, 10] and plan.freed[0] == (8, 12)
    assert torch.equal(new[1:3], table[1:3]) and plan.freed[1] == (1, 1) and plan.freed[2] == (0, 0)


def test_plan_of_a_whole_middle(monkeypatch):
    plan = plan_on_the_cpu(monkeypatch, [1000], [6], block_size=128, sink_tokens=128, recent_tokens=100)
    assert plan.seq_lens == [232] and plan.requests.tolist() == [[1000, 128, 896, 768]]
    assert plan.table(torch.arange(8)[None])[0].tolist() == [0, 7, 1, 2, 3, 4, 5, 6]


def test_tables_that_do_not_hold_the_requests_are_refused(monkeypatch):
    plan = plan_on_the_cpu(monkeypatch, [1000, 300], [6, 0], block_size=128)
    for bad in (torch.zeros(2, 7, dtype=torch.int32), torch.zeros(1, 9, dtype=torch.int32), torch.zeros(16, dtype=torch.int32)):
        with pytest.raises(ValueError, match="(?i)block.table"):
            plan.table(bad)
    assert plan.table(torch.zeros(2, 8, dtype=torch.int32)).shape == (2, 8)


@pytest.mark.parametrize("lengths,pages,more", [
    ([1000], [7], dict(sink_tokens=128, recent_tokens=100)),
    ([1000], [7], dict(sink_tokens=1)),
    ([1000], [8], {}),
    ([100], [1], {}),
    ([1000], [-1], {}),
    ([-1], [0], {}),
    ([1000], [1, 1], {}),
    ([1000], [1], dict(sink_tokens=-1)),
    ([1000], [1], dict(block_size=0)),
])
def test_plan_refusals(monkeypatch, lengths, pages, more):
    with pytest.raises(ValueError):
        plan_on_the_cpu(monkeypatch, lengths, pages, **{"block_size": 128, **more})


# ------------------------------------------------------------------ values
def reference(x, lengths, pages, sink, recent, d):
    """The caches, weights and tags after the call, entry by entry (NumPy)."""
    k, v, w, owner, table = (x[n].copy() for n in ("k", "v", "w", "owner", "table"))
    bs, hk = k.shape[1], k.shape[2]
    for r, (length, many) in enumerate(zip(lengths, pages)):
        tail = max(length - recent, 0) // bs * bs if many else 0
        first, drop = (sink, many * bs) if many else (0, 0)
        end = tail - drop
        for h in range(hk):
            row = x["w"][r, h]
            key = np.where(np.isnan(row), np.inf, row)[first:tail].astype(np.float64)
            nan = np.isnan(row[first:tail])
            order = np.lexsort((-np.arange(key.size), nan, key))  # the least first, of equal ones the last
            gone = np.zeros(w.shape[2], bool)
            gone[first + order[:drop]] = True
            holes = [t for t in range(first, end) if gone[t]]
            movers = [t for t in range(end, tail) if not gone[t]]
            assert len(holes) == len(movers)
            for to, at in zip(holes, movers):
                bt, bf = table[r, to // bs], table[r, at // bs]
                k[bt, to % bs, h, :8] = x["k"][bf, at % bs, h, :8]
                k[bt, to % bs, h, 32:32 + d // 4] = x["k"][bf, at % bs, h, 32:32 + d // 4]
                v[bt, to % bs, h, :d // 4] = x["v"][bf, at % bs, h, :d // 4]
                if owner[bt % owner.shape[0], to % bs] == bt:
                    owner[bt % owner.shape[0], to % bs] = -1
            w[r, h] = 0
            w[r, h, :end] = row[:end]
            w[r, h, holes] = row[movers]
            w[r, h, end:length - drop] = row[tail:length]
    return k, v, w, owner


def make(lengths, hk, d, bs, seed, weights, width=1, cols=None):
    g = np.random.default_rng(seed)
    per = max(-(-max(lengths) // bs), 1) + 1
    blocks = per * len(lengths) + 3
    table = g.permutation(blocks)[:per * len(lengths)].reshape(len(lengths), per).astype(np.int32)
    k, v = (g.integers(0, 256, (blocks, bs, hk, d * width), dtype=np.uint8) for _ in "kv")
    rows = blocks // 2 + 1
    owner = np.where(g.random((rows, bs)) < 0.5, -1, np.arange(rows)[:, None] + rows * g.integers(0, 2, (rows, bs)))
    w = g.random((len(lengths) + 1, hk, cols or max(lengths) + 37)).astype(np.float32)
    if weights == "coarse":
        w = np.floor(w * 5) / 5
    elif weights == "equal":
        w[:] = 0.25
    elif weights == "special":
        w = w - 0.5
        pick = g.integers(0, 8, w.shape)
        for i, value in enumerate((math.nan, math.inf, -math.inf, 0.0, -0.0, 1e-42)):
            w[pick == i] = value
    elif weights == "rising":
        w = np.sort(w, -1)
    elif weights == "falling":
        w = -np.sort(-w, -1)
    return dict(k=k, v=v, w=np.ascontiguousarray(w, np.float32), owner=owner.astype(np.int64), table=table)


CASES = [
    # lengths, pages, sink, recent, hk, d, bs, legacy
    ([1500], [4], 128, 256, 1, 256, 128, False),
    ([1000, 1000], [6, 6], 128, 100, 2, 256, 128, False),           # all of the middle
    ([1000, 300, 0, 999], [7, 0, 0, 1], 0, 0, 2, 128, 128, False),  # no sink, no recent, no drop
    ([5000, 77, 2049], [30, 1, 60], 5, 3, 1, 128, 32, True),
    ([9000, 8200], [2, 3], 17, 1000, 3, 256, 1536, False),
    ([33000], [129], 1, 300, 2, 256, 128, False),
]


@pytest.mark.gpu
@pytest.mark.parametrize("weights", ["plain", "coarse", "equal", "special", "rising", "falling"])
@pytest.mark.parametrize("lengths,pages,sink,recent,hk,d,bs,legacy", CASES)
def test_every_byte(cuda, lengths, pages, sink, recent, hk, d, bs, legacy, weights):
    from oscar_amd import ops

    x = make(lengths, hk, d, bs, sum(lengths) + d, weights, 2 if legacy else 1)
    k, v, w, owner = reference(x, lengths, pages, sink, recent, d)
    dev = {n: torch.from_numpy(a.copy()).to(cuda) for n, a in x.items()}
    kc, vc = dev["k"].view(torch.int8), dev["v"].view(torch.int8)
    arena = torch.zeros(*owner.shape, hk, d, device=cuda)
    plan = ops.plan_evict(lengths, pages, block_size=bs, sink_tokens=sink, recent_tokens=recent, device=cuda)
    out = torch.full_like(dev["w"], 7.0)
    got = ops.evict(plan, dev["w"], kc, vc, dev["table"], head_dim=d, stage=(arena, arena, dev["owner"]), weights_out=out)
    assert got is out
    reqs = len(lengths)
    assert np.array_equal(got[:reqs].cpu().numpy().view(np.uint32), w[:reqs].view(np.uint32))
    assert np.array_equal(got[reqs:].cpu().numpy().view(np.uint32), x["w"][reqs:].view(np.uint32))
    assert np.array_equal(dev["w"].cpu().numpy().view(np.uint32), x["w"].view(np.uint32))
    assert np.array_equal(dev["k"].cpu().numpy(), k) and np.array_equal(dev["v"].cpu().numpy(), v)
    assert np.array_equal(dev["owner"].cpu().numpy(), owner) and torch.equal(dev["table"].cpu(), torch.from_numpy(x["table"]))


@pytest.mark.gpu
def test_strided_weights_no_window_and_new_output(cuda):
    from oscar_amd import ops

    lengths, pages = [700, 1300], [2, 5]
    x = make(lengths, 2, 128, 128, 3, "coarse")
    k, v, w, _ = reference(x, lengths, pages, 64, 70, 128)
    dev = {n: torch.from_numpy(a.copy()).to(cuda) for n, a in x.items()}
    big = torch.zeros(5, 2, x["w"].shape[2] + 64, device=cuda)
    big[1:4, :, 32:-32] = dev["w"]
    plan = ops.plan_evict(lengths, pages, block_size=128, sink_tokens=64, recent_tokens=70, device=cuda)
    got = ops.evict(plan, big[1:4, :, 32:-32], dev["k"].view(torch.int8), dev["v"].view(torch.int8), dev["table"].long(), head_dim=128)
    assert np.array_equal(got[:2].cpu().numpy(), w[:2]) and np.array_equal(dev["k"].cpu().numpy(), k)
    assert np.array_equal(dev["v"].cpu().numpy(), v)


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["heads outermost", "columns beside each other", "requests beside each other"])
def test_weights_of_other_layouts(cuda, layout):
    """[KV heads, requests, columns], and lists whose old and new weights share a buffer."""
    from oscar_amd import ops

    lengths, pages = [700, 1300], [2, 5]
    x = make(lengths, 2, 128, 128, 3, "plain")
    k, v, w, _ = reference(x, lengths, pages, 64, 70, 128)
    reqs, hk, cols = x["w"].shape
    if layout == "heads outermost":
        old, new = torch.zeros(2, hk, reqs, cols, device=cuda).transpose(1, 2)
    elif layout == "columns beside each other":
        old, new = torch.zeros(reqs, hk, 2 * cols, device=cuda).split(cols, -1)
    else:
        old, new = torch.zeros(reqs, 2, hk, cols, device=cuda).unbind(1)
    old.copy_(torch.from_numpy(x["w"]))
    kc, vc = (torch.from_numpy(x[n].copy()).to(cuda) for n in "kv")
    plan = ops.plan_evict(lengths, pages, block_size=128, sink_tokens=64, recent_tokens=70, device=cuda)
    got = ops.evict(plan, old, kc.view(torch.int8), vc.view(torch.int8), torch.from_numpy(x["table"]).to(cuda), head_dim=128, weights_out=new)
    assert got is new and np.array_equal(got[:2].cpu().numpy(), w[:2]) and np.array_equal(old.cpu().numpy(), x["w"])
    assert np.array_equal(kc.cpu().numpy(), k) and np.array_equal(vc.cpu().numpy(), v)


@pytest.mark.gpu
def test_bad_pages_and_records_touch_nothing_else(cuda):
    """A page id outside the cache, a record that does not fit: bounds hold, the rest is done."""
    from oscar_amd import ops

    lengths, pages = [1000, 1000], [3, 3]
    x = make(lengths, 1, 128, 128, 5, "plain")
    _, _, w, _ = reference(x, lengths, pages, 0, 0, 128)
    dev = {n: torch.from_numpy(a.copy()).to(cuda) for n, a in x.items()}
    plan = ops.plan_evict(lengths, pages, block_size=128, device=cuda)
    before = dev["k"].clone()
    dev["table"][0, :4], dev["table"][0, 4:] = 1 << 30, -5
    plan.requests[1] = torch.tensor([1000, 0, 896, 1024], dtype=torch.int32)
    got = ops.evict(plan, dev["w"], dev["k"].view(torch.int8), dev["v"].view(torch.int8), dev["table"], head_dim=128)
    assert torch.equal(dev["k"], before)
    assert np.array_equal(got[0].cpu().numpy(), w[0]) and torch.equal(got[1], dev["w"][1])


@pytest.mark.gpu
@pytest.mark.parametrize("record", [[1000, 10, -2 ** 31, 128], [-2 ** 31, 10, -2 ** 31, 0], [1000, 900, 896, 0], [1000, 2 ** 31 - 1, 896, 128],
                                    [2 ** 31 - 1, 0, 896, 128], [1000, 0, 896, -2 ** 31]])
def test_records_at_the_ends_of_the_integers_change_nothing(cuda, record):
    from oscar_amd import ops

    x = make([1000], 1, 128, 128, 5, "plain")
    dev = {n: torch.from_numpy(a.copy()).to(cuda) for n, a in x.items()}
    plan = ops.plan_evict([1000], [3], block_size=128, device=cuda)
    plan.requests[0] = torch.tensor(record, dtype=torch.int32)
    before = dev["k"].clone()
    got = ops.evict(plan, dev["w"], dev["k"].view(torch.int8), dev["v"].view(torch.int8), dev["table"], head_dim=128)
    assert torch.equal(dev["k"], before) and torch.equal(got, dev["w"])


@pytest.mark.gpu
def test_wrapper_refusals_on_the_device(cuda):
    from oscar_amd import ops

    x = make([1000], 1, 128, 128, 5, "plain")
    dev = {n: torch.from_numpy(a.copy()).to(cuda) for n, a in x.items()}
    good = dict(plan=ops.plan_evict([1000], [2], block_size=128, device=cuda), weights=dev["w"], k_cache=dev["k"].view(torch.int8),
                v_cache=dev["v"].view(torch.int8), block_table=dev["table"], head_dim=128)
    for change in (dict(plan=ops.plan_evict([1000], [2], block_size=64, device=cuda)), dict(weights=dev["w"][..., :999]),
                   dict(weights=dev["w"].double()), dict(weights=dev["w"].repeat(1, 2, 1)), dict(weights=dev["w"][:0]),
                   dict(weights_out=dev["w"]), dict(weights_out=dev["w"][:, :, 1:]), dict(block_table=dev["table"][:, :7]),
                   dict(block_table=dev["table"][:0]), dict(stage=(dev["w"], dev["w"], dev["owner"]))):
        with pytest.raises(ValueError):
            ops.evict(**{**good, **change})
    with pytest.raises(RuntimeError):
        ops.evict(**{**good, "block_table": dev["table"].cpu()})


@pytest.mark.gpu
def test_captured(cuda):
    from oscar_amd import ops

    lengths, pages = [2000, 1300], [5, 2]
    x = make(lengths, 2, 128, 128, 3, "plain")
    a, b = ({n: torch.from_numpy(t.copy()).to(cuda) for n, t in x.items()} for _ in range(2))
    plan = ops.plan_evict(lengths, pages, block_size=128, device=cuda)
    run = (lambda s, out: ops.evict(plan, s["w"], s["k"].view(torch.int8), s["v"].view(torch.int8), s["table"], head_dim=128,
                                    weights_out=out))
    outs = [torch.empty_like(a["w"]) for _ in range(2)]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        run({n: t.clone() for n, t in a.items()}, outs[0])
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            run(a, outs[0])
    for step in range(3):
        for s in (a, b):
            s["w"].mul_(-1).add_(step)
        torch.cuda.synchronize()
        graph.replay()
        run(b, outs[1])
        torch.cuda.synchronize()
        assert torch.equal(outs[0][:2], outs[1][:2]) and torch.equal(a["k"], b["k"]) and torch.equal(a["v"], b["v"])
