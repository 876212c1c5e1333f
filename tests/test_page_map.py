"""Pages, slots and positions of a step (ops.map_slots, ops.release_pages): refusals on the
CPU, every number against a plain evaluation on the GPU.  Whole numbers, so all are equal."""
import ctypes as C

import numpy as np
import pytest
import torch

from oscar_amd import _lib, ops

INT_MAX = 2 ** 31 - 1


# ------------------------------------------------------------------ refusals (no launch)
def map_args(**changes):
    fixed = dict(lengths=4096, counts=4096, num_reqs=2, block_size=128, num_tokens=10, block_table=4096, block_table_stride=4,
                 block_table_rows=2, block_table_cols=4, pool_pages=4096, pool_count=4096, pool_size=8, query_start_loc=4096,
                 seq_lens=4096, slots=4096, positions=4096, granted=4096)
    return _lib.MapArgs(**{**fixed, **changes})


def release_args(**changes):
    fixed = dict(lengths=4096, new_lengths=4096, num_reqs=2, block_size=128, block_table=4096, block_table_stride=4,
                 block_table_rows=2, block_table_cols=4, pool_pages=4096, pool_count=4096, pool_size=8)
    return _lib.ReleaseArgs(**{**fixed, **changes})


@pytest.mark.parametrize("changes,message", [
    (dict(num_reqs=-1), "at most"), (dict(num_reqs=65537, block_table_rows=65537), "at most"), (dict(num_tokens=-1), "at most"),
    (dict(num_tokens=2 ** 30 + 1), "at most"), (dict(keep=4096, num_tokens=65537), "at most"), (dict(block_size=0), "block_size"),
    (dict(lengths=None), "missing pointer"), (dict(counts=None), "missing pointer"), (dict(slots=None), "missing pointer"),
    (dict(granted=None), "missing pointer"), (dict(pool_count=None), "missing pointer"), (dict(pool_size=-1), "missing pointer"),
    (dict(pool_pages=None), "missing pointer"), (dict(block_table_rows=1), "block-table rows"),
    (dict(block_table_stride=3), "block-table rows"), (dict(block_table_cols=-1), "block-table rows"),
])
def test_map_refusals(changes, message):
    lib = _lib.load()
    assert lib.oscarop_map_v1(C.byref(map_args(**changes)), None) == -22
    assert message in lib.oscar_last_error().decode()


def test_map_workspace():
    lib = _lib.load()
    assert lib.oscarop_map_v1(None, None) == lib.oscarop_release_v1(None, None) == -22
    size = lib.oscarop_map_workspace_bytes_v1
    assert size(3, 5000, 0) == size(3, 100, 1) == 0 and size(3, 5000, 1) >= 4 * (3 + 79)
    assert size(-1, 1, 0) == size(1, -1, 0) == size(65537, 1, 0) == size(1, 65537, 1) == size(1, 2 ** 30 + 1, 0) == -22
    assert lib.oscarop_map_v1(C.byref(map_args(keep=4096, num_tokens=5000)), None) == -28
    assert "workspace" in lib.oscar_last_error().decode()


@pytest.mark.parametrize("changes,message", [
    (dict(num_reqs=-1), "at most"), (dict(num_reqs=65537), "at most"), (dict(block_size=0), "block_size"),
    (dict(lengths=None), "missing pointer"), (dict(new_lengths=None), "missing pointer"), (dict(pool_pages=None), "missing pointer"),
    (dict(block_table_rows=1), "block-table rows"), (dict(block_table_stride=3), "block-table rows"),
])
def test_release_refusals(changes, message):
    lib = _lib.load()
    assert lib.oscarop_release_v1(C.byref(release_args(**changes)), None) == -22
    assert message in lib.oscar_last_error().decode()
    assert lib.oscarop_release_v1(C.byref(release_args(num_reqs=0)), None) == 0


def test_wrappers_refuse_host_tensors():
    pool = ops.PagePool(torch.zeros(4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))
    x = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="device tensors"):
        ops.map_slots(pool, torch.zeros(1, 4, dtype=torch.int32), x, x, tokens=1, block_size=128)
    with pytest.raises(RuntimeError, match="device tensors"):
        ops.release_pages(pool, torch.zeros(1, 4, dtype=torch.int32), x, x, block_size=128)


@pytest.mark.gpu
def test_wrapper_refusals(cuda):
    pool = ops.PagePool.of(8, cuda)
    x, table = torch.zeros(2, dtype=torch.int32, device=cuda), torch.zeros(2, 4, dtype=torch.int32, device=cuda)
    call = lambda pool=pool, table=table, lengths=x, counts=x, tokens=4, bs=128, keep=None: ops.map_slots(  # noqa: E731
        pool, table, lengths, counts, tokens=tokens, block_size=bs, keep=keep)
    for bad, message in ((dict(lengths=x.long()), "lengths"), (dict(counts=x[:1]), "counts"), (dict(table=table.long()), "rows"),
                         (dict(table=table[:1]), "rows"), (dict(table=table.t()), "columns"), (dict(table=table[:1].expand(2, 4)), "overlap"),
                         (dict(tokens=-1), "tokens"), (dict(bs=0), "block_size"), (dict(keep=x.bool()), "keep"),
                         (dict(pool=ops.PagePool(pool.pages.long(), pool.count)), "pool"),
                         (dict(pool=ops.PagePool(pool.pages, pool.pages)), "count")):
        with pytest.raises(ValueError, match=message):
            call(**bad)
    with pytest.raises(ValueError):
        ops.map_slots(pool, table, x, x, tokens=65537, block_size=128, keep=torch.ones(65537, dtype=torch.bool, device=cuda))


# ------------------------------------------------------------------ against a plain evaluation
def ceil_div(a, b):
    return -(-a // b)


def plain_map(pages, free, table, lengths, counts, tokens, bs, keep=None):
    table, reqs, cols = table.copy(), len(lengths), table.shape[1]
    starts, at = [], 0
    for c in counts:
        starts.append(min(at, tokens))
        at += max(int(c), 0)
    starts.append(min(at, tokens))
    free = min(max(free, 0), len(pages))
    grown, need, at = [], [], 0
    for length, c in zip(lengths, counts):
        c = max(int(c), 0)
        fits = length >= 0 and at + c <= tokens
        g = 0
        if fits:
            g = c if keep is None else int(keep[at:at + c].sum())
            fits = length + g <= INT_MAX and ceil_div(length + g, bs) <= cols
        grown.append(g)
        need.append(ceil_div(length + g, bs) - ceil_div(length, bs) if fits else None)
        at += c
    used, granted = 0, []
    for k in need:
        used += k or 0
        granted.append(k is not None and (k == 0 or used <= free))
    taken = sum(k for k, ok in zip(need, granted) if ok)
    top, slots, positions = free - taken, np.full(tokens, -1, np.int64), np.zeros(tokens, np.int64)
    lens = [int(n) for n in lengths]
    for r in range(reqs):
        a, b = starts[r], starts[r + 1]
        positions[a:b] = np.arange(lengths[r], lengths[r] + b - a) if lengths[r] >= 0 else 0
        if not granted[r]:
            continue
        first = ceil_div(lengths[r], bs)
        table[r, first:first + need[r]] = pages[top:top + need[r]]
        top += need[r]
        place = int(lengths[r])
        for i in range(a, b):
            if keep is None or keep[i]:
                page = int(table[r, place // bs])
                slots[i] = page * bs + place % bs if page >= 0 else -1
                place += 1
        lens[r] = place
    return dict(qsl=starts, seq_lens=lens, slots=slots, positions=positions, granted=granted), table, free - taken


def on(device, x, dtype=np.int32):
    return torch.from_numpy(np.ascontiguousarray(np.asarray(x, dtype))).to(device)


def check_map(cuda, lengths, counts, cols, pages, free, tokens, bs, keep=None, seed=0):
    g = np.random.default_rng(seed)
    table = g.integers(0, 10 ** 6, (len(lengths), cols)).astype(np.int32)
    stack = g.permutation(np.arange(pages) + 10 ** 6).astype(np.int32)
    want, new_table, left = plain_map(stack, free, table, lengths, counts, tokens, bs, keep)
    pool = ops.PagePool(on(cuda, stack), on(cuda, [free]))
    dev_table = on(cuda, table)
    got = ops.map_slots(pool, dev_table, on(cuda, lengths), on(cuda, counts), tokens=tokens, block_size=bs,
                        keep=None if keep is None else on(cuda, keep, bool))
    for name, value in want.items():
        assert getattr(got, name).tolist() == list(value), name
    assert np.array_equal(dev_table.cpu().numpy(), new_table)
    assert pool.count.item() == left and np.array_equal(pool.pages.cpu().numpy(), stack)
    return got, pool, dev_table, table, stack


@pytest.mark.gpu
@pytest.mark.parametrize("bs", [128, 32, 100, 1])
@pytest.mark.parametrize("reqs", [1, 3, 65, 1000, 1025, 5000])
@pytest.mark.parametrize("kind", ["decode", "prompts", "keep", "dry", "rough"])
def test_map(cuda, kind, reqs, bs):
    """Decode steps, prompts among them, marked rows, a pool that runs dry, and requests that do
    not fit (negative lengths and counts, tables too narrow, rows past the step's)."""
    g = np.random.default_rng(reqs * 7 + bs)
    lengths = g.integers(0, 40 * bs, reqs)
    lengths[:: 3] -= lengths[:: 3] % bs  # at the border of a page
    counts = g.integers(0, 5, reqs)
    if kind != "decode":
        counts[g.integers(0, reqs, 3)] = g.integers(1, 700, 3)
    total, cols = int(counts.sum()), 41 + 700 // bs
    tokens, keep, pages, free = total + 7, None, 5000, 4000
    if kind == "keep":
        counts = np.minimum(counts, 8)
        total = int(counts.sum())
        tokens = total + 5
        keep = g.random(tokens) < 0.4
    if kind == "dry":
        free = int(g.integers(0, reqs // 8 + 2))
    if kind == "rough":
        cols, tokens = 30, max(total - 3, 0)
        lengths[g.integers(0, reqs, 2)] = -5
        counts[g.integers(0, reqs, 2)] = -1
        lengths[-1] = INT_MAX - 1
    if bs == 1 and kind != "dry":
        pages, free = 60000, 50000
    check_map(cuda, lengths, counts, cols, pages, free, tokens, bs, keep, seed=reqs)


@pytest.mark.gpu
def test_map_at_the_ends_of_the_integers(cuda):
    """Sums past 32 bits, a count outside the pool, empty steps and pools."""
    for lengths, counts, tokens, free in (([5, 5, 5], [INT_MAX, INT_MAX, 2], 100, 10), ([0, 7], [INT_MAX, 1], 2 ** 20, 10),
                                          ([INT_MAX, 3], [1, 1], 10, 10), ([1, 2], [0, 0], 0, 10), ([127, 128], [1, 1], 2, 0),
                                          ([127, 128], [1, 1], 2, 999), ([127, 128], [1, 1], 2, -4), ([-2 ** 31, 9], [1, 2], 3, 5)):
        check_map(cuda, lengths, counts, 40, 16, free, tokens, 128)
    pool = ops.PagePool.of(4, cuda)
    got = ops.map_slots(pool, torch.zeros(0, 4, dtype=torch.int32, device=cuda), on(cuda, []), on(cuda, []), tokens=3, block_size=128)
    assert got.slots.tolist() == [-1] * 3 and got.positions.tolist() == [0] * 3 and got.qsl.tolist() == [0]
    # a page that the table lacks
    table = torch.full((1, 2), -1, dtype=torch.int32, device=cuda)
    got = ops.map_slots(pool, table, on(cuda, [10]), on(cuda, [2]), tokens=2, block_size=128)
    assert got.slots.tolist() == [-1, -1] and got.granted.tolist() == [True] and pool.pages[:4].tolist() == [3, 2, 1, 0]


@pytest.mark.gpu
@pytest.mark.parametrize("reqs,most", [(1, 3), (70, 400), (3000, 5)])
def test_release_undoes_a_map(cuda, reqs, most):
    g = np.random.default_rng(reqs)
    lengths, counts = g.integers(0, 4000, reqs), g.integers(0, most, reqs)
    got, pool, table, _, stack = check_map(cuda, lengths, counts, 48, 9000, 8500, int(counts.sum()), 128)
    ops.release_pages(pool, table, got.seq_lens, on(cuda, lengths), block_size=128)
    assert pool.count.item() == 8500 and np.array_equal(pool.pages.cpu().numpy(), stack)


@pytest.mark.gpu
def test_release_conditions(cuda):
    """Whole pages behind the new length; a longer, negative or too long one gives nothing, nor
    does what the pool has no room for, and what comes after it."""
    table = on(cuda, np.arange(24).reshape(6, 4))
    pool = ops.PagePool(torch.full((10,), -7, dtype=torch.int32, device=cuda), on(cuda, [2]))
    old, new = [500, 256, 300, 600, 400, 129], [129, 0, 301, 1, -1, 128]
    ops.release_pages(pool, table, on(cuda, old), on(cuda, new), block_size=128)
    assert pool.pages.tolist() == [-7, -7, 2, 3, 4, 5, 21, -7, -7, -7] and pool.count.item() == 7
    ops.release_pages(pool, table, on(cuda, [128, 512, 128]), on(cuda, [0, 0, 0]), block_size=128)  # room for three
    assert pool.pages.tolist() == [-7, -7, 2, 3, 4, 5, 21, 0, -7, -7] and pool.count.item() == 8
    with pytest.raises(ValueError, match="new_lengths"):
        ops.release_pages(pool, table, on(cuda, [1, 2]), on(cuda, [1]), block_size=128)


@pytest.mark.gpu
def test_an_eviction_gives_its_pages_back(cuda):
    """plan_evict's lengths and table: the pages of drop.freed, in their order."""
    drop = ops.plan_evict([700, 300, 900], [2, 0, 3], block_size=128, device=cuda)
    table = on(cuda, np.random.default_rng(1).permutation(30).reshape(3, 10))
    pool = ops.PagePool(torch.zeros(30, dtype=torch.int32, device=cuda), on(cuda, [0]))
    new = drop.table(table)
    ops.release_pages(pool, new, on(cuda, drop.lengths), on(cuda, drop.seq_lens), block_size=128)
    want = sum((new[r, a:b].tolist() for r, (a, b) in enumerate(drop.freed)), [])
    assert pool.count.item() == 5 and pool.pages[:5].tolist() == want


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [40, 6000])
def test_captured_map(cuda, tokens):
    """A padded step in a graph: lengths, counts and marks change between the replays, and the pool
    and the table go on from replay to replay."""
    g, reqs, bs = np.random.default_rng(tokens), 5, 32
    lengths, counts = on(cuda, [0] * reqs), on(cuda, [0] * reqs)
    keep, table = torch.zeros(tokens, dtype=torch.bool, device=cuda), torch.zeros(reqs, 400, dtype=torch.int32, device=cuda)
    pool = ops.PagePool.of(1500, cuda)
    ops.map_slots(pool, table, lengths, counts, tokens=tokens, block_size=bs, keep=keep)  # before: libraries, scratch
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.map_slots(pool, table, lengths, counts, tokens=tokens, block_size=bs, keep=keep)
        lengths.copy_(out.seq_lens)
    host_table, host, free = table.cpu().numpy(), np.zeros(reqs, np.int64), 1500
    stack = pool.pages.cpu().numpy()
    for _ in range(5):
        c = g.integers(0, tokens // reqs, reqs)
        marks = g.random(tokens) < 0.5
        counts.copy_(on(cuda, c))
        keep.copy_(on(cuda, marks, bool))
        graph.replay()
        torch.cuda.synchronize()
        want, host_table, free = plain_map(stack, free, host_table, host, c, tokens, bs, marks)
        for name, value in want.items():
            assert getattr(out, name).tolist() == list(value), name
        host = np.asarray(want["seq_lens"])
        assert np.array_equal(table.cpu().numpy(), host_table) and pool.count.item() == free


@pytest.mark.gpu
def test_strides_and_streams(cuda):
    """A wider table's columns, lists out of larger ones, and another stream than the default."""
    wide = torch.zeros(3, 64, dtype=torch.int32, device=cuda)
    lists = on(cuda, [[100, 0, 5, 9], [129, 0, 300, 9], [5, 0, 1, 9]])
    pool = ops.PagePool.of(32, cuda)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = ops.map_slots(pool, wide[:, 10:20], lists[:, 0], lists[:, 2], tokens=400, block_size=128)
    stream.synchronize()
    want, table, left = plain_map(pool.pages.cpu().numpy(), 32, np.zeros((3, 10), np.int32), [100, 129, 5], [5, 300, 1], 400, 128)
    assert got.slots.tolist() == list(want["slots"]) and np.array_equal(wide[:, 10:20].cpu().numpy(), table)
    assert not wide[:, :10].any() and not wide[:, 20:].any() and pool.count.item() == left
