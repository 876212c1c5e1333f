"""A serving loop whose pages, slots, drafts and reads are all dealt on the device: map_slots,
store, page_bounds, tree_mask, attention_tree, select_pages, attention_selected, release_pages
together; the structs of their C calls; and the same calls as torch operators."""
import ctypes as C
import re
import subprocess

import numpy as np
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import oscar_amd.torch_ops  # noqa: F401  (registers the operators)
from oracle.attention import read_history
from oscar_amd import _lib, ops
from test_capi import HEADER
from test_page_select import plain_choice
from test_tree_attention import attn_args, bits, check, random_parents, reference

D, HQ, HK, BS, SCALE = 256, 12, 2, 128, 256 ** -0.5

STRUCTS = {"oscarop_map_args_v1": _lib.MapArgs, "oscarop_release_args_v1": _lib.ReleaseArgs, "oscarop_tree_args_v1": _lib.TreeArgs,
           "oscarop_tree_sizes_v1": _lib.TreeSizes, "oscarop_tree_attn_args_v1": _lib.TreeAttnArgs, "oscarop_bounds_args_v1": _lib.BoundsArgs,
           "oscarop_select_args_v1": _lib.SelectArgs}


def test_structs_match_c_layout(tmp_path):
    header = HEADER.with_name("oscar_operators.h")
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{header}"', "int main(void) {"]
    for name, py in STRUCTS.items():
        lines.append(f'printf("{name} size %zu\\n", sizeof({name}));')
        lines += [f'printf("{name} {field} %zu\\n", offsetof({name}, {field}));' for field, _ in py._fields_]
    (tmp_path / "layout.c").write_text("\n".join([*lines, "return 0; }"]))
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", str(tmp_path / "layout.c"), "-o", str(tmp_path / "layout")], check=True)
    got = dict(line.rsplit(" ", 1) for line in subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True).stdout.splitlines())
    for name, py in STRUCTS.items():
        assert int(got[f"{name} size"]) == C.sizeof(py)
        for field, _ in py._fields_:
            assert int(got[f"{name} {field}"]) == getattr(py, field).offset, (name, field)


def test_packed_fields_are_the_structs():
    """struct.pack of ascending numbers, read back through the structs."""
    def flat(x):
        for name, _ in x._fields_:
            y = getattr(x, name)
            if isinstance(y, C._Pointer):
                y = C.cast(y, C.c_void_p).value
            yield from flat(y) if isinstance(y, C.Structure) else y if isinstance(y, C.Array) else [y]

    for pack, py in ((ops._MAP, _lib.MapArgs), (ops._RELEASE, _lib.ReleaseArgs), (ops._ATTN, _lib.AttnArgs), (ops._SELECT, _lib.SelectArgs),
                     (ops._BOUNDS, _lib.BoundsArgs), (ops._TREE_MASK, _lib.TreeArgs), (ops._ROTATE, _lib.RotateArgs)):
        many = len(list(flat(py())))
        data = pack(*range(1, many + 1))
        assert len(data) == C.sizeof(py) and list(flat(py.from_buffer_copy(data))) == list(range(1, many + 1)), py
    assert C.sizeof(_lib.TreeAttnArgs) == C.sizeof(_lib.AttnArgs) + len(ops._TREE(1, 2, 3))


def test_every_declared_operator_is_exported():
    text = re.sub(r"/\*.*?\*/", "", HEADER.with_name("oscar_operators.h").read_text(), flags=re.S)
    lib = _lib.load()
    names = set(re.findall(r"(oscarop_[a-z_0-9]+)\s*\(", text))
    assert {"oscarop_map_v1", "oscarop_attn_tree_v1", "oscarop_select_v1", "oscarop_attn_selected_v1"} <= names
    for name in names:
        assert hasattr(lib, name), name


def test_torch_operators_are_registered_and_give_shapes():
    mutated = {"map_slots": {"pool_count", "block_table"}, "release_pages": {"pool_pages", "pool_count"}, "tree_mask": set(),
               "attention_tree": set(), "page_bounds": {"bounds"}, "attention_selected": set()}
    for name, want in mutated.items():
        schema = str(getattr(torch.ops.oscar_amd, name).default._schema)
        assert set(re.findall(r"Tensor\(a\d+!\)\?? (\w+)", schema)) == want, schema
    with FakeTensorMode():
        ints = lambda *s: torch.empty(*s, dtype=torch.int32, device="cuda")  # noqa: E731
        qsl, seqs, slots, positions, granted = torch.ops.oscar_amd.map_slots(ints(9), ints(1), ints(3, 4), ints(3), ints(3), 20, 128)
        assert (qsl.shape, seqs.shape, slots.shape, positions.shape, granted.shape) == ((4,), (3,), (20,), (20,), (3,))
        assert slots.dtype == positions.dtype == torch.int64 and granted.dtype == torch.bool
        assert torch.ops.oscar_amd.release_pages(ints(9), ints(1), ints(3, 4), ints(3), ints(3), 128) is None
        mask, depths = torch.ops.oscar_amd.tree_mask(ints(20), ints(4), 65)
        assert mask.shape == (20, 2) and mask.dtype == torch.int64 and depths.shape == (20,)
        q, kc = torch.empty(20, 6, 256, dtype=torch.bfloat16, device="cuda"), torch.empty(8, 128, 1, 256, dtype=torch.int8, device="cuda")
        out, lse = torch.ops.oscar_amd.attention_tree(q, q[:, :1], q[:, :1], kc, kc, ints(1, 8), [0, 20], [300], mask, 0.1, 256)
        assert out.shape == (20, 6, 256) and lse.shape == (20, 6) and out.dtype == torch.float32
        bounds = torch.empty(8, 1, 2, 256, dtype=torch.float16, device="cuda")
        assert torch.ops.oscar_amd.page_bounds(kc, bounds, ints(1, 8), ints(1), ints(1), 5, 256) is None
        out, lse, pages = torch.ops.oscar_amd.attention_selected(q, q[:, :1], q[:, :1], kc, kc, bounds, ints(1, 8), [0, 20], [300], 4, 0.1, 256)
        assert out.shape == (20, 6, 256) and lse.shape == (20, 6) and pages.shape == (1, 1, 4) and pages.dtype == torch.int32


class Loop:
    """A pool, its caches and what the host expects them to hold."""

    def __init__(self, cuda, reqs, blocks, cols):
        self.dev, self.g = cuda, torch.Generator().manual_seed(8)
        self.pool = ops.PagePool(torch.randperm(blocks, generator=self.g).to(cuda, torch.int32), torch.tensor([blocks], dtype=torch.int32, device=cuda))
        self.table = torch.zeros(reqs, cols, dtype=torch.int32, device=cuda)
        self.lengths = torch.zeros(reqs, dtype=torch.int32, device=cuda)
        self.caches = [torch.zeros(blocks, BS, HK, D, dtype=torch.int8, device=cuda) for _ in range(2)]
        self.bounds = torch.zeros(blocks, HK, 2, D, dtype=torch.float16, device=cuda)
        # each request's tokens on pages of its own, in their order
        self.flat = [torch.zeros(reqs * cols, BS, HK, D, dtype=torch.int8, device=cuda) for _ in range(2)]
        self.host, self.cols = [0] * reqs, cols

    def rand(self, n, heads):
        return torch.randn(n, heads, D, generator=self.g).bfloat16().to(self.dev)

    def write(self, counts, k, v, keep=None, max_new=None):
        """A step's rows into the cache; the host's lists and own pages along with them."""
        m = ops.map_slots(self.pool, self.table, self.lengths, torch.tensor(counts, dtype=torch.int32, device=self.dev), tokens=k.shape[0],
                          block_size=BS, keep=keep)
        ops.store(k, v, *self.caches, m.slots, head_dim=D)
        ops.page_bounds(self.caches[0], self.bounds, self.table, self.lengths, m.seq_lens, max_new=max_new or max(counts), head_dim=D)
        at, slots = 0, []
        for r, n in enumerate(counts):
            for i in range(at, at + n):
                if keep is None or keep[i]:
                    slots.append(r * self.cols * BS + self.host[r])
                    self.host[r] += 1
                else:
                    slots.append(-1)
            at += n
        slots += [-1] * (k.shape[0] - at)
        ops.store(k, v, *self.flat, torch.tensor(slots, device=self.dev), head_dim=D)
        self.lengths = m.seq_lens
        assert m.granted.all() and m.seq_lens.tolist() == self.host
        return m

    def check(self):
        """The cache through its table is the flat one, the bounds those of its keys."""
        used = []
        for r, n in enumerate(self.host):
            pages = self.table[r, :-(-n // BS)].long()
            used += pages.tolist()
            own = torch.arange(r * self.cols, r * self.cols + len(pages), device=self.dev)
            for c, f in zip(self.caches, self.flat):
                assert torch.equal(c[pages].flatten(0, 1)[:n], f[own].flatten(0, 1)[:n])
            keys = torch.from_numpy(self.history(r, n)[0])
            for i, p in enumerate(pages):
                x = keys[i * BS:(i + 1) * BS].half()
                assert torch.equal(self.bounds[p].cpu(), torch.stack([x.amin(0), x.amax(0)], 1))
        assert len(set(used)) == len(used) and int(self.pool.count) == self.pool.pages.shape[0] - len(used)

    def history(self, r, n, rounding="f16"):
        own = np.arange(r * self.cols, (r + 1) * self.cols, dtype=np.int32)
        flat = [f.cpu().numpy().view(np.uint8) for f in self.flat]
        return read_history(*flat, own, 0, n, HK, D, None, rounding)


@pytest.mark.gpu
def test_drafts_and_sparse_steps_on_the_device(cuda):
    """Prompts; then rounds of a drafted tree, of which one path is kept, and of a token that reads
    chosen pages; a request that ends and gives its pages to the next."""
    loop, rng, budget = Loop(cuda, 3, 40, 12), np.random.default_rng(2), 4
    prompts = [260, 1100, 90]
    n = sum(prompts)
    loop.write(prompts, loop.rand(n + 3, HK), loop.rand(n + 3, HK))  # (three rows of padding)
    loop.check()
    for turn, nodes in enumerate(([5, 33, 1], [64, 0, 9], [1, 70, 2])):
        qsl, n = [0] + np.cumsum(nodes).tolist(), sum(nodes)
        parents = sum((random_parents(rng, m, "random") for m in nodes), [])
        mask, depths = ops.tree_mask(torch.tensor(parents, dtype=torch.int32, device=cuda), torch.tensor(qsl, dtype=torch.int32, device=cuda),
                                     max_nodes=max(nodes))
        q, k, v = loop.rand(n, HQ), loop.rand(n, HK), loop.rand(n, HK)
        plan = ops.plan_tree(qsl, [h + m for h, m in zip(loop.host, nodes)], num_kv_heads=HK, group=HQ // HK, head_dim=D, device=cuda)
        out, lse = ops.attention_tree(q, k, v, *loop.caches, loop.table, plan, mask, SCALE, head_dim=D)
        keep = torch.zeros(n, dtype=torch.bool)
        for r, m in enumerate(nodes):
            if not m:
                continue
            a, b = qsl[r], qsl[r + 1]
            see = bits(mask[a:b].cpu().numpy(), m)
            old = loop.history(r, loop.host[r], "bf16")[0], loop.history(r, loop.host[r])[1]
            keys, values = (np.concatenate([x, y[a:b].float().cpu().numpy()]) for x, y in zip(old, (k, v)))
            want = reference(q[a:b].float().cpu().numpy(), keys, values, np.concatenate([np.ones((m, loop.host[r]), bool), see], 1), SCALE, 0.0)
            check((out[a:b], lse[a:b]), (*want, keys.shape[0] * np.abs(values).max() * 2.0 ** -32))
            keep[a:b] = torch.from_numpy(see[rng.integers(m)])  # a path to the root
        assert (depths.cpu() >= 0).all()
        loop.write(nodes, k, v, keep.to(cuda))
        loop.check()

        q, k, v = loop.rand(3, HQ), loop.rand(3, HK), loop.rand(3, HK)
        before, lengths = list(loop.host), loop.lengths
        plan = ops.plan_selected([0, 1, 2, 3], [h + 1 for h in before], has_new=True, block_size=BS, budget=budget, first_pages=1, last_pages=2,
                                 num_kv_heads=HK, group=HQ // HK, head_dim=D, device=cuda)
        table, pages = ops.select_pages(q, loop.bounds, loop.table, plan)
        want = plain_choice(q.cpu(), loop.bounds.cpu(), loop.table.cpu(), [0, 1, 2, 3], [h + 1 for h in before], True, BS, budget, 1, 2, HK)
        assert torch.equal(pages.cpu(), want) and (turn or want[1, 0, 1] > 0)
        out, lse = ops.attention_selected(q, k, v, *loop.caches, table, plan, SCALE, head_dim=D)
        for r, h in enumerate(before):
            old = loop.history(r, h, "bf16")[0], loop.history(r, h)[1]
            for head in range(HK):
                at = np.concatenate([np.arange(p * BS, min(p * BS + BS, h)) for p in pages[r, head].tolist() if p >= 0])
                keys, values = (np.concatenate([x[at, head:head + 1], y[r:r + 1, head:head + 1].float().cpu().numpy()]) for x, y in zip(old, (k, v)))
                some = slice(head * HQ // HK, (head + 1) * HQ // HK)
                want = reference(q[r:r + 1, some].float().cpu().numpy(), keys, values, np.ones((1, len(keys)), bool), SCALE, 0.0)
                check((out[r:r + 1, some], lse[r:r + 1, some]), (*want, len(keys) * np.abs(values).max() * 2.0 ** -32))
        assert loop.lengths is lengths
        loop.write([1, 1, 1], k, v)
        loop.check()
        # request `turn` ends; a new one takes its place, on pages that came back
        ends = loop.lengths.clone()
        ends[turn] = 0
        ops.release_pages(loop.pool, loop.table, loop.lengths, ends, block_size=BS)
        loop.lengths, loop.host[turn] = ends, 0
        loop.check()
        counts = [0, 0, 0]
        counts[turn] = 300
        loop.write(counts, loop.rand(300, HK), loop.rand(300, HK))
        loop.check()
    ops.release_pages(loop.pool, loop.table, loop.lengths, loop.lengths * 0, block_size=BS)
    assert int(loop.pool.count) == 40 and sorted(loop.pool.pages.tolist()) == list(range(40))


@pytest.mark.parametrize("scale", [0.0, -0.1, float("nan"), float("inf")])
def test_scales_refused(scale):
    lib = _lib.load()
    a = attn_args(scale=scale)
    assert lib.oscarop_attn_tree_v1(C.byref(a), None, None) == -22 and b"scale" in lib.oscar_last_error()
    assert lib.oscarop_attn_selected_v1(C.byref(a.attn), None, 4, None) == -22 and b"scale" in lib.oscar_last_error()


@pytest.mark.gpu
def test_accepted_nodes_and_the_window(cuda):
    """The store of a tree's accepted rows keeps their FP32 copies, as one of these rows alone does, and
    the next tree reads them."""
    loop = Loop(cuda, 2, 20, 8)
    loop.write([300, 140], loop.rand(440, HK), loop.rand(440, HK))
    stages = [tuple([torch.zeros(64, BS, HK, D, device=cuda), torch.zeros(64, BS, HK, D, device=cuda),
                     torch.full((64, BS), -1, dtype=torch.int64, device=cuda)]) for _ in range(2)]
    nodes, kept = [9, 6], [[0, 3, 4, 8], [1, 2]]
    keep = torch.zeros(15, dtype=torch.bool)
    keep[[0, 3, 4, 8, 10, 11]] = True
    k, v = loop.rand(15, HK), loop.rand(15, HK)
    m = ops.map_slots(loop.pool, loop.table, loop.lengths, torch.tensor(nodes, dtype=torch.int32, device=cuda), tokens=15, block_size=BS,
                      keep=keep.to(cuda))
    window = dict(head_dim=D, stage_mode=ops.STAGE_WRITE, num_reqs=2, recent_tokens=64)
    caches = [[c.clone() for c in loop.caches] for _ in range(2)]
    ops.store(k, v, *caches[0], m.slots, stage=stages[0], qsl_dev=m.qsl, seqs_dev=m.seq_lens, **window)
    rows = keep.nonzero()[:, 0].to(cuda)
    starts = torch.tensor([0, len(kept[0]), len(kept[0]) + len(kept[1])], dtype=torch.int32, device=cuda)
    ops.store(k[rows], v[rows], *caches[1], m.slots[rows], stage=stages[1], qsl_dev=starts, seqs_dev=m.seq_lens, **window)
    assert all(torch.equal(a, b) for a, b in zip((*caches[0], *stages[0]), (*caches[1], *stages[1])))
    assert (stages[0][2] >= 0).sum() == 6
    # all nodes of a chain see the copies: their products with the copies' own keys
    q = loop.rand(2, HQ)
    plan = ops.plan_tree([0, 1, 2], [305, 143], num_kv_heads=HK, group=HQ // HK, head_dim=D, device=cuda)
    mask, _ = ops.tree_mask(torch.tensor([-1, -1], dtype=torch.int32, device=cuda), torch.tensor([0, 1, 2], dtype=torch.int32, device=cuda), max_nodes=1)
    new = [loop.rand(2, HK) for _ in range(2)]
    out, lse = ops.attention_tree(q, *new, *caches[0], loop.table, plan, mask, SCALE, stages[0], head_dim=D)
    for r, h in enumerate([304, 142]):
        table, st = loop.table[r].cpu().numpy(), tuple(x.cpu().numpy() for x in stages[0])
        flat = [c.cpu().numpy().view(np.uint8) for c in caches[0]]
        old = read_history(*flat, table, 0, h, HK, D, st, "bf16")[0], read_history(*flat, table, 0, h, HK, D, st, "f16")[1]
        plain = read_history(*flat, table, 0, h, HK, D, None, "bf16")[0]
        assert (np.abs(old[0] - plain).max((1, 2)) > 0).sum() == len(kept[r])
        keys, values = (np.concatenate([x, y[r:r + 1].float().cpu().numpy()]) for x, y in zip(old, new))
        want = reference(q[r:r + 1].float().cpu().numpy(), keys, values, np.ones((1, h + 1), bool), SCALE, 0.0)
        check((out[r:r + 1], lse[r:r + 1]), (*want, (h + 1) * np.abs(values).max() * 2.0 ** -32))


@pytest.mark.gpu
def test_a_step_in_one_graph(cuda):
    """Slots, write, bounds, choice: one graph, replayed as the requests grow past the ends of their
    pages, against the same calls one by one."""
    loops = [Loop(cuda, 2, 30, 10) for _ in range(2)]
    for loop in loops:
        loop.write([380, 510], loop.rand(890, HK), loop.rand(890, HK))
    graphed, eager = loops
    counts = torch.ones(2, dtype=torch.int32, device=cuda)
    q, k, v = graphed.rand(2, HQ), graphed.rand(2, HK), graphed.rand(2, HK)
    most = ops.plan_selected([0, 1, 2], [400, 530], has_new=False, block_size=BS, budget=3, num_kv_heads=HK, group=HQ // HK, head_dim=D,
                             device=cuda)

    def step(loop, lengths):
        m = ops.map_slots(loop.pool, loop.table, lengths, counts, tokens=2, block_size=BS)
        ops.store(k, v, *loop.caches, m.slots, head_dim=D)
        ops.page_bounds(loop.caches[0], loop.bounds, loop.table, lengths, m.seq_lens, max_new=1, head_dim=D)
        most.seqs.copy_(m.seq_lens)  # the lists on the device are the step's own
        table, pages = ops.select_pages(q, loop.bounds, loop.table, most)
        lengths.copy_(m.seq_lens)
        return m.slots, table, pages

    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(graphed, graphed.lengths)
    for turn in range(10):
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, generator=graphed.g))
        graph.replay()
        want = step(eager, eager.lengths)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), turn
        assert all(torch.equal(a, b) for a, b in zip((*graphed.caches, graphed.bounds, graphed.table, graphed.lengths, graphed.pool.count),
                                                     (*eager.caches, eager.bounds, eager.table, eager.lengths, eager.pool.count)))
    assert graphed.lengths.tolist() == [390, 520]  # (both have taken a page)


@pytest.mark.gpu
def test_torch_operators_match_the_wrappers(cuda):
    a, b = Loop(cuda, 2, 30, 10), Loop(cuda, 2, 30, 10)
    t = torch.ops.oscar_amd
    counts = torch.tensor([700, 300], dtype=torch.int32, device=cuda)
    m = ops.map_slots(a.pool, a.table, a.lengths, counts, tokens=1005, block_size=BS)
    got = t.map_slots(b.pool.pages, b.pool.count, b.table, b.lengths, counts, 1005, BS)
    assert all(torch.equal(x, y) for x, y in zip((m.qsl, m.seq_lens, m.slots, m.positions, m.granted), got))
    assert torch.equal(a.table, b.table) and torch.equal(a.pool.count, b.pool.count)
    k, v = a.rand(1005, HK), a.rand(1005, HK)
    ops.store(k, v, *a.caches, m.slots, head_dim=D)
    ops.page_bounds(a.caches[0], a.bounds, a.table, a.lengths, m.seq_lens, max_new=700, head_dim=D)
    t.page_bounds(a.caches[0], b.bounds, a.table, a.lengths, m.seq_lens, 700, D)
    assert torch.equal(a.bounds, b.bounds) and a.bounds.any()
    parents = torch.tensor([-1, 0, 0, 2, -1, 4], dtype=torch.int32, device=cuda)
    starts = torch.tensor([0, 4, 6], dtype=torch.int32, device=cuda)
    mask, depths = ops.tree_mask(parents, starts, max_nodes=4)
    assert all(torch.equal(x, y) for x, y in zip((mask, depths), t.tree_mask(parents, starts, 4)))
    q, k, v = a.rand(6, HQ), a.rand(6, HK), a.rand(6, HK)
    plan = ops.plan_tree([0, 4, 6], [704, 302], num_kv_heads=HK, group=HQ // HK, head_dim=D, device=cuda)
    out, lse = ops.attention_tree(q, k, v, *a.caches, a.table, plan, mask, SCALE, head_dim=D)
    got = t.attention_tree(q, k, v, *a.caches, a.table, [0, 4, 6], [704, 302], mask, SCALE, D)
    assert torch.equal(out, got[0]) and torch.equal(lse, got[1]) and out.any()
    plan = ops.plan_selected([0, 4, 6], [704, 302], has_new=True, block_size=BS, budget=4, num_kv_heads=HK, group=HQ // HK, head_dim=D, device=cuda)
    table, pages = ops.select_pages(q, a.bounds, a.table, plan)
    out, lse = ops.attention_selected(q, k, v, *a.caches, table, plan, SCALE, head_dim=D)
    got = t.attention_selected(q, k, v, *a.caches, a.bounds, a.table, [0, 4, 6], [704, 302], 4, SCALE, D)
    # (the decode's waves take tiles as they get to them: its last bits are not fixed)
    assert torch.equal(pages, got[2]) and (out - got[0]).abs().max() <= 1e-3 and (lse - got[1]).abs().max() <= 1e-5
    ops.release_pages(a.pool, a.table, m.seq_lens, m.seq_lens - 250, block_size=BS)
    t.release_pages(b.pool.pages, b.pool.count, b.table, m.seq_lens, m.seq_lens - 250, BS)
    assert torch.equal(a.pool.pages, b.pool.pages) and torch.equal(a.pool.count, b.pool.count)
    torch.library.opcheck(t.tree_mask, (parents, starts, 4))
    torch.library.opcheck(t.map_slots, (b.pool.pages, b.pool.count, b.table, b.lengths * 0, counts * 0 + 3, 6, BS))
    torch.library.opcheck(t.page_bounds, (a.caches[0], b.bounds, a.table, a.lengths, m.seq_lens, 700, D), test_utils=("test_schema", "test_faketensor"))
