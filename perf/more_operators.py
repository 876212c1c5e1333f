"""Operators of a serving step over the INT2 cache, in their plain form and as a user calls them.

map     pages for a step's tokens out of the pool, slots and positions of its rows, and back
tree    ancestor masks of drafted trees, and attention of their nodes over the paged history
bounds  for each page and channel the least and the largest key that the page holds
sparse  the pages whose bounds promise the largest scores, and attention over these alone

A case's fields: ``kind``; ``hq`` / ``hk`` / ``d`` (query heads, KV heads, head width);
``dtype`` of the activations; request i has ``histories[i]`` cached tokens and ``chunks[i]``
rows of this step.

Where ``own`` is false ``run`` computes with elementary torch operations, scores of pages in
64 bits (pages next to each other in their order differ little), the rest in 32.
"""
import math
import random

import numpy as np
import torch

own = False

BLOCK = 128           # tokens per cache page
RECENT = 256          # FP32 window per request (the default)
ARENA_TOKENS = 8192   # seats of the window arena (the default)
FIRST, LAST = 1, 3    # pages that are always read: the first, and the last with the window
KINDS = {"bf16": torch.bfloat16, "fp16": torch.float16}

# one rank of the served model: 6 query heads on 1 KV head of width 256, bf16
_MODEL = dict(hq=6, hk=1, d=256, dtype="bf16")
_NARROW = dict(hq=16, hk=2, d=128, dtype="fp16")


def _text(values):
    return ",".join(str(int(v)) for v in values)


def _numbers(text):
    return [int(v) for v in text.split(",")]


def _ragged(n, low, high, seed):
    r = random.Random(seed)
    return [r.randint(low, high) for _ in range(n)]


def _case(kind, name, histories, chunks, **other):
    return dict(_MODEL, name=name, kind=kind, histories=_text(histories), chunks=_text(chunks), **other)


def listed():
    mixed = [2000 if i % 32 == 5 else 1 + i % 4 for i in range(256)]
    return [
        # one user's next token
        _case("map", "map_1x1", [1500], [1], keep=False, short=False),
        # a full server's step: verifications, and some prompts among them
        _case("map", "map_256_mixed", _ragged(256, 0, 30000, 3), mixed, keep=False, short=False),
        # drafted trees after their verification: the accepted nodes' slots, from a pool that runs dry
        _case("map", "map_48_keep", _ragged(48, 100, 30000, 4), [32] * 48, keep=True, short=True),
        # one user early in a chat, a small tree
        _case("tree", "tree_1x500_16", [500], [16], cap=0.0),
        # long contexts, a tree of 32 nodes each
        _case("tree", "tree_8x24k_32", [24576] * 8, [32] * 8, cap=0.0),
        # narrow heads in fp16, capped scores, ragged contexts and trees
        dict(_case("tree", "tree_12_ragged_64", _ragged(12, 700, 16000, 6), _ragged(12, 20, 64, 7), cap=30.0), **_NARROW),
        # the pages that a step of 24 verifying users touched
        _case("bounds", "bounds_24x4", _ragged(24, 1024, 32000, 5), [4] * 24),
        # the pages of four long prompts
        _case("bounds", "bounds_4x30000", [0] * 4, [30000] * 4),
        # one user's long context, an eighth of its pages
        _case("sparse", "sparse_1x32k", [32000], [1], budget=32),
        # the serving steady state: eight long contexts verifying drafts, a quarter of their pages
        _case("sparse", "sparse_8x24k", [24576] * 8, [4] * 8, budget=48),
        # very long contexts
        _case("sparse", "sparse_16x128k", [131072] * 16, [1] * 16, budget=64),
        # narrow heads in fp16, each of two KV heads with pages of its own
        dict(_case("sparse", "sparse_12_ragged", _ragged(12, 3000, 60000, 8), [2] * 12, budget=40), **_NARROW),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """One more case: the same kinds of call over their whole ranges, odd sizes among them."""
    shape = dict(_MODEL)
    shape.update(rng.choice([{}, {}, dict(hq=10, hk=2), dict(hq=8, d=128), dict(_NARROW), dict(dtype="fp16")]))
    kind = rng.choice(["map", "tree", "tree", "bounds", "sparse", "sparse"])
    if kind == "map":
        n = _log(rng, 1, 400)
        histories = [0 if rng.random() < 0.1 else _log(rng, 1, 32000) for _ in range(n)]
        keep = rng.random() < 0.35
        most = rng.choice([4, 16, 64])
        chunks = [rng.randint(0, most) if keep or rng.random() < 0.95 else _log(rng, 64, 3000) for _ in range(n)]
        chunks[0] = max(chunks[0], 1)
        return dict(shape, kind=kind, histories=_text(histories), chunks=_text(chunks), keep=keep, short=rng.random() < 0.25)
    if kind == "bounds":
        n = _log(rng, 1, 48)
        histories = [rng.randint(0, 32000) for _ in range(n)]
        chunks = [rng.randint(0, 5) for _ in range(n)] if rng.random() < 0.6 else [_log(rng, 100, 90000 // n) for _ in range(n)]
        chunks[0] = max(chunks[0], 1)
        return dict(shape, kind=kind, histories=_text(histories), chunks=_text(chunks))
    if kind == "tree":
        n = _log(rng, 1, 16)
        top = min(24576, 240000 // (n * shape["hk"]))
        low = _log(rng, 16, top // 2)
        histories = [rng.randint(low, top) for _ in range(n)]
        if rng.random() < 0.15:
            histories[0] = 0
        chunks = [rng.randint(1, rng.choice([8, 32, 64, 64, 150])) for _ in range(n)]
        cap = rng.choice([0.0, 0.0, float(rng.randint(15, 60))])
        case = dict(shape, kind=kind, histories=_text(histories), chunks=_text(chunks), cap=cap)
        while _tree_flops(case) > 3.5e10:
            chunks = [max(1, c * 2 // 3) for c in chunks]
            case["chunks"] = _text(chunks)
        return case
    n = _log(rng, 1, 16)
    top = min(131072, 1800000 // (n * shape["hk"]))
    low = _log(rng, 300, top // 2)
    histories = [rng.randint(low, top) for _ in range(n)]
    return dict(shape, kind=kind, histories=_text(histories), chunks=_text([rng.randint(1, 5)] * n),
                budget=rng.randint(FIRST + LAST + 1, 64))


# ---------------------------------------------------------------- inputs (plain torch)
def _device():
    return torch.device("cuda", torch.cuda.current_device())


def _rotation(d, gen):
    """A random-sign normalised Hadamard matrix, fp32."""
    h = torch.ones(1, 1, dtype=torch.float64)
    while h.shape[0] < d:
        h = torch.cat([torch.cat([h, h], 1), torch.cat([h, -h], 1)], 0)
    sign = (torch.rand(d, generator=gen, device=gen.device) < 0.5).double() * 2 - 1
    return (sign[:, None] * h.to(gen.device) / math.sqrt(d)).float().contiguous()


def _fill(cache_k, cache_v, d, gen):
    """Every slot of the caches as a server leaves it: the INT2 codes, scales and zeros of
    rotated vectors (K slot: four fp16 constants, codes from byte 32; V slot: codes).  Tokens
    of a page share a part of their keys, as neighbours in a text do."""
    k, v = cache_k.view(torch.uint8).view(-1, cache_k.shape[-1]), cache_v.view(torch.uint8).view(-1, cache_v.shape[-1])
    shifts = torch.tensor([1, 4, 16, 64], device=k.device)
    page = BLOCK * cache_k.shape[2]
    for a in range(0, k.shape[0], page << 9):
        b = min(a + (page << 9), k.shape[0])
        meta = []
        for slots, at, shared in ((k, 32, 0.7), (v, 0, 0.0)):
            y = torch.randn(b - a, d, generator=gen, device=k.device) * 1.4
            if shared:
                y.view(-1, page, d).add_(torch.randn((b - a) // page, 1, d, generator=gen, device=k.device) * shared)
            low, high = y.amin(1, keepdim=True), y.amax(1, keepdim=True)
            scale, zero = ((high - low) / 3).half(), low.half()
            codes = ((y - zero.float()) / scale.float() + 0.5).floor().clamp(0, 3).to(torch.int64)
            slots[a:b, at:at + d // 4] = (codes.view(b - a, d // 4, 4) * shifts).sum(-1).to(torch.uint8)
            meta += [scale, zero]
        k[a:b, :8] = torch.cat(meta, 1).contiguous().view(torch.uint8)


def _unpack(codes, scale, zero):
    """fp32 values of code bytes [..., d / 4] and their constants [..., 1]."""
    shifts = torch.tensor([0, 2, 4, 6], dtype=torch.uint8, device=codes.device)
    return ((codes[..., None] >> shifts) & 3).reshape(*codes.shape[:-1], -1).float() * scale + zero


def _read(cache_k, cache_v, d, slots):
    """The fp32 K and V values of cache slots [..., Hk] (a token slot for each KV head)."""
    hk = cache_k.shape[2]
    heads = torch.arange(hk, device=slots.device)
    k = cache_k.view(torch.uint8).view(-1, hk, cache_k.shape[-1])[slots, heads]
    v = cache_v.view(torch.uint8).view(-1, hk, cache_v.shape[-1])[slots, heads]
    meta = k[..., :8].contiguous().view(torch.float16).float()
    return (_unpack(k[..., 32:32 + d // 4], meta[..., 0:1], meta[..., 1:2]),
            _unpack(v[..., :d // 4], meta[..., 2:3], meta[..., 3:4]))


def _keys(cache_k, d, pages):
    """The keys that slots hold, as fp16, of whole pages: [pages, BLOCK, Hk, D]."""
    k = cache_k.view(torch.uint8)[pages]
    meta = k[..., :4].contiguous().view(torch.float16).float()
    return _unpack(k[..., 32:32 + d // 4], meta[..., 0:1], meta[..., 1:2]).half()


def _last_of(seats):
    """Indexes of the last occurrence of each seat, ascending."""
    _, first = np.unique(seats[::-1], return_index=True)
    return np.sort(len(seats) - 1 - first)


def _table(lengths, seed, spare):
    """A block table of permuted pages for these lengths, and the pages that are left."""
    pages = [-(-n // BLOCK) for n in lengths]
    order = np.random.default_rng(seed).permutation(sum(pages) + spare).astype(np.int32)
    table = np.zeros((len(pages), max(max(pages), 1)), np.int32)
    at = 0
    for r, p in enumerate(pages):
        table[r, :p] = order[at:at + p]
        at += p
    return table, order[at:]


def _paged(case, lengths, gen, seed):
    """Filled caches, their window arena and a block table of permuted pages."""
    dev, d, hk = _device(), case["d"], case["hk"]
    table, rest = _table(lengths, seed, 8)
    blocks = sum(-(-n // BLOCK) for n in lengths) + len(rest)
    k_cache = torch.zeros(blocks, BLOCK, hk, d, dtype=torch.int8, device=dev)
    v_cache = torch.zeros_like(k_cache)
    _fill(k_cache, v_cache, d, gen)
    rows = max(-(-ARENA_TOKENS // BLOCK), -(-RECENT // BLOCK) + 3)
    stage_k = torch.zeros(rows, BLOCK, hk, d, dtype=torch.float32, device=dev)
    stage_v = torch.zeros_like(stage_k)
    owner = torch.full((rows, BLOCK), -1, dtype=torch.int64, device=dev)
    return dict(k_cache=k_cache, v_cache=v_cache, stage_k=stage_k, stage_v=stage_v, owner=owner, host_table=table,
                table=torch.from_numpy(table).to(dev))


def _stage_last(x, case, histories, gen):
    """The window arena: the last RECENT tokens of each history, where the seat is still theirs."""
    table, rows, dev = x["host_table"], x["owner"].shape[0], x["owner"].device
    d, hk = case["d"], case["hk"]
    held = []
    for r, h in enumerate(histories):
        pos = np.arange(max(h - RECENT, 0), h)
        held.append(table[r, pos // BLOCK].astype(np.int64) * BLOCK + pos % BLOCK)
    held = np.concatenate(held)
    if not held.size:
        return
    seats = held // BLOCK % rows * BLOCK + held % BLOCK
    last = _last_of(seats)
    seat, slot = torch.from_numpy(seats[last]).to(dev), torch.from_numpy(held[last]).to(dev)
    for arena, y in zip((x["stage_k"], x["stage_v"]),
                        _read(x["k_cache"], x["v_cache"], d, slot[:, None].expand(-1, hk))):
        spread = y.amax(-1, keepdim=True) - y.amin(-1, keepdim=True)
        noise = torch.rand(y.shape, generator=gen, device=dev) - 0.5
        arena.view(rows * BLOCK, hk, d)[seat] = y + noise * spread / 3
    x["owner"].view(-1)[seat] = slot // BLOCK


def _parents(chunks, seed):
    """Drafted trees, parents before their children: the root (the last accepted token, -1 for
    its parent), then nodes under random ones, the shallow more often; now and then a
    second root."""
    r, out = random.Random(seed), []
    for n in chunks:
        out += [-1 if not i or r.random() < 0.02 else int(i * r.random() ** 2) for i in range(n)]
    return out


def _accepted(parents, chunks, seed):
    """The nodes from the root to a random node of each tree."""
    r, keep, at = random.Random(seed), [False] * len(parents), 0
    for n in chunks:
        node = r.randrange(n) if n else -1
        while node >= 0:
            keep[at + node] = True
            node = parents[at + node]
        at += n
    return keep


def _numbers_of(case):
    histories, chunks = _numbers(case["histories"]), _numbers(case["chunks"])
    return histories, chunks, [0] + np.cumsum(chunks).tolist(), [h + c for h, c in zip(histories, chunks)]


def _inputs(case, seed):
    """Everything a call reads, from the seed alone, as a dict of tensors and host lists."""
    dev = _device()
    gen = torch.Generator(device=dev).manual_seed(seed)
    histories, chunks, starts, lengths = _numbers_of(case)
    n, kind = starts[-1], case["kind"]
    x = dict(histories=histories, chunks=chunks, starts=starts, lengths=lengths)
    x["dev_histories"] = torch.tensor(histories, dtype=torch.int32, device=dev)
    x["dev_chunks"] = torch.tensor(chunks, dtype=torch.int32, device=dev)
    if kind == "map":
        table, rest = _table(histories, seed, sum(-(-c // BLOCK) + 1 for c in chunks))
        wide = max(-(-v // BLOCK) for v in lengths) + 2
        table = np.concatenate([table, np.zeros((len(table), max(wide - table.shape[1], 0)), np.int32)], 1)
        # a pool with room for all, or one that runs dry
        free = sum(-(-b // BLOCK) - -(-a // BLOCK) for a, b in zip(histories, lengths))
        free = free // 8 if case["short"] else free + 5
        keep = _accepted(_parents(chunks, seed), chunks, seed) if case["keep"] else None
        x.update(table=torch.from_numpy(table).to(dev), pages=torch.from_numpy(rest.copy()).to(dev),
                 count=torch.tensor([min(free, len(rest))], dtype=torch.int32, device=dev), rows=n + n % 7,
                 keep=None if keep is None else torch.tensor(keep + [True] * (n % 7), device=dev))
        return x
    d, hq, hk, dtype = case["d"], case["hq"], case["hk"], KINDS[case["dtype"]]
    x.update(_paged(case, lengths, gen, seed))
    if kind == "bounds":
        x["dev_lengths"] = torch.tensor(lengths, dtype=torch.int32, device=dev)
        x["bounds"] = torch.zeros(x["k_cache"].shape[0], hk, 2, d, dtype=torch.float16, device=dev)
        return x
    _stage_last(x, case, histories, gen)

    def rows(heads, scale):
        return (torch.randn(n, heads, d, generator=gen, device=dev) * scale).to(dtype)

    x.update(q=rows(hq, 2.5), k=rows(hk, 1.4), v=rows(hk, 1.4), rv=_rotation(d, gen))
    x["dev_starts"] = torch.tensor(starts, dtype=torch.int32, device=dev)
    if kind == "tree":
        x["parents"] = torch.tensor(_parents(chunks, seed), dtype=torch.int32, device=dev)
        return x
    # the bounds that the steps before left: of each page's tokens up to the history's end
    x["bounds"] = torch.empty(x["k_cache"].shape[0], hk, 2, d, dtype=torch.float16, device=dev)
    for a in range(0, x["bounds"].shape[0], 512):
        keys = _keys(x["k_cache"], d, slice(a, a + 512))
        x["bounds"][a:a + 512] = torch.stack([keys.amin(1), keys.amax(1)], 2)
    for r, h in enumerate(histories):
        if h % BLOCK:
            page = int(x["host_table"][r, h // BLOCK])
            keys = _keys(x["k_cache"], d, slice(page, page + 1))[:, :h % BLOCK]
            x["bounds"][page] = torch.stack([keys.amin(1), keys.amax(1)], 2)[0]
    return x


def prepare(case, seed):
    state = dict(_inputs(case, seed), **{k: case[k] for k in ("kind", "hq", "hk", "d", "dtype")})
    state.update(cap=case.get("cap", 0.0), budget=case.get("budget", 0))
    if case["kind"] in ("tree", "sparse"):
        state["stage"] = (state["stage_k"], state["stage_v"], state["owner"])
    if own:
        # the batch's plan, which a model's layers share, and the pool, which a server keeps
        from oscar_amd import ops

        sizes = dict(num_kv_heads=case["hk"], group=case["hq"] // case["hk"], head_dim=case["d"], device=_device(),
                     window=(0, RECENT))
        if case["kind"] == "map":
            state["pool"] = ops.PagePool(state["pages"], state["count"])
        elif case["kind"] == "tree":
            state["plan"] = ops.plan_tree(state["starts"], state["lengths"], **sizes)
        elif case["kind"] == "sparse":
            state["plan"] = ops.plan_selected(state["starts"], state["lengths"], has_new=True, block_size=BLOCK,
                                              budget=case["budget"], first_pages=FIRST, last_pages=LAST, **sizes)
    return state


# ---------------------------------------------------------------- the plain forms
def _pages(tokens):
    return (tokens + BLOCK - 1) // BLOCK


def _plain_map(s):
    """Pages off the top of the pool's stack, requests in their order and each request's
    ascending, for those that the pool still has pages for; then slots and positions of all
    rows; then the pages go back where they were taken from."""
    table, length, count = s["table"], s["dev_histories"].long(), s["dev_chunks"].long()
    dev, rows, reqs = table.device, s["rows"], table.shape[0]
    starts = torch.cat([count.new_zeros(1), count.cumsum(0)])
    row = torch.arange(rows, device=dev)
    real = row < starts[-1]
    req = torch.searchsorted(starts[1:], row, right=True).clamp(max=reqs - 1)
    keep = real if s["keep"] is None else real & s["keep"]
    before = torch.cat([count.new_zeros(1), keep.long().cumsum(0)])
    grown = length + before[starts[1:]] - before[starts[:-1]]
    old, new = _pages(length), _pages(grown)
    need = torch.where(new <= table.shape[1], new - old, 0)
    upto = need.cumsum(0)
    granted = (new <= table.shape[1]) & ((need == 0) | (upto <= s["count"].long()))
    taken = torch.where(granted, need, 0)
    total = taken.sum()
    col = torch.arange(table.shape[1], device=dev)
    fresh = granted[:, None] & (col >= old[:, None]) & (col < new[:, None])
    at = s["count"].long() - total + (upto - need)[:, None] + col - old[:, None]
    table = torch.where(fresh, s["pages"][at.clamp(0, s["pages"].shape[0] - 1)], table)
    s["table"].copy_(table)
    place = length[req] + before[row] - before[starts[req]]
    page = table[req, (place // BLOCK).clamp(max=table.shape[1] - 1)].long()
    slots = torch.where(keep & granted[req], page * BLOCK + place % BLOCK, -1)
    positions = torch.where(real, length[req] + row - starts[req], 0)
    back = torch.where(fresh, at, s["pages"].shape[0])
    pages = torch.cat([s["pages"], s["pages"][:1]]).scatter(0, back.flatten(), table.flatten())[:-1]
    s["pages"].copy_(pages)
    return dict(starts=starts.int(), lengths=torch.where(granted, grown, length).int(), slots=slots, positions=positions,
                granted=granted, table=s["table"], pages=s["pages"], count=s["count"])


def _plain_masks(s):
    """Bit j of row i: the request's node j is node i or one of its ancestors.  By squaring the
    relation: after k rounds up to 2^k generations."""
    most, parents, dev = max(s["chunks"]), s["parents"].long(), s["parents"].device
    node = torch.arange(most, device=dev)
    count, start = s["dev_chunks"].long()[:, None], s["dev_starts"].long()[:-1, None]
    parent = torch.where(node < count, parents[(start + node).clamp(max=parents.shape[0] - 1)], -1)
    see = (parent[..., None] == node) | (node[:, None] == node)
    see = see.float()
    for _ in range(max(1, (most - 1).bit_length())):
        see = (see @ see).clamp(max=1.0)
    see = see.bool()
    words = -(-most // 64)
    bits = torch.nn.functional.pad(see, (0, 64 * words - most)).view(*see.shape[:2], words, 64)
    mask = (bits.long() << torch.arange(64, device=dev)).sum(-1)
    real = node < count
    return mask[real], (see.sum(-1) - 1)[real].int(), see


def _unpadded(s, x):
    """Padded rows [requests, hk, tokens * group, ...] as the batch's rows [n, hq, ...]."""
    tokens, group = max(s["chunks"]), s["hq"] // s["hk"]
    x = x.view(*x.shape[:2], tokens, group, *x.shape[3:]).transpose(1, 2).reshape(x.shape[0], tokens, s["hq"], *x.shape[3:])
    return x[torch.arange(tokens, device=x.device) < s["dev_chunks"][:, None]]


def _padded_queries(s):
    """The queries as [requests, hk, tokens * group, d], padded to the longest chunk."""
    tokens, group = max(s["chunks"]), s["hq"] // s["hk"]
    at = s["dev_starts"].long()[:-1, None] + torch.arange(tokens, device=s["q"].device)
    q = s["q"][at.clamp(max=s["q"].shape[0] - 1)]
    return q.view(-1, tokens, s["hk"], group, s["d"]).transpose(1, 2).reshape(-1, s["hk"], tokens * group, s["d"])


def _plain_attention(s, table, history, see):
    """Attention over the pages of table [requests, hk, columns] that hold `history` tokens
    and the chunk's rows that a row sees ([requests, tokens, tokens])."""
    d, hk, group, dtype = s["d"], s["hk"], s["hq"] // s["hk"], KINDS[s["dtype"]]
    dev, rows, tokens = table.device, s["owner"].shape[0], max(s["chunks"])
    hist, count, start = history[:, None], s["dev_chunks"].long()[:, None], s["dev_starts"].long()[:-1, None]
    longest = table.shape[2] * BLOCK
    pos = torch.arange(longest, device=dev)
    block = table.long().repeat_interleave(BLOCK, 2).transpose(1, 2).clamp(min=0)
    off = (pos % BLOCK)[None, :, None]
    seat = block % rows * BLOCK + off
    heads = torch.arange(hk, device=dev)
    staged = (s["owner"].view(-1)[seat] == block)[..., None]
    new = (start + torch.arange(tokens, device=dev)).clamp(max=s["q"].shape[0] - 1)
    stored, keys = _read(s["k_cache"], s["v_cache"], d, block * BLOCK + off), []
    for name, old, arena in (("k", stored[0], s["stage_k"]), ("v", stored[1], s["stage_v"])):
        # a history value is fp16(x), and of the activations' type for keys
        old = torch.where(staged, arena.view(-1, hk, d)[seat, heads], old).half()
        old = (old.to(dtype) if name == "k" else old).float()
        keys.append(torch.cat([old, s[name][new].float()], 1).transpose(1, 2))
    x = _padded_queries(s).float() @ keys[0].transpose(-1, -2) * d ** -0.5
    if s["cap"]:
        x = s["cap"] * torch.tanh(x / s["cap"])
    seen = torch.cat([(pos < hist)[:, None].expand(-1, tokens, -1), see], 2)
    seen = seen & (torch.arange(tokens, device=dev) < count)[..., None]
    x = torch.where(seen[:, None].repeat_interleave(group, 2), x, -math.inf)
    top = x.amax(-1, keepdim=True).clamp(min=-1e30)
    x = torch.exp(x - top)
    total = x.sum(-1, keepdim=True)
    out, lse = _unpadded(s, (x @ keys[1]) / total), _unpadded(s, (top + torch.log(total))[..., 0])
    return dict(out=(out @ s["rv"].t()).to(dtype), lse=lse)


def _plain_tree(s):
    mask, depths, see = _plain_masks(s)
    table = s["table"][:, None].expand(-1, s["hk"], -1)
    node = torch.arange(see.shape[-1], device=see.device)
    see = see & (node < s["dev_chunks"][:, None])[:, None]
    return dict(_plain_attention(s, table, s["dev_histories"].long(), see), mask=mask, depths=depths)


def _plain_bounds(s):
    """The pages from each history's last one to the new end, over the tokens that they hold."""
    old, new = s["dev_histories"].long() // BLOCK, _pages(s["dev_lengths"].long())
    old = torch.where(s["dev_chunks"] > 0, old, new)
    col = torch.arange(s["table"].shape[1], device=s["table"].device)
    touched = (col >= old[:, None]) & (col < new[:, None])
    r, c = touched.nonzero(as_tuple=True)
    pages = s["table"][r, c].long()
    keys = _keys(s["k_cache"], s["d"], pages)
    held = (torch.arange(BLOCK, device=col.device) + (c * BLOCK)[:, None]) < s["dev_lengths"][r][:, None]
    held = held[..., None, None]
    s["bounds"][pages] = torch.stack([torch.where(held, keys, math.inf).amin(1), torch.where(held, keys, -math.inf).amax(1)], 2)
    return dict(bounds=s["bounds"])


def _plain_sparse(s):
    """A page's score: the largest over the request's queries of the sum over the channels of
    max(q low, q high).  The first and last pages, and of the others those of the largest
    scores (of equal ones the earlier), ascending; all of a history that fits."""
    dev, hk, budget = s["table"].device, s["hk"], s["budget"]
    history, count = s["dev_histories"].long(), s["dev_chunks"].long()
    pages, cols = _pages(history), s["table"].shape[1]
    group, tokens = s["hq"] // hk, max(s["chunks"])
    q = _padded_queries(s).double()
    bounds = s["bounds"][s["table"].long()].double().transpose(1, 2)  # [requests, hk, columns, 2, d]
    x = q.clamp(min=0) @ bounds[..., 1, :].transpose(-1, -2) + q.clamp(max=0) @ bounds[..., 0, :].transpose(-1, -2)
    real = (torch.arange(tokens, device=dev) < count[:, None])[:, None].repeat_interleave(group, 2)
    x = torch.where(real[..., None], x, -math.inf).amax(2)
    col = torch.arange(cols, device=dev)
    forced = (col < FIRST) | (col >= pages[:, None] - LAST)
    x = torch.where(forced[:, None], math.inf, x)
    x = torch.where((col < pages[:, None])[:, None], x, -math.inf)
    order = torch.sort(x, descending=True, stable=True).indices
    rank = torch.empty_like(order).scatter_(-1, order, col.expand_as(order))
    chosen = (rank < budget) & (col < pages[:, None])[:, None]
    # the chosen columns ascending, -1 behind them
    wide = max(budget, cols)
    key = torch.where(chosen, col, cols).sort(-1).values
    key = torch.nn.functional.pad(key, (0, wide - cols), value=cols)[..., :budget]
    there = key < cols
    table = torch.gather(s["table"][:, None].expand(-1, hk, -1), 2, key.clamp(max=cols - 1))
    table = torch.where(there, table, -1)
    fewer = (pages - budget).clamp(min=0)
    node = torch.arange(tokens, device=dev)
    see = ((node[:, None] >= node) & (node < count[:, None, None]))
    out = _plain_attention(s, table, history - fewer * BLOCK, see)
    return dict(out, table=table.int(), pages=torch.where(there, key, -1).int())


def run(state):
    s, kind = state, state["kind"]
    if not own:
        return {"map": _plain_map, "tree": _plain_tree, "bounds": _plain_bounds, "sparse": _plain_sparse}[kind](s)
    from oscar_amd import ops

    if kind == "map":
        # a step's pages, and back again: a step that is not taken
        m = ops.map_slots(s["pool"], s["table"], s["dev_histories"], s["dev_chunks"], tokens=s["rows"], block_size=BLOCK,
                          keep=s["keep"])
        ops.release_pages(s["pool"], s["table"], m.seq_lens, s["dev_histories"], block_size=BLOCK)
        return dict(starts=m.qsl, lengths=m.seq_lens, slots=m.slots, positions=m.positions, granted=m.granted,
                    table=s["table"], pages=s["pages"], count=s["count"])
    if kind == "bounds":
        return dict(bounds=ops.page_bounds(s["k_cache"], s["bounds"], s["table"], s["dev_histories"], s["dev_lengths"],
                                           max_new=max(s["chunks"]), head_dim=s["d"]))
    scale = s["d"] ** -0.5
    if kind == "tree":
        mask, depths = ops.tree_mask(s["parents"], s["dev_starts"], max_nodes=max(s["chunks"]))
        out, lse = ops.attention_tree(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["table"], s["plan"], mask, scale,
                                      s["stage"], head_dim=s["d"], soft_cap=s["cap"])
        extra = dict(mask=mask, depths=depths)
    else:
        table, pages = ops.select_pages(s["q"], s["bounds"], s["table"], s["plan"])
        out, lse = ops.attention_selected(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], table, s["plan"], scale,
                                          s["stage"], head_dim=s["d"])
        extra = dict(table=table, pages=pages)
    return dict(extra, out=ops.rotate(out, s["rv"], transpose=True, out_dtype=s["q"].dtype), lse=lse)


# ---------------------------------------------------------------- what a pass cannot do without
def _tree_flops(case):
    histories, chunks, _, _ = _numbers_of(case)
    return 4 * case["d"] * case["hq"] * sum(c * h + c * (c + 1) // 2 for h, c in zip(histories, chunks))


def work(case):
    histories, chunks, starts, lengths = _numbers_of(case)
    n, reqs, kind = starts[-1], len(histories), case["kind"]
    if kind == "map":
        fresh = sum(-(-b // BLOCK) - -(-a // BLOCK) for a, b in zip(histories, lengths))
        # lengths and counts in, starts and lengths out, slots and positions; a page read for a
        # request's last token, a new page read and written twice
        return dict(bytes=17 * reqs + 16 * n + (n if case["keep"] else 0) + 4 * reqs + 16 * fresh, flops=0)
    d, hq, hk = case["d"], case["hq"], case["hk"]
    if kind == "bounds":
        total = 0
        for a, c, b in zip(histories, chunks, lengths):
            if c:
                total += hk * ((b - a // BLOCK * BLOCK) * (4 + d // 4) + (-(-b // BLOCK) - a // BLOCK) * 4 * d)
        return dict(bytes=total + 8 * reqs, flops=0)
    slot, flops = 8 + d // 2, 2 * d * d * n * hq
    total = n * (4 * hq * d + 4 * hk * d + 4 * hq) + 4 * d * d
    for h, c in zip(histories, chunks):
        if kind == "sparse":
            pages = -(-h // BLOCK)
            scored = pages - FIRST - LAST if pages > case["budget"] else 0
            total += hk * scored * 4 * d
            flops += scored * 4 * d * c * hq
            h -= max(pages - case["budget"], 0) * BLOCK
        staged = min(h, RECENT)
        total += hk * ((h - staged) * slot + staged * 8 * d)
        flops += 4 * d * hq * (c * h + c * (c + 1) // 2)
    if kind == "tree":
        total += n * (4 + 8 * -(-max(chunks) // 64) + 4)
    return dict(bytes=total, flops=flops)


# ---------------------------------------------------------------- 64 bits
def _exact_map(case, x):
    histories, chunks, starts = x["histories"], x["chunks"], x["starts"]
    table, stack, free = x["table"].cpu().numpy().copy(), x["pages"].cpu().numpy(), int(x["count"])
    keep = [True] * x["rows"] if x["keep"] is None else x["keep"].tolist()
    grown = [h + sum(keep[a:a + c]) for h, c, a in zip(histories, chunks, starts)]
    need = [-(-b // BLOCK) - -(-a // BLOCK) for a, b in zip(histories, grown)]
    granted, used = [], 0
    for k in need:  # no later request gets pages once one went without
        used += k
        granted.append(k == 0 or used <= free)
    at = free - sum(k for k, ok in zip(need, granted) if ok)
    slots, positions = np.full(x["rows"], -1, np.int64), np.zeros(x["rows"], np.int64)
    for r, (h, c, a) in enumerate(zip(histories, chunks, starts)):
        positions[a:a + c] = np.arange(h, h + c)
        if not granted[r]:
            grown[r] = h
            continue
        first = -(-h // BLOCK)
        table[r, first:first + need[r]] = stack[at:at + need[r]]
        at += need[r]
        place = h
        for i in range(a, a + c):
            if keep[i]:
                slots[i] = int(table[r, place // BLOCK]) * BLOCK + place % BLOCK
                place += 1
    as32 = lambda v: torch.from_numpy(np.asarray(v, np.int32))  # noqa: E731
    return dict(starts=as32(starts), lengths=as32(grown), slots=torch.from_numpy(slots),
                positions=torch.from_numpy(positions), granted=torch.tensor(granted), table=torch.from_numpy(table),
                pages=torch.from_numpy(stack), count=x["count"].cpu())


def _exact_bounds(case, x):
    out = x["bounds"].double()
    for r, (h, c, b) in enumerate(zip(x["histories"], x["chunks"], x["lengths"])):
        for col in range(h // BLOCK, -(-b // BLOCK)) if c else ():
            page = int(x["host_table"][r, col])
            k = x["k_cache"][page, :min(BLOCK, b - col * BLOCK)].view(torch.uint8)
            consts = k[..., :4].contiguous().view(torch.float16).double()
            codes = k[..., 32:32 + case["d"] // 4]
            codes = torch.stack([codes & 3, codes >> 2 & 3, codes >> 4 & 3, codes >> 6], -1).flatten(-2).double()
            y = (codes * consts[..., :1] + consts[..., 1:]).float().half().double()
            out[page] = torch.stack([y.min(0).values, y.max(0).values], 1)
    return dict(bounds=out)


def _exact_request(case, x, r, head, table, history):
    """Keys and values [history, d] of the pages in `table` for one KV head, in 64 bits."""
    dtype, rows, dev = KINDS[case["dtype"]], x["owner"].shape[0], x["owner"].device
    pos = np.arange(history)
    block = torch.from_numpy(np.asarray(table, np.int64)[pos // BLOCK]).to(dev)
    off = torch.from_numpy(pos % BLOCK).to(dev)
    mine = (x["owner"][block % rows, off] == block)[:, None]
    k = x["k_cache"].view(torch.uint8)[block, off, head]
    v = x["v_cache"].view(torch.uint8)[block, off, head]
    meta, got = k[:, :8].contiguous().view(torch.float16).float(), []
    for at, codes, arena, narrow in ((0, k[:, 32:32 + case["d"] // 4], x["stage_k"], dtype),
                                     (2, v[:, :case["d"] // 4], x["stage_v"], torch.float16)):
        codes = torch.stack([codes & 3, codes >> 2 & 3, codes >> 4 & 3, codes >> 6], -1).flatten(-2).float()
        y = codes * meta[:, at:at + 1] + meta[:, at + 1:at + 2]
        got.append(torch.where(mine, arena[block % rows, off, head], y).half().to(narrow).double())
    return got


def _exact_rows(case, x, r, h, keys, values, see):
    """Outputs (before the rotation) and log-sum-exps of request r's rows for query head h."""
    a, c, kv = x["starts"][r], x["chunks"][r], h // (case["hq"] // case["hk"])
    keys = torch.cat([keys, x["k"][a:a + c, kv].double()])
    values = torch.cat([values, x["v"][a:a + c, kv].double()])
    s = x["q"][a:a + c, h].double() @ keys.t().contiguous() / math.sqrt(case["d"])
    if case.get("cap"):
        s = torch.tanh(s / case["cap"]) * case["cap"]
    s[:, -c:] = s[:, -c:].masked_fill(~see, -math.inf)
    return torch.softmax(s, -1) @ values, torch.logsumexp(s, -1)


def _exact_attention(case, x):
    hq, hk, d, dev = case["hq"], case["hk"], case["d"], x["q"].device
    group, tree = hq // hk, case["kind"] == "tree"
    out = torch.empty(x["q"].shape, dtype=torch.float64, device=dev)
    lse = torch.empty(out.shape[:2], dtype=torch.float64, device=dev)
    parents = x["parents"].tolist() if tree else None
    masks, depths, tables, chosen = [], [], [], []
    for r, (history, c, a) in enumerate(zip(x["histories"], x["chunks"], x["starts"])):
        see = torch.ones(c, c, dtype=torch.bool).tril()
        if tree:
            see = torch.zeros(c, c, dtype=torch.bool)
            for i in range(c):
                p = parents[a + i]
                if p >= 0:
                    see[i] = see[p]
                see[i, i] = True
                depths.append(int(see[i].sum()) - 1)
                bits = sum(1 << j for j in see[i].nonzero().flatten().tolist())
                masks.append([(w ^ (1 << 63)) - (1 << 63) for w in
                              (bits >> 64 * k & (1 << 64) - 1 for k in range(-(-max(x["chunks"]) // 64)))])
        see = see.to(dev)
        pages = -(-history // BLOCK)
        for kv in range(hk):
            cols = np.arange(pages)
            if not tree and pages > case["budget"]:
                mid = cols[FIRST:pages - LAST]
                b = x["bounds"][torch.from_numpy(x["host_table"][r, mid].astype(np.int64)).to(dev), kv].double()
                best = torch.full((len(mid),), -math.inf, dtype=torch.float64, device=dev)
                for h in range(kv * group, (kv + 1) * group):
                    for i in range(a, a + c):
                        q = x["q"][i, h].double()
                        best = torch.maximum(best, torch.maximum(b[:, 0] * q, b[:, 1] * q).sum(-1))
                order = np.argsort(-best.cpu().numpy(), kind="stable")[:case["budget"] - FIRST - LAST]
                cols = np.sort(np.concatenate([cols[:FIRST], mid[order], cols[pages - LAST:]]))
            table = x["host_table"][r, cols]
            if not tree:
                none = [-1] * (case["budget"] - len(cols))
                chosen.append(cols.tolist() + none)
                tables.append(table.tolist() + none)
            keys, values = _exact_request(case, x, r, kv, table, history - (pages - len(cols)) * BLOCK)
            for h in range(kv * group, (kv + 1) * group):
                out[a:a + c, h], lse[a:a + c, h] = _exact_rows(case, x, r, h, keys, values, see)
    result = dict(out=out @ x["rv"].double().t().contiguous(), lse=lse)
    if tree:
        return dict(result, mask=torch.tensor(masks), depths=torch.tensor(depths, dtype=torch.int32))
    shape = (len(x["chunks"]), hk, case["budget"])
    return dict(result, table=torch.tensor(tables, dtype=torch.int32).view(shape),
                pages=torch.tensor(chosen, dtype=torch.int32).view(shape))


def exact(case, seed):
    x = _inputs(case, seed)
    return {"map": _exact_map, "bounds": _exact_bounds}.get(case["kind"], _exact_attention)(case, x)
