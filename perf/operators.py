"""Operators around the INT2 cache, in their plain form and as a user calls them.

norm_rope  RMS norms of the query and key heads and their position rotation, before the write
decode     attention over the paged INT2 history and a short chunk, scores capped and biased
prompt     the same for one long chunk, with or without a cached history
weights    the attention weight that each cached token received, added to what it had
evict      the tokens of least accumulated weight leave the cache, whole pages at a time

A case's fields: ``kind``; ``hq`` / ``hk`` / ``d`` (query heads, KV heads, head width);
``dtype`` of the activations; for the attention kinds ``cap`` (0: none) and ``alibi``, and a
batch in which request i has ``histories[i]`` cached tokens and ``chunks[i]`` new ones.

Where ``own`` is false ``run`` computes with elementary torch operations in fp32.
"""
import math
import random

import numpy as np
import torch

own = False

BLOCK = 128           # tokens per cache page
RECENT = 256          # FP32 window per request (the default)
SINK = 128            # first tokens that eviction keeps
ARENA_TOKENS = 8192   # seats of the window arena (the default)
EPS = 1e-6
KINDS = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}

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


def _batch(kind, name, histories, chunks, **other):
    return dict(dict(_MODEL, cap=0.0, alibi=False), name=name, kind=kind, histories=_text(histories),
                chunks=_text(chunks), **other)


def listed():
    return [
        # one token of one user: launch and latency
        dict(_MODEL, name="norm_rope_1", kind="norm_rope", tokens=1, rotary=64, offset=1.0, interleaved=False),
        # a long chunk of a prompt on a rank with four KV heads, whole heads rotated in pairs
        dict(name="norm_rope_15361", kind="norm_rope", tokens=15361, hq=24, hk=4, d=128, dtype="bf16", rotary=128,
             offset=0.0, interleaved=True),
        # one user early in a chat, capped scores
        _batch("decode", "decode_1x500_cap", [500], [1], cap=30.0),
        # the serving steady state: eight long contexts verifying drafts, capped scores
        _batch("decode", "verify_8x24k_cap", [24576] * 8, [4] * 8, cap=50.0),
        # narrow heads in fp16 with a distance bias, ragged lengths
        dict(_batch("decode", "decode_24_alibi", _ragged(24, 700, 16000, 6), [2] * 24), **_NARROW, alibi=True),
        # a fresh prompt of ordinary length, cap and bias together
        _batch("prompt", "prompt_2047_cap_alibi", [0], [2047], cap=30.0, alibi=True),
        # a long chunk over a cached prompt, capped scores
        _batch("prompt", "continue_8000_1600_cap", [8000], [1600], cap=50.0),
        # the weights of one decode step of one user
        _batch("weights", "weights_1x500", [500], [1]),
        # the weights of a full server's step, capped scores
        _batch("weights", "weights_24_ragged_cap", _ragged(24, 1024, 32768, 5), [2] * 24, cap=50.0),
        # the weights of a fresh prompt
        _batch("weights", "weights_prompt_2500", [0], [2500]),
        # one user's cache down by four pages
        dict(_MODEL, name="evict_1x1500", kind="evict", lengths="1500", drops="4", coarse=False),
        # a full server: long caches of two KV heads halved, with many equal weights
        dict(_NARROW, name="evict_16_ragged", kind="evict", lengths=_text(_ragged(16, 3000, 32000, 9)),
             drops=_text(v // 2 // BLOCK for v in _ragged(16, 3000, 32000, 9)), coarse=True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _pairs(case):
    """Visible query-key pairs of a batch."""
    return sum(c * h + c * (c + 1) // 2 for h, c in zip(_numbers(case["histories"]), _numbers(case["chunks"])))


def draw(rng):
    """One more case: the same kinds of call over their whole ranges, odd sizes among them."""
    shape = dict(_MODEL)
    shape.update(rng.choice([{}, {}, dict(hq=12, hk=2), dict(hq=8, d=128), dict(_NARROW), dict(dtype="fp16")]))
    kind = rng.choice(["norm_rope", "norm_rope", "decode", "decode", "decode", "prompt", "prompt", "weights", "weights",
                       "weights", "evict", "evict"])
    if kind == "norm_rope":
        return dict(shape, kind=kind, tokens=_log(rng, 1, 60000 // shape["hq"]), rotary=rng.choice([32, 64, 96, shape["d"]]),
                    offset=rng.choice([0.0, 1.0]), interleaved=rng.random() < 0.3,
                    **({} if rng.random() < 0.7 else dict(dtype="fp32")))
    if kind == "evict":
        n = _log(rng, 1, 16)
        lengths = [_log(rng, 700, 32000) for _ in range(n)]
        drops = [rng.randint(1, (v - SINK - RECENT) // BLOCK - 1) for v in lengths]
        if n > 2 and rng.random() < 0.5:  # a request that keeps all it has
            drops[1] = 0
        return dict(shape, kind=kind, lengths=_text(lengths), drops=_text(drops), coarse=rng.random() < 0.3)
    score = rng.choice([dict(cap=0.0, alibi=True), dict(cap=float(rng.randint(15, 60)), alibi=False),
                        dict(cap=float(rng.randint(15, 60)), alibi=True)])
    if kind == "weights" and rng.random() < 0.4:
        score = dict(cap=0.0, alibi=False)
    if kind == "prompt" or kind == "weights" and rng.random() < 0.35:
        histories, chunks = [rng.choice([0, _log(rng, 100, 9000)])], [_log(rng, 40, 2400)]
    else:
        n = _log(rng, 1, 24)
        top = min(32768, 500000 // (n * shape["hk"]))
        low = _log(rng, 64, top // 2)
        histories, chunks = [rng.randint(low, top) for _ in range(n)], [rng.randint(1, 5)] * n
    case = dict(shape, kind=kind, histories=_text(histories), chunks=_text(chunks), **score)
    while 4 * case["d"] * case["hq"] * _pairs(case) > 8.5e10:
        chunks[0] = chunks[0] * 2 // 3
        case["chunks"] = _text(chunks)
    return case


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
    rotated vectors (K slot: four fp16 constants, codes from byte 32; V slot: codes)."""
    k, v = cache_k.view(torch.uint8).view(-1, cache_k.shape[-1]), cache_v.view(torch.uint8).view(-1, cache_v.shape[-1])
    shifts = torch.tensor([1, 4, 16, 64], device=k.device)
    for a in range(0, k.shape[0], 1 << 16):
        b = min(a + (1 << 16), k.shape[0])
        meta = []
        for slots, at in ((k, 32), (v, 0)):
            y = torch.randn(b - a, d, generator=gen, device=k.device) * 1.4
            low, high = y.amin(1, keepdim=True), y.amax(1, keepdim=True)
            scale, zero = ((high - low) / 3).half(), low.half()
            codes = ((y - zero.float()) / scale.float() + 0.5).floor().clamp(0, 3).to(torch.int64)
            slots[a:b, at:at + d // 4] = (codes.view(b - a, d // 4, 4) * shifts).sum(-1).to(torch.uint8)
            meta += [scale, zero]
        k[a:b, :8] = torch.cat(meta, 1).contiguous().view(torch.uint8)


def _read(cache_k, cache_v, d, slots):
    """The fp32 K and V values of cache slots (any shape of token slots, all KV heads)."""
    hk = cache_k.shape[2]
    k = cache_k.view(torch.uint8).view(-1, hk, cache_k.shape[-1])[slots]
    v = cache_v.view(torch.uint8).view(-1, hk, cache_v.shape[-1])[slots]
    meta = k[..., :8].contiguous().view(torch.float16).float()
    shifts = torch.tensor([0, 2, 4, 6], dtype=torch.uint8, device=k.device)
    out = []
    for x, s, z in ((k[..., 32:32 + d // 4], meta[..., 0:1], meta[..., 1:2]), (v[..., :d // 4], meta[..., 2:3], meta[..., 3:4])):
        codes = ((x[..., None] >> shifts) & 3).reshape(*x.shape[:-1], d).float()
        out.append(codes * s + z)
    return out


def _last_of(seats):
    """Indexes of the last occurrence of each seat, ascending."""
    _, first = np.unique(seats[::-1], return_index=True)
    return np.sort(len(seats) - 1 - first)


def _slopes(hq):
    """The geometric slopes of a distance bias: 2^(-8 (h + 1) / hq)."""
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / hq) for h in range(hq)], dtype=torch.float32, device=_device())


def _paged(case, lengths, gen, seed, spare=8):
    """Filled caches, their window arena and a block table of permuted pages."""
    dev, d, hk = _device(), case["d"], case["hk"]
    pages = [-(-n // BLOCK) for n in lengths]
    blocks = sum(pages) + spare
    order = np.random.default_rng(seed).permutation(blocks).astype(np.int32)
    table = np.zeros((len(pages), max(pages)), np.int32)
    at = 0
    for r, p in enumerate(pages):
        table[r, :p] = order[at:at + p]
        at += p
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
    for arena, y in zip((x["stage_k"], x["stage_v"]), _read(x["k_cache"], x["v_cache"], d, slot)):
        spread = y.amax(-1, keepdim=True) - y.amin(-1, keepdim=True)
        noise = torch.rand(y.shape, generator=gen, device=dev) - 0.5
        arena.view(rows * BLOCK, hk, d)[seat] = y + noise * spread / 3
    x["owner"].view(-1)[seat] = slot // BLOCK


def _inputs(case, seed):
    """Everything a call reads, from the seed alone, as a dict of tensors and host lists."""
    dev = _device()
    gen = torch.Generator(device=dev).manual_seed(seed)
    hq, hk, d, dtype = case["hq"], case["hk"], case["d"], KINDS[case["dtype"]]
    if case["kind"] == "norm_rope":
        n, rotary = case["tokens"], case["rotary"]
        # the projection's output: one row per token, queries, keys and values side by side
        row = torch.randn(n, (hq + 2 * hk) * d, generator=gen, device=dev) * 2
        row[:, ::37] *= 6
        row = row.to(dtype)
        inv = 1e6 ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device=dev) / rotary)
        angle = torch.arange(32768, dtype=torch.float64, device=dev)[:, None] * inv
        weight = [(torch.randn(d, generator=gen, device=dev) * 0.2 + 1 - case["offset"]).to(dtype) for _ in "qk"]
        # some requests' tokens, each at its own position
        positions = torch.arange(n, device=dev) + int(torch.randint(0, 32768 - n, (1,), generator=gen, device=dev))
        return dict(q=row[:, :hq * d].view(n, hq, d), k=row[:, hq * d:(hq + hk) * d].view(n, hk, d), positions=positions,
                    cos_sin=torch.cat([angle.cos(), angle.sin()], 1).float().contiguous(), q_weight=weight[0],
                    k_weight=weight[1], q_out=torch.empty(n, hq, d, dtype=dtype, device=dev),
                    k_out=torch.empty(n, hk, d, dtype=dtype, device=dev))
    if case["kind"] == "evict":
        lengths, drops = _numbers(case["lengths"]), _numbers(case["drops"])
        x = _paged(case, lengths, gen, seed)
        _stage_last(x, case, lengths, gen)
        weights = torch.rand(len(lengths), hk, max(lengths) + 100, generator=gen, device=dev) ** 8
        if case["coarse"]:  # many ties
            weights = (weights * 64).floor() / 64
        return dict(x, weights=weights, weights_out=torch.empty_like(weights), lengths=lengths, drops=drops)
    histories, chunks = _numbers(case["histories"]), _numbers(case["chunks"])
    lengths = [h + c for h, c in zip(histories, chunks)]
    n = sum(chunks)
    x = _paged(case, lengths, gen, seed)
    _stage_last(x, case, histories, gen)

    def rows(heads, scale):
        return (torch.randn(n, heads, d, generator=gen, device=dev) * scale).to(dtype)

    starts = [0] + np.cumsum(chunks).tolist()
    x.update(q=rows(hq, 2.5), k=rows(hk, 1.4), v=rows(hk, 1.4), rv=_rotation(d, gen), starts=starts, lengths=lengths,
             histories=histories, chunks=chunks, slopes=_slopes(hq) if case["alibi"] else None)
    x["dev_histories"] = torch.tensor(histories, device=dev)
    x["dev_chunks"] = torch.tensor(chunks, device=dev)
    x["dev_starts"] = torch.tensor(starts[:-1], device=dev)
    if case["kind"] == "weights":
        scores, _ = _scores(dict(x, **_fields(case)), values=False)
        lse = torch.logsumexp(scores, -1)
        x["lse"] = _unpadded(x, lse.view(*lse.shape[:2], max(chunks), hq // hk), hq).contiguous()
        x["weights"] = torch.rand(len(lengths), hk, max(lengths) + 100, generator=gen, device=dev) * 1e-3
    return x


def _fields(case):
    return {k: case[k] for k in ("kind", "hq", "hk", "d", "dtype", "cap")}


def prepare(case, seed):
    x = _inputs(case, seed)
    kind = case["kind"]
    if kind == "norm_rope":
        return dict(x, kind=kind, rotary=case["rotary"], offset=case["offset"], interleaved=case["interleaved"])
    state = dict(x, kind=kind, hq=case["hq"], hk=case["hk"], d=case["d"], dtype=case["dtype"], cap=case.get("cap", 0.0))
    state["stage"] = (x["stage_k"], x["stage_v"], x["owner"])
    if own and kind != "prompt":
        # the batch's plan, which a model's layers share (the caches, weights and inputs are each layer's own)
        from oscar_amd import ops

        dev = x["table"].device
        if kind == "decode":
            state["plan"] = ops.plan_decode(x["starts"], x["lengths"], has_new=True, num_kv_heads=case["hk"],
                                            group=case["hq"] // case["hk"], head_dim=case["d"], device=dev,
                                            window=(0, RECENT))
        elif kind == "weights":
            state["plan"] = ops.plan_weights(x["starts"], x["lengths"], has_new=True, device=dev)
        else:
            state["plan"] = ops.plan_evict(x["lengths"], x["drops"], block_size=BLOCK, sink_tokens=SINK,
                                           recent_tokens=RECENT, device=dev)
    return state


# ---------------------------------------------------------------- the plain forms
def _plain_norm_rope(s):
    n, r = s["q"].shape[0], s["rotary"]
    table = s["cos_sin"][s["positions"]]
    cos, sin = table[:, None, :r // 2], table[:, None, r // 2:]

    def rows(x, weight):
        y = x.float()
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * (weight.float() + s["offset"])
        a, b = (y[..., 0:r:2], y[..., 1:r:2]) if s["interleaved"] else (y[..., :r // 2], y[..., r // 2:r])
        a, b = a * cos - b * sin, b * cos + a * sin
        turned = torch.stack([a, b], -1).reshape(n, -1, r) if s["interleaved"] else torch.cat([a, b], -1)
        return torch.cat([turned, y[..., r:]], -1).to(x.dtype)

    return dict(q=rows(s["q"], s["q_weight"]), k=rows(s["k"], s["k_weight"]))


def _unpadded(s, x, hq):
    """Padded rows [requests, hk, tokens, group, ...] as the batch's rows [n, hq, ...]."""
    x = x.transpose(1, 2).reshape(x.shape[0], x.shape[2], hq, *x.shape[4:])
    return x[torch.arange(x.shape[1], device=x.device) < s["dev_chunks"][:, None]]


def _scores(s, values=True):
    """Masked scores [requests, hk, tokens * group, keys] of a batch padded to its longest
    request, and the values [requests, hk, keys, d]."""
    d, hk, group, dtype = s["d"], s["hk"], s["hq"] // s["hk"], KINDS[s["dtype"]]
    dev, rows = s["table"].device, s["owner"].shape[0]
    hist, count, start = s["dev_histories"][:, None], s["dev_chunks"][:, None], s["dev_starts"][:, None]
    most, tokens = max(s["lengths"]), max(s["chunks"])
    pos = torch.arange(most, device=dev)
    block = s["table"].long()[:, pos // BLOCK]
    seat = block % rows * BLOCK + pos % BLOCK
    new = (start + (pos - hist).clamp(0)).clamp(max=s["q"].shape[0] - 1)
    is_new = (pos >= hist)[..., None, None]
    staged = (s["owner"].view(-1)[seat] == block)[..., None, None]
    out = []
    stored = _read(s["k_cache"], s["v_cache"], d, block * BLOCK + pos % BLOCK)
    for name, old, arena in (("k", stored[0], s["stage_k"]), ("v", stored[1], s["stage_v"]))[:2 if values else 1]:
        # a history value is fp16(x), and of the activations' type for keys and in a prompt
        old = torch.where(staged, arena.view(-1, hk, d)[seat], old).half()
        old = old.to(dtype) if name == "k" or s["kind"] == "prompt" else old
        out.append(torch.where(is_new, s[name][new].float(), old.float()).transpose(1, 2))
    query = (start + torch.arange(tokens, device=dev)).clamp(max=s["q"].shape[0] - 1)
    q = s["q"][query].float().view(len(s["lengths"]), tokens, hk, group, d).transpose(1, 2).reshape(-1, hk, tokens * group, d)
    x = q @ out[0].transpose(-1, -2) * d ** -0.5
    if s["cap"]:
        x = s["cap"] * torch.tanh(x / s["cap"])
    at = hist + torch.arange(tokens, device=dev)  # the position of each query
    if s["slopes"] is not None:
        distance = (pos - at[..., None]).float()[:, None, :, None]
        x = (x.view(-1, hk, tokens, group, most) + s["slopes"].view(hk, 1, group, 1) * distance).view_as(x)
    seen = pos <= at[..., None]
    seen = seen & (torch.arange(tokens, device=dev) < count)[..., None]
    x = torch.where(seen[:, None].repeat_interleave(group, 2), x, -math.inf)
    return x, out[1] if values else None


def _plain_attention(s):
    x, v = _scores(s)
    top = x.amax(-1, keepdim=True).clamp(min=-1e30)
    x = torch.exp(x - top)
    total = x.sum(-1, keepdim=True)
    out = (x @ v) / total
    tokens, group = max(s["chunks"]), s["hq"] // s["hk"]
    out = _unpadded(s, out.view(*out.shape[:2], tokens, group, s["d"]), s["hq"])
    lse = top + torch.log(total)
    lse = _unpadded(s, lse.view(*lse.shape[:2], tokens, group), s["hq"])
    if s["kind"] == "prompt" and s["histories"] == [0]:
        return dict(out=out.to(KINDS[s["dtype"]]))
    return dict(out=(out @ s["rv"].t()).to(KINDS[s["dtype"]]), lse=lse)


def _plain_weights(s):
    x, _ = _scores(s, values=False)
    tokens, group = max(s["chunks"]), s["hq"] // s["hk"]
    at = s["dev_starts"][:, None] + torch.arange(tokens, device=x.device)
    lse = s["lse"][at.clamp(max=s["lse"].shape[0] - 1)].view(-1, tokens, s["hk"], group).transpose(1, 2)
    s["weights"][..., :x.shape[-1]] += torch.exp(x - lse.reshape(x.shape[0], s["hk"], -1, 1)).sum(2)
    return dict(weights=s["weights"])


def _plain_evict(s):
    """Of the tokens [SINK, tail) those of least weight go; the kept ones behind the new end
    take the places of the dropped ones before it, both in ascending order.  The weights
    follow, zero behind the new length."""
    w, dev, hk = s["weights"], s["weights"].device, s["hk"]
    length = torch.tensor(s["lengths"], device=dev)
    drop = torch.tensor(s["drops"], device=dev)[:, None] * BLOCK
    tail = (((length - RECENT).clamp(min=0) // BLOCK) * BLOCK)[:, None]
    end = tail - drop
    pos = torch.arange(w.shape[-1], device=dev)
    middle = (pos >= SINK) & (pos < tail)
    order = torch.sort(torch.where(middle[:, None], w, -math.inf), descending=True, stable=True).indices
    rank = torch.empty_like(order).scatter_(-1, order, pos.expand_as(order))
    kept = middle[:, None] & (rank < (tail - SINK - drop)[:, None])
    hole = middle[:, None] & ~kept & (pos < end)[:, None]
    mover = kept & (pos >= end)[:, None]
    r, h, to = hole.nonzero(as_tuple=True)
    r2, h2, at = mover.nonzero(as_tuple=True)  # as many per request and head, in the same order
    # behind the new end: the tail, then zeros
    source = torch.where(pos < end, pos, pos + drop).clamp(max=w.shape[-1] - 1)
    out = torch.gather(w, -1, source[:, None].expand(w.shape))
    out[r, h, to] = w[r2, h2, at]
    out = torch.where((pos < length[:, None] - drop)[:, None], out, 0.0)
    block = s["table"].long()
    for cache, at_byte, many in ((s["k_cache"], 0, 8), (s["k_cache"], 32, s["d"] // 4), (s["v_cache"], 0, s["d"] // 4)):
        part = cache[..., at_byte:at_byte + many]
        part[block[r, to // BLOCK], to % BLOCK, h] = part[block[r2, at // BLOCK], at % BLOCK, h2]
    # a written slot loses its window copy
    rows, taken = s["owner"].shape[0], block[r, to // BLOCK]
    seat = taken % rows * BLOCK + to % BLOCK
    flat = s["owner"].view(-1)
    mine = torch.zeros_like(flat, dtype=torch.bool)
    mine[seat[flat[seat] == taken]] = True
    flat[mine] = -1
    return dict(weights=out, k_cache=s["k_cache"], v_cache=s["v_cache"], owner=s["owner"])


def run(state):
    s, kind = state, state["kind"]
    if not own:
        if kind == "norm_rope":
            return _plain_norm_rope(s)
        return {"weights": _plain_weights, "evict": _plain_evict}.get(kind, _plain_attention)(s)
    from oscar_amd import ops

    if kind == "norm_rope":
        q, k = ops.norm_rope(s["q"], s["k"], s["positions"], s["cos_sin"], q_weight=s["q_weight"], k_weight=s["k_weight"],
                             eps=EPS, weight_offset=s["offset"], interleaved=s["interleaved"], q_out=s["q_out"],
                             k_out=s["k_out"])
        return dict(q=q, k=k)
    scale = s["d"] ** -0.5
    if kind == "evict":
        weights = ops.evict(s["plan"], s["weights"], s["k_cache"], s["v_cache"], s["table"], head_dim=s["d"],
                            stage=s["stage"], weights_out=s["weights_out"])
        return dict(weights=weights, k_cache=s["k_cache"], v_cache=s["v_cache"], owner=s["owner"])
    score = dict(soft_cap=s["cap"], alibi_slopes=s["slopes"])
    if kind == "weights":
        ops.accumulate_weights(s["q"], s["k"], s["k_cache"], s["v_cache"], s["table"], s["plan"], scale, s["lse"],
                               s["weights"], s["stage"], head_dim=s["d"], **score)
        return dict(weights=s["weights"])
    if kind == "decode":
        out, lse = ops.attention_decode(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["table"], s["plan"], scale,
                                        s["stage"], head_dim=s["d"], **score)
    elif s["histories"] == [0]:
        return dict(out=ops.attention_prefill(s["q"], s["k"], s["v"], scale, head_dim=s["d"], **score))
    else:
        lse = torch.empty(s["q"].shape[:2], dtype=torch.float32, device=s["q"].device)
        out = ops.attention_prefill(s["q"], s["k"], s["v"], scale, head_dim=s["d"], history=s["histories"][0],
                                    k_cache=s["k_cache"], v_cache=s["v_cache"], block_table_row=s["table"][0],
                                    stage=s["stage"], lse=lse, **score)
    return dict(out=ops.rotate(out, s["rv"], transpose=True, out_dtype=s["q"].dtype), lse=lse)


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    d, hq, hk, kind = case["d"], case["hq"], case["hk"], case["kind"]
    size = {"bf16": 2, "fp16": 2, "fp32": 4}[case["dtype"]]
    if kind == "norm_rope":
        n = case["tokens"]
        return dict(bytes=n * ((hq + hk) * d * size * 2 + 8 + 4 * case["rotary"]) + 2 * d * size,
                    flops=n * (hq + hk) * (4 * d + 3 * case["rotary"]))
    slot = 8 + d // 2
    if kind == "evict":
        total = 0.0
        for length, pages in zip(_numbers(case["lengths"]), _numbers(case["drops"])):
            tail = (length - RECENT) // BLOCK * BLOCK
            middle, drop = tail - SINK, pages * BLOCK
            # every weight is read and written; the dropped tokens' share of kept ones moves
            total += hk * (8 * length + drop * (1 - drop / middle) * 2 * slot) + 4 * (length // BLOCK)
        return dict(bytes=total, flops=0)
    histories, chunks = _numbers(case["histories"]), _numbers(case["chunks"])
    n = sum(chunks)
    if kind == "weights":
        total = n * (hq * d * size + hq * 4 + hk * d * size)
        for h, c in zip(histories, chunks):
            staged = min(h, RECENT)
            total += hk * ((h - staged) * (8 + d // 4) + staged * 4 * d + 8 * (h + c))
        return dict(bytes=total, flops=2 * d * hq * _pairs(case))
    total = n * (2 * hq * d * size + 2 * hk * d * size)
    cached = 0
    for h, c in zip(histories, chunks):
        staged = min(h, RECENT)
        total += hk * ((h - staged) * slot + staged * 8 * d)
        cached += c if kind == "decode" or h else 0
    return dict(bytes=total + cached * hq * 4 + (4 * d * d if cached else 0),
                flops=4 * d * hq * _pairs(case) + 2 * d * d * cached * hq)


# ---------------------------------------------------------------- 64 bits
def _exact_norm_rope(case, x):
    n, r, p = case["tokens"], case["rotary"], x["positions"]
    table = x["cos_sin"].double()[p]
    unit = torch.complex(table[:, :r // 2], table[:, r // 2:])[:, None]
    out = {}
    for name in "qk":
        y = x[name].double()
        y = y / (y.pow(2).sum(-1, keepdim=True) / case["d"] + EPS).sqrt() * (x[name + "_weight"].double() + case["offset"])
        if case["interleaved"]:
            z = torch.view_as_complex(y[..., :r].reshape(n, -1, r // 2, 2).contiguous()) * unit
            y[..., :r] = torch.view_as_real(z).reshape(n, -1, r)
        else:
            z = torch.complex(y[..., :r // 2].contiguous(), y[..., r // 2:r].contiguous()) * unit
            y[..., :r] = torch.cat([z.real, z.imag], -1)
        out[name] = y
    return out


def _exact_request(case, x, r):
    """Keys and values [length, hk, d] of request r, in 64 bits."""
    h, c, a = x["histories"][r], x["chunks"][r], x["starts"][r]
    dtype, rows = KINDS[case["dtype"]], x["owner"].shape[0]
    pos = np.arange(h)
    block = torch.from_numpy(x["host_table"][r, pos // BLOCK].astype(np.int64)).to(x["owner"].device)
    off = torch.from_numpy(pos % BLOCK).to(block.device)
    mine = (x["owner"][block % rows, off] == block)[:, None, None]
    got = []
    for old, arena, new, narrow in zip(_read(x["k_cache"], x["v_cache"], case["d"], block * BLOCK + off),
                                       (x["stage_k"], x["stage_v"]), (x["k"], x["v"]), (True, case["kind"] == "prompt")):
        old = torch.where(mine, arena[block % rows, off], old).half()
        got.append(torch.cat([(old.to(dtype) if narrow else old).double(), new[a:a + c].double()]))
    return got


def _exact_scores(case, x, r, head, keys, a, b):
    """Masked scores of queries [a, b) of request r and one head, in 64 bits."""
    h = x["histories"][r]
    q = x["q"][x["starts"][r] + a:x["starts"][r] + b, head].double()
    s = q @ keys.t().contiguous() * case["d"] ** -0.5
    if case["cap"]:
        s = torch.tanh(s / case["cap"]) * case["cap"]
    distance = torch.arange(keys.shape[0], device=s.device)[None] - (h + torch.arange(a, b, device=s.device))[:, None]
    if case["alibi"]:
        s += x["slopes"][head].double() * distance
    return s.masked_fill(distance > 0, -math.inf)


def _exact_batch(case, x):
    hq, hk, d = case["hq"], case["hk"], case["d"]
    group, weights = hq // hk, case["kind"] == "weights"
    out = torch.empty(x["q"].shape, dtype=torch.float64, device=x["q"].device)
    lse = torch.empty(out.shape[:2], dtype=torch.float64, device=out.device)
    added = x["weights"].double() if weights else None
    for r, c in enumerate(x["chunks"]):
        keys, values = _exact_request(case, x, r)
        start = x["starts"][r]
        for head in range(hq):
            k = keys[:, head // group].contiguous()
            for a in range(0, c, 1024):
                b = min(a + 1024, c)
                s = _exact_scores(case, x, r, head, k, a, b)
                if weights:
                    p = torch.exp(s - x["lse"][start + a:start + b, head, None].double())
                    added[r, head // group, :p.shape[1]] += p.sum(0)
                    continue
                lse[start + a:start + b, head] = torch.logsumexp(s, -1)
                out[start + a:start + b, head] = torch.softmax(s, -1) @ values[:, head // group].contiguous()
    if weights:
        return dict(weights=added)
    if case["kind"] == "prompt" and x["histories"] == [0]:
        return dict(out=out)
    return dict(out=out @ x["rv"].double().t().contiguous(), lse=lse)


def _exact_evict(case, x):
    w = x["weights"].double().cpu().numpy()
    for r, (length, pages) in enumerate(zip(x["lengths"], x["drops"])):
        tail = (length - RECENT) // BLOCK * BLOCK
        end, many = tail - pages * BLOCK, pages * BLOCK
        for head in range(case["hk"]):
            row = w[r, head]
            # the least first; of equal ones the last first
            middle = np.arange(SINK, tail)
            gone = set(middle[np.lexsort((-middle, row[SINK:tail]))][:many].tolist())
            holes = sorted(p for p in gone if p < end)
            kept = [p for p in range(end, tail) if p not in gone]
            row[holes] = row[kept]
            rest = row[tail:length].copy()
            row[end:] = 0
            row[end:end + rest.size] = rest
    return dict(weights=torch.from_numpy(w), k_cache=None, v_cache=None, owner=None)


def exact(case, seed):
    x = _inputs(case, seed)
    return {"norm_rope": _exact_norm_rope, "evict": _exact_evict}.get(case["kind"], _exact_batch)(case, x)
