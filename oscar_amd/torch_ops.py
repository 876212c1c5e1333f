"""The C-ABI entry points as torch operators (``torch.ops.oscar_amd.*``).

Each operator calls the same library entry point as :mod:`oscar_amd.ops` and carries a
fake (meta) implementation, so the calls are visible to torch: schema-checked, traced
by ``torch.compile`` / ``torch.fx`` with the right output shapes and mutated inputs,
and dispatched on the CUDA (HIP) key only.  A nonzero status raises, as the direct
wrappers do.

Operators (tensors in the layouts of the C structs; optional staging tensors are the
layer's FP32 window arena):

* ``rotate(x, r, transpose) -> Tensor``: x @ R or x @ R^T in x's dtype
  (``oscar_rotate_v1``; backend.py:371,382).
* ``store(key, value, k_cache!, v_cache!, slot_mapping, stage_k!, stage_v!, owner!,
  head_dim, rk, rv, k_clip, v_clip, stage_mode, query_start_loc, seq_lens,
  recent_tokens, sink_tokens_eff) -> ()``: the write path (``oscar_store_v1``;
  store_kernel.py:54-102, backend.py:130-198,513-555); the arena tensors are passed
  (None without a window) because they are mutated.
* ``attention_decode(q, k_new, v_new, k_cache, v_cache, block_table, query_start_loc,
  seq_lens, scale, head_dim, stage_k, stage_v, owner, sink_tokens_eff, recent_tokens,
  soft_cap, alibi_slopes) -> (out_rot, lse)``: plan + split-K decode + merge
  (``oscar_attn_plan_v1`` / ``oscar_attn_decode_v1``; slab_attention.py:23-92,376-476); the request lists are
  host integers.
* ``attention_prefill(q, k, v, scale, head_dim, history, k_cache, v_cache,
  block_table_row, stage_k, stage_v, owner, soft_cap, alibi_slopes) -> (out, lse)``:
  fresh-only (history 0, output in q's dtype, lse empty) or continuation prefill (fp32 rotated output and LSE)
  (``oscar_attn_prefill_v1``; prefill.py:69-72, slab_attention.py:376-476).
* ``norm_rope(q, k, positions, cos_sin, q_weight, k_weight, eps, weight_offset,
  interleaved) -> (q, k)``: head norms with the position rotation (``oscarop_norm_rope_v1``).
* ``accumulate_weights(q, k_new, k_cache, v_cache, block_table, query_start_loc, seq_lens,
  scale, lse, weights!, head_dim, stage_k, stage_v, owner, soft_cap, alibi_slopes) -> ()``:
  the attention weight each cached token received (``oscarop_attn_weights_v1``); the request
  lists are host integers.
* ``evict(weights, k_cache!, v_cache!, block_table, seq_lens, drop_pages, stage_k, stage_v,
  owner!, head_dim, sink_tokens, recent_tokens) -> weights``: drops the tokens of
  least weight, whole pages at a time (``oscarop_evict_v1``).
* ``map_slots(pool_pages, pool_count!, block_table!, lengths, counts, tokens, block_size,
  keep) -> (query_start_loc, seq_lens, slots, positions, granted)``: a step's pages, slots and
  positions from lengths on the device (``oscarop_map_v1``); ``release_pages(pool_pages!,
  pool_count!, block_table, lengths, new_lengths, block_size) -> ()``: pages behind the new
  lengths back to the pool (``oscarop_release_v1``).
* ``tree_mask(parents, query_start_loc, max_nodes) -> (mask, depths)``: ancestors of drafted
  nodes (``oscarop_tree_mask_v1``); ``attention_tree(q, k_new, v_new, k_cache, v_cache,
  block_table, query_start_loc, seq_lens, mask, scale, head_dim, stage_k, stage_v, owner,
  soft_cap) -> (out_rot, lse)``: their attention (``oscarop_tree_plan_v1`` /
  ``oscarop_attn_tree_v1``).
* ``page_bounds(k_cache, bounds!, block_table, lengths, seq_lens, max_new, head_dim) -> ()``: the
  least and the largest keys of the pages that a step touched (``oscarop_page_bounds_v1``);
  ``attention_selected(q, k_new, v_new, k_cache, v_cache, bounds, block_table,
  query_start_loc, seq_lens, budget, scale, head_dim, first_pages, last_pages, stage_k,
  stage_v, owner, sink_tokens_eff, recent_tokens, soft_cap) -> (out_rot, lse, pages)``: the
  choice of pages and the attention over them (``oscarop_select_v1`` /
  ``oscarop_attn_selected_v1``).
"""
from __future__ import annotations

import torch

from . import ops

_LIB = "oscar_amd"


def _stage(stage_k, stage_v, owner):
    if stage_k is None and stage_v is None and owner is None:
        return None
    if stage_k is None or stage_v is None or owner is None:
        raise ValueError("the window arena needs stage_k, stage_v and owner together")
    return (stage_k, stage_v, owner)


# ------------------------------------------------------------------ rotate
@torch.library.custom_op(f"{_LIB}::rotate", mutates_args=(), device_types="cuda")
def rotate(x: torch.Tensor, r: torch.Tensor, transpose: bool = False) -> torch.Tensor:
    return ops.rotate(x, r, transpose=transpose)


@rotate.register_fake
def _(x, r, transpose=False):
    return torch.empty_like(x)


# ------------------------------------------------------------------ store
@torch.library.custom_op(f"{_LIB}::store", mutates_args=("k_cache", "v_cache", "stage_k", "stage_v", "owner"),
                         device_types="cuda")
def store(key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
          slot_mapping: torch.Tensor, stage_k: torch.Tensor | None, stage_v: torch.Tensor | None,
          owner: torch.Tensor | None, head_dim: int, rk: torch.Tensor | None = None,
          rv: torch.Tensor | None = None, k_clip: float = 0.0, v_clip: float = 0.0, stage_mode: int = 0,
          query_start_loc: torch.Tensor | None = None, seq_lens: torch.Tensor | None = None,
          recent_tokens: int = 0, sink_tokens_eff: int = 0) -> None:
    num_reqs = 0 if seq_lens is None else int(seq_lens.numel())
    ops.store(key, value, k_cache, v_cache, slot_mapping, head_dim=head_dim, rk=rk, rv=rv,
              k_clip=k_clip, v_clip=v_clip, stage=_stage(stage_k, stage_v, owner), stage_mode=stage_mode,
              qsl_dev=query_start_loc, seqs_dev=seq_lens, num_reqs=num_reqs,
              recent_tokens=recent_tokens, sink_tokens_eff=sink_tokens_eff)


@store.register_fake
def _(key, value, k_cache, v_cache, slot_mapping, stage_k, stage_v, owner, head_dim, rk=None, rv=None,
      k_clip=0.0, v_clip=0.0, stage_mode=0, query_start_loc=None, seq_lens=None, recent_tokens=0,
      sink_tokens_eff=0):
    return None


# ------------------------------------------------------------------ decode
@torch.library.custom_op(f"{_LIB}::attention_decode", mutates_args=(), device_types="cuda")
def attention_decode(q: torch.Tensor, k_new: torch.Tensor | None, v_new: torch.Tensor | None,
                     k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                     query_start_loc: list[int], seq_lens: list[int], scale: float, head_dim: int,
                     stage_k: torch.Tensor | None = None, stage_v: torch.Tensor | None = None,
                     owner: torch.Tensor | None = None, sink_tokens_eff: int = 0,
                     recent_tokens: int = 0, soft_cap: float = 0.0,
                     alibi_slopes: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    hq, hk = q.shape[1], k_cache.shape[2]
    stage = _stage(stage_k, stage_v, owner)
    window = (sink_tokens_eff, recent_tokens) if stage is not None else (0, 0)
    plan = ops.plan_decode(list(query_start_loc), list(seq_lens), has_new=k_new is not None,
                           num_kv_heads=hk, group=hq // hk, head_dim=head_dim, device=q.device, window=window)
    return ops.attention_decode(q, k_new, v_new, k_cache, v_cache, block_table, plan, scale, stage,
                                head_dim=head_dim, soft_cap=soft_cap, alibi_slopes=alibi_slopes)


@attention_decode.register_fake
def _(q, k_new, v_new, k_cache, v_cache, block_table, query_start_loc, seq_lens, scale, head_dim,
      stage_k=None, stage_v=None, owner=None, sink_tokens_eff=0, recent_tokens=0, soft_cap=0.0, alibi_slopes=None):
    n, hq = q.shape[0], q.shape[1]
    return (q.new_empty((n, hq, head_dim), dtype=torch.float32), q.new_empty((n, hq), dtype=torch.float32))


# ------------------------------------------------------------------ prefill
@torch.library.custom_op(f"{_LIB}::attention_prefill", mutates_args=(), device_types="cuda")
def attention_prefill(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float, head_dim: int,
                      history: int = 0, k_cache: torch.Tensor | None = None,
                      v_cache: torch.Tensor | None = None, block_table_row: torch.Tensor | None = None,
                      stage_k: torch.Tensor | None = None, stage_v: torch.Tensor | None = None,
                      owner: torch.Tensor | None = None, soft_cap: float = 0.0,
                      alibi_slopes: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    n, hq = q.shape[0], q.shape[1]
    lse = torch.empty((n, hq) if history > 0 else (0,), dtype=torch.float32, device=q.device)
    out = ops.attention_prefill(q, k, v, scale, head_dim=head_dim, history=history, k_cache=k_cache,
                                v_cache=v_cache, block_table_row=block_table_row,
                                stage=_stage(stage_k, stage_v, owner), lse=lse if history > 0 else None,
                                soft_cap=soft_cap, alibi_slopes=alibi_slopes)
    return out, lse


@attention_prefill.register_fake
def _(q, k, v, scale, head_dim, history=0, k_cache=None, v_cache=None, block_table_row=None,
      stage_k=None, stage_v=None, owner=None, soft_cap=0.0, alibi_slopes=None):
    n, hq = q.shape[0], q.shape[1]
    if history > 0:
        return (q.new_empty((n, hq, head_dim), dtype=torch.float32), q.new_empty((n, hq), dtype=torch.float32))
    return q.new_empty((n, hq, head_dim)), q.new_empty((0,), dtype=torch.float32)


# ------------------------------------------------------------------ head norms and rotation
@torch.library.custom_op(f"{_LIB}::norm_rope", mutates_args=(), device_types="cuda")
def norm_rope(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, cos_sin: torch.Tensor,
              q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None, eps: float = 1e-6,
              weight_offset: float = 0.0, interleaved: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    return ops.norm_rope(q, k, positions, cos_sin, q_weight=q_weight, k_weight=k_weight, eps=eps,
                         weight_offset=weight_offset, interleaved=interleaved)


@norm_rope.register_fake
def _(q, k, positions, cos_sin, q_weight=None, k_weight=None, eps=1e-6, weight_offset=0.0, interleaved=False):
    return q.new_empty(q.shape), k.new_empty(k.shape)


# ------------------------------------------------------------------ accumulated weights, eviction
@torch.library.custom_op(f"{_LIB}::accumulate_weights", mutates_args=("weights",), device_types="cuda")
def accumulate_weights(q: torch.Tensor, k_new: torch.Tensor | None, k_cache: torch.Tensor, v_cache: torch.Tensor,
                       block_table: torch.Tensor, query_start_loc: list[int], seq_lens: list[int], scale: float,
                       lse: torch.Tensor, weights: torch.Tensor, head_dim: int, stage_k: torch.Tensor | None = None,
                       stage_v: torch.Tensor | None = None, owner: torch.Tensor | None = None, soft_cap: float = 0.0,
                       alibi_slopes: torch.Tensor | None = None) -> None:
    plan = ops.plan_weights(query_start_loc, seq_lens, has_new=k_new is not None, device=q.device)
    ops.accumulate_weights(q, k_new, k_cache, v_cache, block_table, plan, scale, lse, weights,
                           _stage(stage_k, stage_v, owner), head_dim=head_dim, soft_cap=soft_cap, alibi_slopes=alibi_slopes)


@accumulate_weights.register_fake
def _(q, k_new, k_cache, v_cache, block_table, query_start_loc, seq_lens, scale, lse, weights, head_dim, stage_k=None,
      stage_v=None, owner=None, soft_cap=0.0, alibi_slopes=None):
    return None


@torch.library.custom_op(f"{_LIB}::evict", mutates_args=("k_cache", "v_cache", "owner"), device_types="cuda")
def evict(weights: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
          seq_lens: list[int], drop_pages: list[int], stage_k: torch.Tensor | None, stage_v: torch.Tensor | None,
          owner: torch.Tensor | None, head_dim: int, sink_tokens: int = 0, recent_tokens: int = 0) -> torch.Tensor:
    plan = ops.plan_evict(seq_lens, drop_pages, block_size=k_cache.shape[1], sink_tokens=sink_tokens,
                          recent_tokens=recent_tokens, device=weights.device)
    return ops.evict(plan, weights, k_cache, v_cache, block_table, head_dim=head_dim,
                     stage=_stage(stage_k, stage_v, owner))


@evict.register_fake
def _(weights, k_cache, v_cache, block_table, seq_lens, drop_pages, stage_k, stage_v, owner, head_dim, sink_tokens=0,
      recent_tokens=0):
    return weights.new_empty(weights.shape)


# ------------------------------------------------------------------ pages and slots
@torch.library.custom_op(f"{_LIB}::map_slots", mutates_args=("pool_count", "block_table"), device_types="cuda")
def map_slots(pool_pages: torch.Tensor, pool_count: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor,
              counts: torch.Tensor, tokens: int, block_size: int,
              keep: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    m = ops.map_slots(ops.PagePool(pool_pages, pool_count), block_table, lengths, counts, tokens=tokens, block_size=block_size,
                      keep=keep)
    # (outputs of an operator share no memory)
    return m.qsl, m.seq_lens.clone(), m.slots, m.positions.clone(), m.granted


@map_slots.register_fake
def _(pool_pages, pool_count, block_table, lengths, counts, tokens, block_size, keep=None):
    reqs = lengths.shape[0]
    return (lengths.new_empty(reqs + 1), lengths.new_empty(reqs), lengths.new_empty(tokens, dtype=torch.int64),
            lengths.new_empty(tokens, dtype=torch.int64), lengths.new_empty(reqs, dtype=torch.bool))


@torch.library.custom_op(f"{_LIB}::release_pages", mutates_args=("pool_pages", "pool_count"), device_types="cuda")
def release_pages(pool_pages: torch.Tensor, pool_count: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor,
                  new_lengths: torch.Tensor, block_size: int) -> None:
    ops.release_pages(ops.PagePool(pool_pages, pool_count), block_table, lengths, new_lengths, block_size=block_size)


@release_pages.register_fake
def _(pool_pages, pool_count, block_table, lengths, new_lengths, block_size):
    return None


# ------------------------------------------------------------------ drafted trees
@torch.library.custom_op(f"{_LIB}::tree_mask", mutates_args=(), device_types="cuda")
def tree_mask(parents: torch.Tensor, query_start_loc: torch.Tensor, max_nodes: int) -> tuple[torch.Tensor, torch.Tensor]:
    return ops.tree_mask(parents, query_start_loc, max_nodes=max_nodes)


@tree_mask.register_fake
def _(parents, query_start_loc, max_nodes):
    n = parents.shape[0]
    return parents.new_empty((n, -(-max_nodes // 64)), dtype=torch.int64), parents.new_empty(n)


@torch.library.custom_op(f"{_LIB}::attention_tree", mutates_args=(), device_types="cuda")
def attention_tree(q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                   block_table: torch.Tensor, query_start_loc: list[int], seq_lens: list[int], mask: torch.Tensor, scale: float,
                   head_dim: int, stage_k: torch.Tensor | None = None, stage_v: torch.Tensor | None = None,
                   owner: torch.Tensor | None = None, soft_cap: float = 0.0) -> tuple[torch.Tensor, torch.Tensor]:
    hq, hk = q.shape[1], k_cache.shape[2]
    plan = ops.plan_tree(query_start_loc, seq_lens, num_kv_heads=hk, group=hq // hk, head_dim=head_dim, device=q.device)
    return ops.attention_tree(q, k_new, v_new, k_cache, v_cache, block_table, plan, mask, scale, _stage(stage_k, stage_v, owner),
                              head_dim=head_dim, soft_cap=soft_cap)


@attention_tree.register_fake
def _(q, k_new, v_new, k_cache, v_cache, block_table, query_start_loc, seq_lens, mask, scale, head_dim, stage_k=None,
      stage_v=None, owner=None, soft_cap=0.0):
    n, hq = q.shape[0], q.shape[1]
    return (q.new_empty((n, hq, head_dim), dtype=torch.float32), q.new_empty((n, hq), dtype=torch.float32))


# ------------------------------------------------------------------ chosen pages
@torch.library.custom_op(f"{_LIB}::page_bounds", mutates_args=("bounds",), device_types="cuda")
def page_bounds(k_cache: torch.Tensor, bounds: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor,
                seq_lens: torch.Tensor, max_new: int, head_dim: int) -> None:
    ops.page_bounds(k_cache, bounds, block_table, lengths, seq_lens, max_new=max_new, head_dim=head_dim)


@page_bounds.register_fake
def _(k_cache, bounds, block_table, lengths, seq_lens, max_new, head_dim):
    return None


@torch.library.custom_op(f"{_LIB}::attention_selected", mutates_args=(), device_types="cuda")
def attention_selected(q: torch.Tensor, k_new: torch.Tensor | None, v_new: torch.Tensor | None, k_cache: torch.Tensor,
                       v_cache: torch.Tensor, bounds: torch.Tensor, block_table: torch.Tensor, query_start_loc: list[int],
                       seq_lens: list[int], budget: int, scale: float, head_dim: int, first_pages: int = 1,
                       last_pages: int = 1, stage_k: torch.Tensor | None = None, stage_v: torch.Tensor | None = None,
                       owner: torch.Tensor | None = None, sink_tokens_eff: int = 0, recent_tokens: int = 0,
                       soft_cap: float = 0.0) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The choice and the attention in one: (out_rot, lse, chosen columns)."""
    hq, hk = q.shape[1], k_cache.shape[2]
    stage = _stage(stage_k, stage_v, owner)
    window = (sink_tokens_eff, recent_tokens) if stage is not None else (0, 0)
    plan = ops.plan_selected(query_start_loc, seq_lens, has_new=k_new is not None, block_size=k_cache.shape[1], budget=budget,
                             first_pages=first_pages, last_pages=last_pages, num_kv_heads=hk, group=hq // hk,
                             head_dim=head_dim, device=q.device, window=window)
    table, pages = ops.select_pages(q, bounds, block_table, plan)
    out, lse = ops.attention_selected(q, k_new, v_new, k_cache, v_cache, table, plan, scale, stage, head_dim=head_dim,
                                      soft_cap=soft_cap)
    return out, lse, pages


@attention_selected.register_fake
def _(q, k_new, v_new, k_cache, v_cache, bounds, block_table, query_start_loc, seq_lens, budget, scale, head_dim,
      first_pages=1, last_pages=1, stage_k=None, stage_v=None, owner=None, sink_tokens_eff=0, recent_tokens=0, soft_cap=0.0):
    n, hq = q.shape[0], q.shape[1]
    return (q.new_empty((n, hq, head_dim), dtype=torch.float32), q.new_empty((n, hq), dtype=torch.float32),
            block_table.new_empty((len(seq_lens), k_cache.shape[2], budget)))
