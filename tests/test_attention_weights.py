"""Accumulated attention weights (ops.accumulate_weights): refusals on the CPU, values against
a 64-bit evaluation on the GPU.

Tolerance, relative to the weight that a call adds: a score is a sum of d <= 256 exact
products, added in at most d / 8 dependent fp32 steps, so it errs by at most
32 x 2^-24 sum|q k| scale < 4e-5 for these inputs (sum|q k| scale < 21); a cap's tanh adds
cap 2^-22 < 1.5e-5, the log-sum-exp's own rounding to fp32 and to log2 units 2^-20, the exp2
2^-22; summing R rows in fp32 R 2^-24 (R < 400 in a lane).  Together below 1e-4; adding to
the old weight rounds once more, 2^-24 of the result.
"""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from oracle import cases
from oracle.attention import read_history
from oscar_amd import _lib

REL_TOL = 1e-4


def scores(q, keys, scale, cap, slopes, limit0):
    """64-bit masked scores [hq, n, t]; query i sees the first limit0 + i keys."""
    n, hq, _ = q.shape
    hk = keys.shape[1]
    q, keys = torch.as_tensor(np.asarray(q)).double(), torch.as_tensor(np.asarray(keys)).double()
    distance = torch.arange(keys.shape[0])[None] - (limit0 + torch.arange(n) - 1)[:, None]
    out = []
    for h in range(hq):
        s = q[:, h] @ keys[:, h * hk // hq].t() * scale
        s = cap * torch.tanh(s / cap) if cap else s
        s = s + slopes[h].double().cpu() * distance if slopes is not None else s
        out.append(s.masked_fill(distance > 0, -math.inf))
    return torch.stack(out)


# ------------------------------------------------------------------ refusals (no launch)
def args(**changes):
    """Arguments that pass every check; the addresses are never read."""
    a = _lib.WeightsArgs()
    cache = _lib.Cache(k=1 << 12, v=1 << 12, num_blocks=4, block_size=128, num_kv_heads=1, head_dim=256)
    cache.k_stride[:] = cache.v_stride[:] = [128 * 256, 256, 256]
    fixed = dict(q=2 << 12, num_tokens=3, num_q_heads=6, q_stride_token=1536, cache=cache, block_table=3 << 12,
                 block_table_stride=4, block_table_rows=2, block_table_cols=4, query_start_loc=4 << 12, seq_lens=5 << 12,
                 num_reqs=2, q_dtype=_lib.OSCAR_BF16, max_seq_len=300, max_query_len=2, scale=0.0625, lse=6 << 12,
                 weights=7 << 12, weights_stride_request=300, weights_stride_head=300, weights_cols=300)
    for name, value in {**fixed, **changes}.items():
        if name.startswith("cache_"):
            setattr(a.cache, name[6:], value)
        else:
            setattr(a, name, value)
    return a


@pytest.mark.parametrize("changes,message", [
    (dict(cache_head_dim=64), "head_dim 64 unsupported"),
    (dict(q_dtype=_lib.OSCAR_F32), "q_dtype"),
    (dict(num_reqs=-1), "negative size"),
    (dict(max_query_len=-1), "negative size"),
    (dict(num_q_heads=5, cache_num_kv_heads=2), "multiple"),
    (dict(q=None), "missing pointer"),
    (dict(lse=None), "missing pointer"),
    (dict(weights=None), "missing pointer"),
    (dict(num_reqs=70000, block_table_rows=70000), "too many"),
    (dict(num_tokens=(1 << 24) + 1), "too many"),
    (dict(max_seq_len=(1 << 30) + 1), "too many"),
    (dict(max_query_len=(1 << 24) + 1), "too many"),
    (dict(weights_cols=(1 << 30) + 1, weights_stride_head=1 << 31, weights_stride_request=1 << 31), "too many"),
    (dict(block_table_rows=1), "block-table rows"),
    (dict(block_table_cols=0), "block-table rows"),
    (dict(cache_block_size=48), "block_size"),
    (dict(weights_stride_head=299), "overlap"),
    (dict(weights_stride_request=299), "overlap"),
    (dict(weights_cols=0), "overlap"),
    (dict(cache_k=(1 << 12) + 8), "cache slots"),
    (dict(q_stride_token=1537), "aligned"),
    (dict(k_new=(8 << 12) + 2, k_new_stride_token=256), "aligned"),
])
def test_refusals(changes, message):
    lib, a = _lib.load(), args(**changes)
    assert lib.oscarop_attn_weights_v1(C.byref(a), None, None) == -22
    assert message in lib.oscar_last_error().decode()


def test_refused_arena_and_cap_and_empty_calls():
    lib = _lib.load()
    stage = _lib.Staging(stage_k=1 << 12, stage_v=1 << 12, owner=1 << 12, rows=0)
    a = args(staging=C.pointer(stage))
    assert lib.oscarop_attn_weights_v1(C.byref(a), None, None) == -22 and "arena" in lib.oscar_last_error().decode()
    score = _lib.Score(-1.0, None)
    assert lib.oscarop_attn_weights_v1(C.byref(args()), C.byref(score), None) == -22
    for empty in (dict(num_reqs=0), dict(num_tokens=0), dict(max_seq_len=0)):
        assert lib.oscarop_attn_weights_v1(C.byref(args(**empty)), None, None) == 0
    assert lib.oscarop_attn_weights_v1(None, None, None) == -22
    assert lib.oscarop_attn_weights_workspace_bytes_v1(None) == -22
    assert lib.oscarop_attn_weights_workspace_bytes_v1(C.byref(args())) >= 0


@pytest.mark.parametrize("seq,nq,hq,hk", [(2500, 2500, 6, 1), (8700, 700, 6, 1), (6000, 6000, 6, 1), (100000, 100000, 6, 1), (50, 700, 6, 1),
                                          (600, 600, 16, 2), (33, 33, 8, 8), (1, 1, 64, 1), (1 << 30, 1 << 24, 6, 1)])
def test_the_workspace_holds_whole_chunks_within_its_limit(seq, nq, hq, hk):
    """A workspace is the sums of two or more row chunks, 256 MB at most, and no batch that fills
    the chip by its keys alone has one."""
    lib = _lib.load()
    a = args(num_reqs=1, num_q_heads=hq, max_seq_len=seq, max_query_len=nq, weights_cols=seq, cache_num_kv_heads=hk)
    need = lib.oscarop_attn_weights_workspace_bytes_v1(C.byref(a))
    chunks, rest = divmod(need, 4 * hk * seq)
    assert rest == 0 and chunks != 1 and 0 <= need <= 256 << 20
    assert chunks <= max(1, -(-nq * (hq // hk) // 32))
    if -(-seq // 256) * hk >= 512 or nq * (hq // hk) <= 32:
        assert need == 0


@pytest.mark.parametrize("changes", [dict(num_reqs=1 << 16), dict(cache_num_kv_heads=1 << 16, num_q_heads=1 << 16),
                                     dict(num_reqs=4, cache_num_kv_heads=(1 << 62) + 1, num_q_heads=(1 << 62) + 1),
                                     dict(num_q_heads=1 << 44, max_query_len=1 << 24)])
def test_sizes_that_the_call_refuses_have_no_workspace(changes):
    assert _lib.load().oscarop_attn_weights_workspace_bytes_v1(C.byref(args(**changes))) == -22


@pytest.mark.parametrize("changes", [dict(num_tokens=1 << 20, num_q_heads=1 << 44), dict(num_tokens=1 << 60, num_q_heads=16),
                                     dict(num_q_heads=(1 << 20) + 1), dict(cache_num_kv_heads=1 << 16, num_q_heads=1 << 16)])
def test_sizes_whose_product_wraps_around_are_refused(changes):
    lib = _lib.load()
    assert lib.oscarop_attn_weights_v1(C.byref(args(**changes)), None, None) == -22
    assert "too many" in lib.oscar_last_error().decode()


def test_plan_refusals():
    from oscar_amd import ops

    for qsl, seqs, new in (([0, 2], [], True), ([0, 2, 1], [5, 5], True), ([0, 2], [1], True), ([0, 2], [-1], False),
                           ([-1, 2], [5], True)):
        with pytest.raises(ValueError):
            ops.plan_weights(qsl, seqs, has_new=new, device="cuda")


def test_the_sizes_of_a_plan_follow_its_lists():
    """A caller may change a plan's host lists between calls, as it does the device's."""
    from oscar_amd import ops

    plan = ops.WeightsPlan([0, 2, 2, 5], [300, 900, 40], True, None, None)
    assert ops._plan_sizes(plan, 128) == (3, 300, 3)  # (a request without queries reads nothing)
    assert ops._plan_sizes(plan, 32) == (10, 300, 3)
    plan.host_seqs[0] = 1000
    assert ops._plan_sizes(plan, 32) == (32, 1000, 3)
    plan.host_qsl = [0, 2, 4, 5]
    assert ops._plan_sizes(plan, 32) == (32, 1000, 2) and ops._plan_sizes(plan, 128) == (8, 1000, 2)
    plan.has_new = False
    plan.host_seqs[0] = 898
    assert ops._plan_sizes(plan, 32) == (29, 900, 2)
    table = torch.zeros(3, 28, dtype=torch.int32)
    with pytest.raises(ValueError, match="cannot cover"):
        ops._check_table(table, plan, 32)
    plan.host_seqs[:] = [896, 896, 896]
    ops._check_table(table, plan, 32)


@pytest.mark.parametrize("kind", [list, tuple, np.array, torch.tensor])
def test_a_plan_may_hold_its_lists_as_arrays(kind):
    from oscar_amd import ops

    plan = ops.WeightsPlan(kind([0, 2, 2, 5]), kind([300, 900, 40]), True, None, None)
    for _ in range(2):
        assert ops._plan_sizes(plan, 128) == (3, 300, 3)
    plan.host_seqs = kind([600, 900, 40])
    assert ops._plan_sizes(plan, 128) == (5, 600, 3)


def test_block_tables_are_laid_out_by_rows():
    from oscar_amd import ops

    t = torch.arange(24, dtype=torch.int32).view(4, 6)
    for same in (t, t[1:3], t[:, 1:4]):
        assert ops._rows_apart(same).data_ptr() == same.data_ptr()
    for other in (t.t(), t[:, ::2], t[:1].expand(3, 6), t[:, :1].t(), t[:, 2:3].expand(4, 5), t.long(), t[:, :1].long().t(),
                  t[:, 0::7], torch.arange(5, dtype=torch.int32)[:, None].t()):
        got = ops._rows_apart(other)
        assert torch.equal(got, other.int()) and got.stride(1) == 1 and got.stride(0) >= got.shape[1]


# ------------------------------------------------------------------ values
BATCHES = [
    ("mtp_window", [129, 1025, 3, 300], [4, 3, 1, 2], {}),
    ("one_key", [1], [1], {"window": False}),
    ("nothing_cached", [0, 0], [1, 45], {}),
    ("cache_only", [0, 257, 3, 263], [1, 1, 4, 5], {"fresh": False}),
    ("long_no_window", [9000, 31], [2, 1], {"window": False, "bs": 64}),
    ("d128_hk2", [129, 700, 64], [4, 2, 33], {"d": 128, "hk": 2, "group": 4}),
    ("chunks", [500, 2000], [411, 90], {}),
    ("wide_group", [333], [3], {"group": 40}),
    ("legacy_pages_32", [700, 97], [4, 1], {"legacy": True, "hk": 2, "group": 3, "bs": 32}),
    ("prompt", [0], [1111], {"d": 128, "hk": 2, "group": 8}),
]


@pytest.mark.gpu
@pytest.mark.parametrize("cap,steep", [(0.0, 0.0), (30.0, 0.0), (0.0, 1.0), (2.0, 0.5)])
@pytest.mark.parametrize("name,prefixes,lengths,opts", BATCHES, ids=[b[0] for b in BATCHES])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_values(cuda, name, prefixes, lengths, opts, cap, steep, dtype):
    from oscar_amd import ops

    d, hk, group = opts.get("d", 256), opts.get("hk", 1), opts.get("group", 6)
    hq, fresh = hk * group, opts.get("fresh", True)
    c = cases.make_case(prefixes, lengths, d=d, hk=hk, group=group, bs=opts.get("bs", 128), fresh=fresh,
                        window=opts.get("window", True), legacy=opts.get("legacy", False))
    slopes = torch.tensor([steep * 2.0 ** (-8.0 * (h + 1) / hq) for h in range(hq)]) if steep else None
    q, k = (None if c[x] is None else torch.from_numpy(c[x] * (2 if x == "q" else 1)).to(dtype) for x in "qk")
    g = torch.Generator().manual_seed(7)
    wide = torch.rand(len(prefixes) + 1, hk, max(c["seqs"]) + 9, generator=g)
    want, lse = wide.double().clone(), torch.zeros(q.shape[0], hq)
    for r, (a, b, seq) in enumerate(zip(c["qsl"], c["qsl"][1:], c["seqs"])):
        hist = seq - (b - a) if fresh else seq
        keys, _ = read_history(c["k8"], c["v8"], c["bt"][r], 0, hist, hk, d, c["stage"], "bf16" if dtype == torch.bfloat16 else "f16")
        keys = np.concatenate([keys, k[a:b].float()]) if fresh else keys
        if seq == 0:
            lse[a:b] = -math.inf
            continue
        s = scores(q[a:b].float(), keys, c["scale"], cap, slopes, seq - (b - a) + 1)
        lse[a:b] = torch.logsumexp(s, -1).t().float()
        p = torch.exp(s - lse[a:b].double().t()[..., None]).nan_to_num(0.0)
        want[r, :, :seq] += p.view(hk, group, b - a, seq).sum((1, 2))
    put = (lambda x: None if x is None else x.to(cuda))
    kc, vc = (torch.from_numpy(c[x]).view(torch.int8).to(cuda) for x in ("k8", "v8"))
    stage = None if c["stage"] is None else tuple(torch.from_numpy(a).to(cuda) for a in c["stage"])
    plan = ops.plan_weights(c["qsl"], c["seqs"], has_new=fresh, device=cuda)
    weights, bt = wide.to(cuda), torch.from_numpy(c["bt"]).to(cuda)
    call = (lambda w: ops.accumulate_weights(put(q), put(k), kc, vc, bt, plan, c["scale"], put(lse), w, stage, head_dim=d,
                                             soft_cap=cap, alibi_slopes=put(slopes)))
    got = call(weights)
    assert got is weights
    added = want - wide.double()
    tol = REL_TOL * added + 2.0 ** -24 * want + 1e-12
    assert ((got.double().cpu() - want).abs() <= tol).all()
    untouched = added == 0
    assert torch.equal(got.cpu()[untouched], wide[untouched])
    # a part of a larger tensor; the same bits
    big = torch.full((len(prefixes) + 3, hk, wide.shape[2] + 32), 5.0, device=cuda)
    big[1:len(prefixes) + 2, :, 16:16 + wide.shape[2]] = wide.to(cuda)
    call(big[1:len(prefixes) + 2, :, 16:16 + wide.shape[2]])
    assert torch.equal(big[1:len(prefixes) + 2, :, 16:16 + wide.shape[2]], got)
    big[1:len(prefixes) + 2, :, 16:16 + wide.shape[2]] = 5.0
    assert (big == 5.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("name,prefixes,lengths,opts", [
    ("more_key_groups_than_the_table", [33000], [200], {"window": False}),
    ("prompts_beside_each_other", [0, 0, 300], [1500, 700, 1000], {"d": 128, "hk": 2, "group": 4}),
])
def test_values_of_many_row_chunks(cuda, name, prefixes, lengths, opts):
    test_values(cuda, name, prefixes, lengths, opts, 30.0, 1.0, torch.bfloat16)


@pytest.mark.gpu
def test_lists_of_another_batch_than_the_call_is_sized_for(cuda):
    """Row chunks and their order come from the largest sizes alone: the device's lists may hold
    any other requests within them."""
    from oscar_amd import ops

    c = cases.make_case([900, 0, 5], [1200, 700, 1], window=False)
    q, k = (torch.from_numpy(c[x]).bfloat16().to(cuda) for x in "qk")
    kc, vc = (torch.from_numpy(c[x]).view(torch.int8).to(cuda) for x in ("k8", "v8"))
    bt, lse = torch.from_numpy(c["bt"]).to(cuda), torch.full((1901, 6), 5.0, device=cuda)
    bt = torch.cat([bt, bt.new_zeros(3, 20 - bt.shape[1])], 1) if bt.shape[1] < 20 else bt
    own = ops.plan_weights(c["qsl"], c["seqs"], has_new=True, device=cuda)
    call = (lambda plan: ops.accumulate_weights(q, k, kc, vc, bt, plan, 0.0625, lse, torch.zeros(3, 1, 2560, device=cuda), head_dim=256))
    want = call(own)
    for qsl, seqs in (([0, 1901, 1901, 1901], [1901, 0, 0]), ([0, 40, 1900, 1901], [2500, 1860, 1]), ([0, 1, 2, 1901], [1, 1, 2500])):
        plan = ops.plan_weights(qsl, seqs, has_new=True, device=cuda)
        plan.qsl.copy_(own.qsl)
        plan.seqs.copy_(own.seqs)
        got = call(plan)
        assert ((got - want).abs() <= 2e-6 * want + 1e-12).all()


@pytest.mark.gpu
def test_rows_that_hold_infinities_and_nan(cuda):
    """A row with lse = -inf adds nothing, with lse = +inf zeros; NaN stays with its request."""
    from oscar_amd import ops

    c = cases.make_case([300, 40], [3, 2])
    q, k = (torch.from_numpy(c[x]).bfloat16().to(cuda) for x in "qk")
    kc, vc = (torch.from_numpy(c[x]).view(torch.int8).to(cuda) for x in ("k8", "v8"))
    plan = ops.plan_weights(c["qsl"], c["seqs"], has_new=True, device=cuda)
    bt = torch.from_numpy(c["bt"]).to(cuda)
    run = (lambda lse: ops.accumulate_weights(q, k, kc, vc, bt, plan, 0.0625, lse, torch.zeros(2, 1, 320, device=cuda), head_dim=256))
    base = torch.full((5, 6), 3.0, device=cuda)
    some = base.clone()
    some[1], some[3, 2] = -math.inf, math.inf
    got, whole = run(some), run(base)
    assert got.isfinite().all() and (got <= whole).all() and got[0].sum() < whole[0].sum() and got[1].sum() < whole[1].sum()
    some[0, 0] = math.nan
    got = run(some)
    assert got[0, 0, :301].isnan().all() and got[1].isfinite().all()


@pytest.mark.gpu
def test_a_batch_that_does_not_fit_becomes_nan(cuda):
    """Lengths that only the device holds: the C entry reads nothing for such a request."""
    from oscar_amd import ops

    c = cases.make_case([300, 40], [3, 2])
    q, k = (torch.from_numpy(c[x]).bfloat16().to(cuda) for x in "qk")
    kc, vc = (torch.from_numpy(c[x]).view(torch.int8).to(cuda) for x in ("k8", "v8"))
    bt, lse = torch.from_numpy(c["bt"]).to(cuda), torch.zeros(5, 6, device=cuda)
    plan = ops.plan_weights(c["qsl"], c["seqs"], has_new=True, device=cuda)
    want = ops.accumulate_weights(q, k, kc, vc, bt, plan, 0.0625, lse, torch.zeros(2, 1, 320, device=cuda), head_dim=256)
    for bad in ([321, 42], [2, 42], [2000000000, 42]):
        plan.seqs.copy_(torch.tensor(bad, dtype=torch.int32))
        got = ops.accumulate_weights(q, k, kc, vc, bt, plan, 0.0625, lse, torch.zeros(2, 1, 320, device=cuda), head_dim=256)
        assert got[0, 0, :min(bad[0], 320)].isnan().all() and torch.equal(got[1], want[1])
    plan.seqs.copy_(torch.tensor(c["seqs"], dtype=torch.int32))
    plan.qsl.copy_(torch.tensor([0, 3, 900], dtype=torch.int32))
    got = ops.accumulate_weights(q, k, kc, vc, bt, plan, 0.0625, lse, torch.zeros(2, 1, 320, device=cuda), head_dim=256)
    assert torch.equal(got[0], want[0]) and got[1, 0, :42].isnan().all()


@pytest.mark.gpu
def test_wrapper_refusals_on_the_device(cuda):
    from oscar_amd import ops

    c = cases.make_case([300], [3])
    q, k = (torch.from_numpy(c[x]).bfloat16().to(cuda) for x in "qk")
    kc, vc = (torch.from_numpy(c[x]).view(torch.int8).to(cuda) for x in ("k8", "v8"))
    good = dict(q=q, k_new=k, k_cache=kc, v_cache=vc, block_table=torch.from_numpy(c["bt"]).to(cuda),
                plan=ops.plan_weights(c["qsl"], c["seqs"], has_new=True, device=cuda), scale=0.0625,
                lse=torch.zeros(3, 6, device=cuda), weights=torch.zeros(1, 1, 303, device=cuda), head_dim=256)
    ops.accumulate_weights(**good)
    for change in (dict(k_new=None), dict(k_new=k.half()), dict(k_new=k[:2]), dict(q=q.float()), dict(q=q[:2]),
                   dict(lse=good["lse"].double()), dict(lse=good["lse"][:2]), dict(weights=torch.zeros(1, 1, 302, device=cuda)),
                   dict(weights=torch.zeros(1, 2, 303, device=cuda)), dict(weights=torch.zeros(0, 1, 303, device=cuda)),
                   dict(weights=torch.zeros(1, 1, 303, device=cuda).double()), dict(weights=torch.zeros(1, 1, 606, device=cuda)[..., ::2]),
                   dict(block_table=good["block_table"][:, :2]), dict(block_table=good["block_table"][:0]), dict(soft_cap=-1.0)):
        with pytest.raises(ValueError):
            ops.accumulate_weights(**{**good, **change})
    two = ops.plan_weights([0, 1, 3], [100, 100], has_new=True, device=cuda)
    with pytest.raises(ValueError, match="overlap"):
        ops.accumulate_weights(**{**good, "plan": two, "block_table": good["block_table"].repeat(2, 1),
                                  "weights": torch.zeros(1, 1, 303, device=cuda).expand(2, 1, 303)})


@pytest.mark.gpu
def test_current_keys_of_fewer_rows_than_the_queries(cuda):
    """A padded batch whose keys are not padded: lists on the device that reach past the keys
    read nothing."""
    from oscar_amd import ops

    c = cases.make_case([300, 40], [3, 2])
    q, k = (torch.from_numpy(c[x]).bfloat16().to(cuda) for x in "qk")
    q = torch.cat([q, torch.full_like(q[:4], math.nan)])
    kc, vc = (torch.from_numpy(c[x]).view(torch.int8).to(cuda) for x in ("k8", "v8"))
    bt, lse = torch.from_numpy(c["bt"]).to(cuda), torch.zeros(9, 6, device=cuda)
    plan = ops.plan_weights(c["qsl"], c["seqs"], has_new=True, device=cuda)
    call = (lambda: ops.accumulate_weights(q, k, kc, vc, bt, plan, 0.0625, lse, torch.zeros(2, 1, 320, device=cuda), head_dim=256))
    want = call()
    assert want.isfinite().all() and (want[1, 0, :40] > 0).all()
    plan.qsl.copy_(torch.tensor([0, 3, 6], dtype=torch.int32))
    got = call()
    assert torch.equal(got[0], want[0]) and got[1, 0, :42].isnan().all()


@pytest.mark.gpu
def test_a_captured_prompt_keeps_its_workspace(cuda):
    """Row chunks go through a workspace: the captured call's stays its own, whatever sizes run
    and whatever is allocated afterwards, also under a replay on another stream."""
    from oscar_amd import ops

    gen = torch.Generator(device=cuda).manual_seed(3)
    kc = torch.zeros(4, 128, 1, 256, dtype=torch.int8, device=cuda)
    bt = torch.zeros(1, 40, dtype=torch.int32, device=cuda)

    def prompt(n):
        q, k = (torch.randn(n, h, 256, generator=gen, device=cuda).bfloat16() for h in (6, 1))
        lse = torch.full((n, 6), 3.0, device=cuda)
        plan = ops.plan_weights([0, n], [n], has_new=True, device=cuda)
        return lambda w: ops.accumulate_weights(q, k, kc, kc, bt, plan, 0.0625, lse, w, head_dim=256)

    small, large = prompt(700), prompt(4000)
    want, weights = (torch.zeros(1, 1, 4096, device=cuda) for _ in range(2))
    small(want)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        small(torch.zeros_like(weights))
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            small(weights)
    beside = torch.zeros_like(weights)
    for step in range(3):
        weights.zero_()
        beside.zero_()
        torch.cuda.synchronize()
        other = [torch.full((1 << 20,), 7.0, device=cuda) for _ in range(4)]
        with torch.cuda.stream(side):
            large(beside)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(weights, want), step
        if step == 0:
            first = beside.clone()
        assert torch.equal(beside, first) and all((x == 7.0).all() for x in other)


@pytest.mark.gpu
def test_captured_with_lengths_that_grow(cuda):
    """The plan's device lists may change between replays, within the sizes captured."""
    from oscar_amd import ops

    c = cases.make_case([700, 33], [3, 1])
    q, k = (torch.from_numpy(c[x]).bfloat16().to(cuda) for x in "qk")
    kc, vc = (torch.from_numpy(c[x]).view(torch.int8).to(cuda) for x in ("k8", "v8"))
    bt, lse = torch.from_numpy(c["bt"]).to(cuda), torch.full((4, 6), 4.0, device=cuda)
    plan = ops.plan_weights(c["qsl"], c["seqs"], has_new=True, device=cuda)
    weights = torch.zeros(2, 1, 1024, device=cuda)
    call = (lambda w: ops.accumulate_weights(q, k, kc, vc, bt, plan, 0.0625, lse, w, head_dim=256))
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        call(torch.zeros_like(weights))
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            call(weights)
    want = torch.zeros_like(weights)
    for extra in (0, 20, 100):
        plan.seqs.copy_(torch.tensor([c["seqs"][0] + extra, c["seqs"][1] + extra], dtype=torch.int32))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        call(want)
        torch.cuda.synchronize()
        assert torch.equal(weights, want) and weights[0, 0, 700 + extra] > 0


@pytest.mark.gpu
def test_values_of_many_requests(cuda):
    """As many key groups as the chip holds workgroups: rows are not cut into chunks, and sums go
    straight to the weights."""
    test_values(cuda, "", [260] * 127 + [200], [40] * 128, {"d": 128, "hk": 2, "group": 4}, 30.0, 1.0, torch.bfloat16)
    test_values(cuda, "", [240] * 127 + [3000], [40] * 128, {"hk": 2, "group": 2, "window": False}, 0.0, 0.0, torch.float16)


@pytest.mark.gpu
def test_a_misfit_among_many_requests(cuda):
    from oscar_amd import ops

    c = cases.make_case([260] * 128, [40] * 128, d=128, hk=2, group=4)
    q, k = (torch.from_numpy(c[x]).bfloat16().to(cuda) for x in "qk")
    kc, vc = (torch.from_numpy(c[x]).view(torch.int8).to(cuda) for x in ("k8", "v8"))
    bt, lse = torch.from_numpy(c["bt"]).to(cuda), torch.full((5120, 8), 3.0, device=cuda)
    plan = ops.plan_weights(c["qsl"], c["seqs"], has_new=True, device=cuda)
    call = (lambda: ops.accumulate_weights(q, k, kc, vc, bt, plan, 0.0625, lse, torch.zeros(128, 2, 320, device=cuda), head_dim=128))
    want = call()
    assert want.isfinite().all()
    plan.seqs[5], plan.seqs[9], plan.seqs[127] = 321, 39, 2000000000
    got = call()
    bad = torch.tensor([5, 9, 127])
    assert got[5].isnan().all() and got[9, :, :39].isnan().all() and (got[9, :, 39:] == 0).all() and got[127].isnan().all()
    rest = [r for r in range(128) if r not in bad]
    assert torch.equal(got[rest], want[rest])


@pytest.mark.gpu
def test_a_long_prompt_sums_many_rows(cuda):
    """131072 tokens of 6 heads: key 0 gets 786432 equal weights.  An fp32 sum of the 24576 row
    blocks one after the other is off by 2.3e-4.  Here an exp2 errs by 2^-22, its factor by
    2^-24, the sum of a block's 32 rows by 17 2^-24, the result by 2^-24: below 2^-19."""
    from oscar_amd import ops

    n = 131072
    q, k = torch.zeros(n, 6, 128, dtype=torch.bfloat16, device=cuda), torch.ones(n, 1, 128, dtype=torch.bfloat16, device=cuda)
    kc = torch.zeros(1, 128, 1, 128, dtype=torch.int8, device=cuda)
    plan = ops.plan_weights([0, n], [n], has_new=True, device=cuda)
    got = ops.accumulate_weights(q, k, kc, kc, torch.zeros(1, 1, dtype=torch.int32, device=cuda).expand(1, 1024).contiguous(), plan, 0.0625,
                                 torch.full((n, 6), 3.0, device=cuda), torch.zeros(1, 1, n, device=cuda), head_dim=128)
    want = 6 * math.exp(-3.0) * torch.arange(n, 0, -1, dtype=torch.float64)
    assert ((got[0, 0].double().cpu() - want).abs() <= 2.0 ** -19 * want).all()


@pytest.mark.gpu
def test_lengths_far_past_the_sizes_of_a_small_call(cuda):
    """Few rows, sized for 40 tokens: each wave then goes through more than 64 tiles, whose pages
    it looks up 64 at a time.  A key's sum does not depend on the grid."""
    from oscar_amd import ops

    c = cases.make_case([20000, 33], [3, 2], window=False)
    q, k = (torch.from_numpy(c[x]).bfloat16().to(cuda) for x in "qk")
    kc, vc = (torch.from_numpy(c[x]).view(torch.int8).to(cuda) for x in ("k8", "v8"))
    bt, lse = torch.from_numpy(c["bt"]).to(cuda), torch.full((5, 6), 5.0, device=cuda)
    own = ops.plan_weights(c["qsl"], c["seqs"], has_new=True, device=cuda)
    call = (lambda plan: ops.accumulate_weights(q, k, kc, vc, bt, plan, 0.0625, lse, torch.zeros(2, 1, 20100, device=cuda), head_dim=256))
    want = call(own)
    assert (want[0, 0, :20001] > 0).all() and (want[0, 0, 20003:] == 0).all()
    small = ops.plan_weights(c["qsl"], [40, 35], has_new=True, device=cuda)
    small.seqs.copy_(own.seqs)
    assert torch.equal(call(small), want)


@pytest.mark.gpu
def test_weights_with_the_heads_outermost(cuda):
    """A model may keep [KV heads, requests, columns]: its view by request is taken as it lies."""
    from oscar_amd import ops

    for prefixes, lengths in (([700, 129, 40], [4, 2, 1]), ([0, 300, 40], [700, 90, 1])):
        c = cases.make_case(prefixes, lengths, d=128, hk=2, group=4)
        q, k = (torch.from_numpy(c[x]).bfloat16().to(cuda) for x in "qk")
        kc, vc = (torch.from_numpy(c[x]).view(torch.int8).to(cuda) for x in ("k8", "v8"))
        bt, lse = torch.from_numpy(c["bt"]).to(cuda), torch.full((sum(lengths), 8), 3.0, device=cuda)
        plan = ops.plan_weights(c["qsl"], c["seqs"], has_new=True, device=cuda)
        call = (lambda w: ops.accumulate_weights(q, k, kc, vc, bt, plan, 0.0625, lse, w, head_dim=128))
        want = call(torch.zeros(3, 2, 720, device=cuda))
        got = torch.zeros(2, 3, 720, device=cuda)
        call(got.transpose(0, 1))
        assert torch.equal(got, want.transpose(0, 1))


@pytest.mark.gpu
def test_one_table_row_for_all_requests_and_a_row_out_of_a_column(cuda):
    """Requests that share a prefix's pages read them through one broadcast row."""
    from oscar_amd import ops

    c = cases.make_case([500], [6], window=False)
    q, k, v = (torch.from_numpy(c[x]).bfloat16().to(cuda) for x in "qkv")
    kc, vc = (torch.from_numpy(c[x]).view(torch.int8).to(cuda) for x in ("k8", "v8"))
    bt, lse = torch.from_numpy(c["bt"]).to(cuda), torch.full((6, 6), 5.0, device=cuda)

    def call(table, qsl, seqs):
        plan = ops.plan_decode(qsl, seqs, has_new=True, num_kv_heads=1, group=6, head_dim=256, device=cuda)
        out, _ = ops.attention_decode(q, k, v, kc, vc, table, plan, 0.0625, head_dim=256, soft_cap=20.0)
        return out, ops.accumulate_weights(q, k, kc, vc, table, plan, 0.0625, lse, torch.zeros(len(seqs), 1, 512, device=cuda), head_dim=256)

    for table, full, qsl, seqs in ((bt.expand(2, -1), bt.repeat(2, 1), [0, 2, 6], [502, 504]),
                                   (bt[0][:, None].t(), bt, [0, 6], [506])):
        assert table.stride(0) < table.shape[1]
        for a, b in zip(call(table, qsl, seqs), call(full, qsl, seqs)):
            assert torch.equal(a, b)
    column = bt[0][:, None].contiguous().t()
    plan = ops.plan_evict([500], [1], block_size=128, device=cuda)
    w = torch.rand(1, 1, 512, device=cuda)
    caches = [(kc.clone(), vc.clone()) for _ in range(2)]
    a, b = (ops.evict(plan, w, *pair, table, head_dim=256) for pair, table in zip(caches, (column, bt)))
    assert torch.equal(a, b) and torch.equal(caches[0][0], caches[1][0]) and torch.equal(caches[0][1], caches[1][1])
