"""Attention with capped and distance-biased scores (soft_cap, alibi_slopes): refusals on the
CPU, decode, prefill and the impl's forward against a 64-bit evaluation on the GPU.

Tolerances.  Scores: products of 16-bit values are exact, their fp32 sum over d <= 256 terms
errs by at most d 2^-24 sum|q k| scale; with standard normal rows (times the 2 that the
queries are scaled by) that is below 3e-4, and the cap's tanh adds cap 2^-22 (cap <= 60:
1.5e-5).  LSE: the largest score error, 4e-4 with the logarithm's rounding.  Outputs: a
probability errs by twice that (numerator and sum) and by its rounding to fp16 (half a step,
2^-11); a value by its rounding to the activations' type, which the kernels do at different
places (half a step of bf16, 2^-8), or to fp16 for the product (2^-11): together
2^-8 + 2^-10 + 8e-4 of sum p |v|, and half a step of a 16-bit output.  The prefill holds a
bf16 value v as fp16(v 2^-8): where that is a subnormal (|v| < 2^-6) its rounding is up to
2^-25, which is 2^-17 of v's own scale whatever v is, and the probabilities sum to 1: 2^-17.
"""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from oracle import cases
from oracle.attention import read_history
from oscar_amd import _lib

LSE_TOL = 4e-4
REL_TOL = 2.0 ** -8 + 2.0 ** -10 + 8e-4
ABS_TOL = 2.0 ** -17


def reference(q, k, v, hist, scale, cap, slopes, limit0):
    """64-bit attention of one request: q [n, hq, d], keys and values [t, hk, d]; query i sees
    the first limit0 + i keys and stands at the last of them.  Returns out, lse, sum p |v|."""
    n, hq, d = q.shape
    hk = k.shape[1]
    q, k, v = (torch.as_tensor(np.asarray(x)).double() for x in (q, k, v))
    out, size = torch.zeros(n, hq, d, dtype=torch.float64), torch.zeros(n, hq, d, dtype=torch.float64)
    lse = torch.full((n, hq), -math.inf, dtype=torch.float64)
    if k.shape[0] == 0:
        return out, lse, size
    distance = torch.arange(k.shape[0])[None] - (limit0 + torch.arange(n) - 1)[:, None]
    for h in range(hq):
        s = q[:, h] @ k[:, h * hk // hq].t() * scale
        if cap:
            s = cap * torch.tanh(s / cap)
        if slopes is not None:
            s = s + slopes[h].double().cpu() * distance
        s = s.masked_fill(distance > 0, -math.inf)
        lse[:, h] = torch.logsumexp(s, -1)
        p = torch.softmax(s, -1).nan_to_num(0.0)
        out[:, h], size[:, h] = p @ v[:, h * hk // hq], p @ v[:, h * hk // hq].abs()
    return out, lse, size


def check(out, lse, ref, out_step=0.0):
    want, want_lse, size = ref
    out = out.double().cpu()
    seen = want_lse.isfinite()
    if lse is not None:
        lse = lse.double().cpu()
        assert torch.equal(lse.isfinite(), seen) and (lse[~seen] == -math.inf).all()
        assert (lse - want_lse)[seen].abs().le(LSE_TOL).all()
    assert (out[~seen] == 0).all()
    excess = (out - want).abs() - (REL_TOL * size + out_step * want.abs() + ABS_TOL)
    assert excess.max() <= 0, excess.max()


def slopes_of(hq, steep=1.0):
    return torch.tensor([steep * 2.0 ** (-8.0 * (h + 1) / hq) for h in range(hq)], dtype=torch.float32)


SCORES = [(30.0, 0.0), (0.0, 1.0), (2.0, 0.0), (50.0, 4.0), (25.0, -0.01)]  # cap, steepness of the slopes

# ------------------------------------------------------------------ refusals (no launch)


@pytest.mark.parametrize("cap", [-1.0, math.inf, math.nan])
def test_c_entries_refuse_a_bad_cap(cap):
    lib, score = _lib.load(), _lib.Score(cap, None)
    a, p, s = _lib.AttnArgs(), _lib.PrefillArgs(), _lib.StepArgs()
    a.num_items = a.num_groups = 1
    p.num_tokens = p.num_q_heads = p.num_kv_heads = 1
    p.head_dim, p.q_dtype = 128, _lib.OSCAR_BF16
    p.q = p.k = p.v = p.out = 4096
    for call in (lambda: lib.oscarop_attn_decode_v1(C.byref(a), C.byref(score), None),
                 lambda: lib.oscarop_attn_prefill_v1(C.byref(p), C.byref(score), None),
                 lambda: lib.oscarop_decode_step_v1(C.c_void_p(4096), C.byref(s), C.byref(score), None)):
        assert call() == -22
        assert "soft_cap" in lib.oscar_last_error().decode()


@pytest.mark.parametrize("cap", [-0.5, 2.0 ** -21, 1024.5, 1e30, 3.4e38])
def test_caps_outside_the_range_are_refused(cap):
    """A large cap would lose the score (it keeps cap 2^-22), a tiny one has no scale / cap."""
    from oscar_amd import ops

    test_c_entries_refuse_a_bad_cap(cap)
    with pytest.raises(ValueError, match="soft_cap"):
        ops.score_struct(cap, None, 6, torch.device("cpu"))
    for good in (2.0 ** -20, 1024):
        assert ops.score_struct(good, None, 6, torch.device("cpu")).soft_cap == good


def test_score_struct_refusals():
    from oscar_amd import ops

    cpu = torch.device("cpu")
    good = slopes_of(6)
    assert ops.score_struct(0.0, None, 6, cpu) is None
    assert ops.score_struct(0.0, good, 6, cpu).alibi_slopes == good.data_ptr()
    for bad in (good.double(), good[:5], good[::2].repeat(2)[::2], good.view(2, 3)):
        with pytest.raises(ValueError, match="alibi_slopes"):
            ops.score_struct(0.0, bad, 6, cpu)
    with pytest.raises(ValueError, match="queries on meta"):
        ops.score_struct(0.0, good, 6, torch.device("meta"))
    for cap in (-1.0, math.inf, math.nan):
        with pytest.raises(ValueError, match="soft_cap"):
            ops.score_struct(cap, None, 6, cpu)


@pytest.mark.parametrize("cap,want", [(None, 0), (0, 0), (0.0, 0), (-1.0, 0), (math.inf, 0), (30, 30), (2.0 ** -20, 2.0 ** -20), (1e-9, 2.0 ** -20),
                                      (1024.0, 1024), (1025, 0), (1e30, 0), (np.float32(50), 50)])
def test_a_layer_runs_with_any_cap(cap, want):
    """What models write for no cap, and caps beside the kernels' range, ran before the kernels
    took caps at all."""
    from oscar_amd import ops

    cpu = torch.device("cpu")
    for slopes in (None, slopes_of(6).tolist()):
        score = impl_of(cap, slopes)._score_args(cpu)
        if slopes is None and not want:
            assert score == {}
            continue
        assert score["soft_cap"] == want and (score["alibi_slopes"] is None) == (slopes is None)
        struct = ops.score_struct(score["soft_cap"], score["alibi_slopes"], 6, cpu)
        assert struct.soft_cap == want
    # what is left out of a score that is not capped, and what the least cap adds to a smaller one
    if cap and cap > 1024 and cap < 1e20:
        s = torch.linspace(-14, 14, 999, dtype=torch.float64)
        assert (s - cap * torch.tanh(s / cap)).abs().max() < 2.0 ** -10


# ------------------------------------------------------------------ decode
DECODE = [
    ("mtp_window", [129, 1025, 3, 300], [4, 3, 1, 2], {}),
    ("one_key", [1], [1], {"window": False}),
    ("cache_only", [0, 257, 3, 263], [1, 1, 4, 5], {"fresh": False}),
    ("few_long_items", [9000], [1], {"fresh": False, "target": 2}),
    ("few_long_items_mtp", [8000, 3001], [4, 2], {"target": 3}),
    ("no_window_64", [1025, 2048], [4, 4], {"window": False, "bs": 64}),
    ("d128_hk2", [129, 700], [4, 2], {"d": 128, "hk": 2, "group": 4}),
    ("chunk_240_rows", [3000, 500], [40, 7], {}),
    ("legacy_hk2", [700, 2000], [4, 1], {"legacy": True, "hk": 2, "group": 3}),
]


@pytest.mark.gpu
@pytest.mark.parametrize("cap,steep", SCORES)
@pytest.mark.parametrize("name,prefixes,lengths,opts", DECODE, ids=[c[0] for c in DECODE])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_decode(cuda, name, prefixes, lengths, opts, cap, steep, dtype):
    from oscar_amd import ops

    d, hk, group = opts.get("d", 256), opts.get("hk", 1), opts.get("group", 6)
    c = cases.make_case(prefixes, lengths, d=d, hk=hk, group=group, bs=opts.get("bs", 128), fresh=opts.get("fresh", True),
                        window=opts.get("window", True), legacy=opts.get("legacy", False))
    hq = hk * group
    slopes = slopes_of(hq, steep) if steep else None
    q, k, v = (None if c[x] is None else torch.from_numpy(c[x] * (2 if x == "q" else 1)).to(dtype) for x in "qkv")
    put = (lambda x: None if x is None else x.to(cuda))
    kc, vc = (torch.from_numpy(c[x]).view(torch.int8).to(cuda) for x in ("k8", "v8"))
    stage = None if c["stage"] is None else tuple(torch.from_numpy(a).to(cuda) for a in c["stage"])
    plan = ops.plan_decode(c["qsl"], c["seqs"], has_new=k is not None, num_kv_heads=hk, group=group, head_dim=d, device=cuda,
                           target_items=opts.get("target", 256), window=(128, 256) if stage else (0, 0))
    out, lse = ops.attention_decode(put(q), put(k), put(v), kc, vc, torch.from_numpy(c["bt"]).to(cuda), plan, c["scale"],
                                    stage, head_dim=d, soft_cap=cap, alibi_slopes=put(slopes))
    kind = "bf16" if dtype == torch.bfloat16 else "f16"
    for r, (a, b, seq) in enumerate(zip(c["qsl"], c["qsl"][1:], c["seqs"])):
        hist = seq - (b - a) if k is not None else seq
        hk_, hv = read_history(c["k8"], c["v8"], c["bt"][r], 0, hist, hk, d, c["stage"], kind)
        if k is not None:
            hk_, hv = np.concatenate([hk_, k[a:b].float()]), np.concatenate([hv, v[a:b].float()])
        check(out[a:b], lse[a:b], reference(q[a:b].float(), hk_, hv, hist, c["scale"], cap, slopes, seq - (b - a) + 1))


@pytest.mark.gpu
@pytest.mark.parametrize("cap", [2.0 ** -20, 1024.0])
def test_the_least_and_the_largest_cap(cuda, cap):
    """Scores within LSE_TOL of the formula's: 1024 2^-22 is 2.5e-4, and products that err by
    less than 1e-4 here (a query that is not scaled up)."""
    from oscar_amd import ops

    c = cases.make_case([129, 700, 0], [4, 2, 3])
    q, k, v = (torch.from_numpy(c[x]).bfloat16() for x in "qkv")
    kc, vc = (torch.from_numpy(c[x]).view(torch.int8).to(cuda) for x in ("k8", "v8"))
    stage = tuple(torch.from_numpy(a).to(cuda) for a in c["stage"])
    bt = torch.from_numpy(c["bt"]).to(cuda)
    plan = ops.plan_decode(c["qsl"], c["seqs"], has_new=True, num_kv_heads=1, group=6, head_dim=256, device=cuda)
    out, lse = ops.attention_decode(q.to(cuda), k.to(cuda), v.to(cuda), kc, vc, bt, plan, c["scale"], stage, head_dim=256,
                                    soft_cap=cap)
    long = ops.attention_prefill(q[:4].to(cuda), k[:4].to(cuda), v[:4].to(cuda), c["scale"], head_dim=256, history=129,
                                 k_cache=kc, v_cache=vc, block_table_row=bt[0], stage=stage, soft_cap=cap)
    for r, (a, b, seq) in enumerate(zip(c["qsl"], c["qsl"][1:], c["seqs"])):
        hk_, hv = read_history(c["k8"], c["v8"], c["bt"][r], 0, seq - (b - a), 1, 256, c["stage"], "bf16")
        hk_, hv = np.concatenate([hk_, k[a:b].float()]), np.concatenate([hv, v[a:b].float()])
        ref = reference(q[a:b].float(), hk_, hv, seq - (b - a), c["scale"], cap, None, seq - (b - a) + 1)
        check(out[a:b], lse[a:b], ref)
        if r == 0:
            check(long, None, ref)


@pytest.mark.gpu
def test_no_cap_and_no_slopes_are_the_plain_call(cuda):
    from oscar_amd import ops

    c = cases.make_case([700, 33], [3, 1])
    kc, vc = (torch.from_numpy(c[x]).view(torch.int8).to(cuda) for x in ("k8", "v8"))
    stage = tuple(torch.from_numpy(a).to(cuda) for a in c["stage"])
    q, k, v = (torch.from_numpy(c[x]).bfloat16().to(cuda) for x in "qkv")
    plan = ops.plan_decode(c["qsl"], c["seqs"], has_new=True, num_kv_heads=1, group=6, head_dim=256, device=cuda)
    run = (lambda **kw: ops.attention_decode(q, k, v, kc, vc, torch.from_numpy(c["bt"]).to(cuda), plan, c["scale"], stage,
                                             head_dim=256, **kw))
    plain, (out, lse) = run(), run(soft_cap=0.0, alibi_slopes=None)
    assert torch.equal(plain[0], out) and torch.equal(plain[1], lse)
    zero = run(alibi_slopes=torch.zeros(6, device=cuda))
    assert (zero[1] - plain[1]).abs().max() <= LSE_TOL
    with pytest.raises(ValueError, match="workspace decode"):
        run(soft_cap=1.0, static_scratch=True)


# ------------------------------------------------------------------ prefill
PREFILL = [
    # history, tokens, hq, hk, d, dtype
    (0, 1, 6, 1, 256, torch.bfloat16),
    (0, 33, 8, 1, 128, torch.float16),
    (0, 777, 6, 1, 256, torch.bfloat16),
    (0, 2100, 6, 1, 256, torch.float16),
    (0, 1301, 16, 2, 128, torch.bfloat16),
    (1, 5, 6, 1, 256, torch.bfloat16),
    (100, 70, 8, 2, 256, torch.bfloat16),
    (2900, 611, 6, 1, 256, torch.float16),
    (2900, 130, 16, 2, 128, torch.bfloat16),
]


@pytest.mark.gpu
@pytest.mark.parametrize("cap,steep", SCORES)
@pytest.mark.parametrize("split", [True, False])
@pytest.mark.parametrize("hist,n,hq,hk,d,dtype", PREFILL)
def test_prefill(cuda, hist, n, hq, hk, d, dtype, split, cap, steep):
    from oscar_amd import ops

    c = cases.make_case([hist], [n], d=d, hk=hk, group=hq // hk, seed=hist + n)
    slopes = slopes_of(hq, steep) if steep else None
    q, k, v = (torch.from_numpy(c[x] * (2 if x == "q" else 1)).to(dtype) for x in "qkv")
    more = {}
    if hist:
        lse = torch.empty(n, hq, dtype=torch.float32, device=cuda)
        more = dict(history=hist, k_cache=torch.from_numpy(c["k8"]).view(torch.int8).to(cuda),
                    v_cache=torch.from_numpy(c["v8"]).view(torch.int8).to(cuda), lse=lse,
                    block_table_row=torch.from_numpy(c["bt"][0]).to(cuda),
                    stage=tuple(torch.from_numpy(a).to(cuda) for a in c["stage"]))
    out = ops.attention_prefill(q.to(cuda), k.to(cuda), v.to(cuda), c["scale"], head_dim=d, split=split, soft_cap=cap,
                                alibi_slopes=None if slopes is None else slopes.to(cuda), **more)
    hk_, hv = read_history(c["k8"], c["v8"], c["bt"][0], 0, hist, hk, d, c["stage"],
                           "bf16" if dtype == torch.bfloat16 else "f16")
    ref = reference(q.float(), np.concatenate([hk_, k.float()]), np.concatenate([hv, v.float()]), hist, c["scale"], cap,
                    slopes, hist + 1)
    step = 0.0 if hist else (2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -11)
    check(out, more.get("lse"), ref, step)


@pytest.mark.gpu
@pytest.mark.parametrize("split", [False, True])
@pytest.mark.parametrize("cap,steep", [(50.0, 0.0), (50.0, 1e-6), (0.0, 1e-6)])
def test_many_keys_far_below_the_largest(cuda, cap, steep, split):
    """One key takes nearly all of a row and thousands share the rest, each 2^-19 of it.  Their
    probabilities are subnormal in fp16: each is off by half a step, 2^-25, where the row's
    largest is 2^-1 or more (the reference lies at most one binary order above it): 2^-24 of
    the row's sum a key."""
    from oscar_amd import ops

    n, hq, rows = 6000, 6, 64
    q, k, v = torch.zeros(n, hq, 256), torch.zeros(n, 1, 256), torch.ones(n, 1, 256)
    q[..., 0], k[:, 0, 0], k[0, 0, 0] = 16.0, 2.03125, 16.0 if cap else 15.5
    v[0] = 0.0
    q, k, v = q.bfloat16(), k.bfloat16(), v.bfloat16()
    slopes = slopes_of(hq, steep) if steep else None
    out = ops.attention_prefill(q.to(cuda), k.to(cuda), v.to(cuda), 0.0625, head_dim=256, split=split, soft_cap=cap,
                                alibi_slopes=None if slopes is None else slopes.to(cuda))[-rows:].double().cpu()
    want, _, size = reference(q[-rows:].float(), k.float(), v.float(), n - rows, 0.0625, cap, slopes, n - rows + 1)
    assert 0.004 < want.min() and want.max() < 0.05
    excess = (out - want).abs() - (REL_TOL * size + 2.0 ** -8 * want.abs() + ABS_TOL + n * 2.0 ** -24)
    assert excess.max() <= 0, ((out - want) / want).abs().max()


@pytest.mark.gpu
@pytest.mark.parametrize("below", [16.703125, 15.25])
@pytest.mark.parametrize("split", [False, True])
@pytest.mark.parametrize("cap", [0.0, 512.0])
@pytest.mark.parametrize("n", [1, 3])
def test_a_long_history_far_below_the_own_key(cuda, n, cap, split, below):
    """131072 cached keys, each `below` nats under the row's own key (24.1 and 22 binary orders): in
    fp16 against that key every one would be nothing, or a subnormal of one or two bits.  A key's
    probability is off by 2^-25 of the reference, which lies a binary order above the largest key
    of a unit at most, and a unit has 2^12 keys, or a reference that is lower by the excess: 2^-12
    of the row's sum."""
    from oscar_amd import ops

    hist, d, hq, bs = 131072, 256, 6, 128
    kc, vc = (torch.zeros(1, bs, 1, d, dtype=torch.int8, device=cuda) for _ in range(2))
    own = 16.0
    kc.view(torch.float16)[..., 1] = own - below  # K: every code is the zero point; V: 1
    kc.view(torch.float16)[..., 3] = 1.0
    q, k, v = torch.zeros(n, hq, d), torch.zeros(n, 1, d), torch.zeros(n, 1, d)
    q[..., 0] = 16.0
    k[:, 0, 0] = own
    q, k, v = q.bfloat16(), k.bfloat16(), v.bfloat16()
    slopes, lse = slopes_of(hq, 1e-6), torch.empty(n, hq, device=cuda)
    out = ops.attention_prefill(q.to(cuda), k.to(cuda), v.to(cuda), 0.0625, head_dim=d, history=hist, k_cache=kc, v_cache=vc,
                                block_table_row=torch.zeros(hist // bs, dtype=torch.int32, device=cuda), lse=lse, split=split,
                                soft_cap=cap, alibi_slopes=slopes.to(cuda))
    assert torch.tensor(own - below).half().bfloat16() == own - below
    s_own, s_far = own, own - below
    if cap:
        s_own, s_far = (cap * math.tanh(x / cap) for x in (s_own, s_far))
    pos = torch.arange(hist, dtype=torch.float64)
    for i in range(n):
        for h in range(hq):
            far = torch.exp(s_far - s_own + slopes[h].double() * (pos - (hist + i))).sum()
            near = torch.exp(slopes[h].double() * -torch.arange(i + 1, dtype=torch.float64)).sum()
            want = (far / (far + near)).item()
            assert 0.001 < want < 0.1
            assert (out[i, h].double().cpu() - want).abs().max() <= REL_TOL * want + ABS_TOL + 2.0 ** -12, (i, h, want, out[i, h, 0])
            assert abs(lse[i, h].item() - s_own - math.log((far + near).item())) <= LSE_TOL


@pytest.mark.gpu
@pytest.mark.parametrize("cap", [0.0, 20.0])
def test_overflowing_products_and_later_tokens(cuda, cap):
    """A score that overflows is capped like any other; what a later token holds does not
    reach the queries before it."""
    from oscar_amd import ops

    n, d = 200, 256
    g = torch.Generator(device=cuda).manual_seed(3)
    q, k, v = (torch.randn(n, h, d, generator=g, device=cuda).bfloat16() for h in (6, 1, 1))
    slopes = slopes_of(6).to(cuda)
    want = ops.attention_prefill(q, k, v, 0.0625, head_dim=d, soft_cap=cap, alibi_slopes=slopes)
    k[150], v[150] = float("nan"), float("inf")
    got = ops.attention_prefill(q, k, v, 0.0625, head_dim=d, soft_cap=cap, alibi_slopes=slopes)
    # (a tile of 128 rows takes 21 tokens of six heads; the one that holds token 150 starts at 147)
    assert torch.equal(got[:147], want[:147])
    if cap:
        k[150], v[150], q[100:120], k[3] = 0, 0, 2e30, -2e30
        got = ops.attention_prefill(q, k, v, 0.0625, head_dim=d, soft_cap=cap)
        s = (q.double()[:, 0] @ k.double()[:, 0].t() * 0.0625).clamp(-3e38, 3e38)
        s = (cap * torch.tanh(s / cap)).masked_fill(torch.ones(n, n, device=cuda).triu(1) > 0, -math.inf)
        p = torch.softmax(s, -1)
        bound = (REL_TOL + 2.0 ** -8) * (p @ v.double()[:, 0].abs()) + ABS_TOL
        assert ((got[:, 0].double() - p @ v.double()[:, 0]).abs() <= bound).all()


# ------------------------------------------------------------------ the impl
class _Bag:
    layer_name = "model.layers.0.self_attn.attn"


def impl_of(cap, slopes, hq=6, hk=1, d=256):
    from oscar_amd.backend import OscarAttentionBackendImpl

    impl = OscarAttentionBackendImpl.__new__(OscarAttentionBackendImpl)
    impl.head_size, impl.num_heads, impl.num_kv_heads, impl.scale = d, hq, hk, d ** -0.5
    impl.key_cache = impl.value_cache = None
    impl.logits_soft_cap, impl.alibi_slopes = cap, slopes
    impl._oscar_setup()
    return impl


def step(impl, layer, caches, table, histories, chunks, seed, cuda):
    """One forward over a batch; returns (q, k, v, out)."""
    g = torch.Generator(device=cuda).manual_seed(seed)
    n, bs = sum(chunks), caches[0].shape[1]
    q, k, v = (torch.randn(n, h * impl.head_size, generator=g, device=cuda).bfloat16()
               for h in (2 * impl.num_heads // 2, impl.num_kv_heads, impl.num_kv_heads))
    q = q * 2
    md = _Bag()
    pos = [np.arange(h, h + c) for h, c in zip(histories, chunks)]
    host = table.cpu().numpy()
    md.slot_mapping = torch.from_numpy(np.concatenate([host[r, p // bs].astype(np.int64) * bs + p % bs
                                                       for r, p in enumerate(pos)])).to(cuda)
    md.num_actual_tokens, md.block_tables = n, table
    md.query_start_loc_cpu = torch.tensor([0] + np.cumsum(chunks).tolist(), dtype=torch.int32)
    md.seq_lens_list = [h + c for h, c in zip(histories, chunks)]
    out = torch.empty_like(q)
    impl.forward(layer, q, k, v, caches, md, output=out)
    return q.view(n, -1, impl.head_size), k.view(n, -1, impl.head_size), v.view(n, -1, impl.head_size), out.view(n, -1, impl.head_size)


@pytest.mark.gpu
@pytest.mark.parametrize("cap,steep", [(20.0, 0.0), (0.0, 1.0), (20.0, 1.0)])
def test_forward_uses_the_layers_scores(cuda, cap, steep):
    """A fresh prompt, a verify step (native), a mixed batch, cached chunks of both routes
    (split-K, prefill): every row as attention over what the cache then holds."""
    from oscar_amd import ops

    slopes = slopes_of(6, steep).tolist() if steep else None
    impl, layer, bs = impl_of(cap, slopes), _Bag(), 128
    caches = tuple(torch.zeros(64, bs, 1, 256, dtype=torch.int8, device=cuda) for _ in range(2))
    table = torch.randperm(64, generator=torch.Generator().manual_seed(1)).view(2, 32).int().to(cuda)
    rk, rv = (torch.from_numpy(cases.hadamard_rotation(256, s)).to(cuda) for s in (1, 2))
    layer._oscar_rots = (rk, rv)
    fixed = slopes_of(6, steep) if steep else None
    lengths = [0, 0]
    for seed, (histories, chunks) in enumerate([([0, 0], [300, 41]), ([300, 41], [4, 4]), ([304, 0], [2, 90]),
                                                ([306, 90], [700, 1])]):
        before = [x.clone() for x in caches] + [x.clone() for x in impl._stage(layer) or ()]
        q, k, v, out = step(impl, layer, caches, table, histories, chunks, seed, cuda)
        start = 0
        for r, (h, c) in enumerate(zip(histories, chunks)):
            rows = slice(start, start + c)
            start += c
            if h == 0:
                ref = reference(q[rows].float().cpu(), k[rows].float().cpu(), v[rows].float().cpu(), 0, impl.scale, cap, fixed, 1)
                check(out[rows], None, ref, 2.0 ** -8)
                continue
            # rotated rows in bf16, as the store leaves them for the read
            qr, kr, vr = (ops.rotate(x[rows].contiguous(), m).float().cpu() for x, m in ((q, rk), (k, rk), (v, rv)))
            stage = tuple(x.cpu().numpy() for x in impl._stage(layer))
            k8, v8 = (x.view(torch.uint8).cpu().numpy() for x in caches)
            hist_k, hist_v = read_history(k8, v8, table[r].cpu().numpy(), 0, h, 1, 256, stage, "bf16")
            want, lse, size = reference(qr, np.concatenate([hist_k, kr]), np.concatenate([hist_v, vr]), h, impl.scale, cap,
                                        fixed, h + 1)
            # back to the model's domain: a row's error may turn into any of its places
            m = rv.double().cpu()
            bound = (size.norm(dim=-1, keepdim=True) * (REL_TOL + 2.0 ** -8) + 16 * ABS_TOL)
            assert ((out[rows].double().cpu() - want @ m.t()).abs() <= bound).all()
        lengths = [h + c for h, c in zip(histories, chunks)]
        assert len(before) >= 2 and not torch.equal(before[0], caches[0])


@pytest.mark.gpu
def test_captured_with_eager_calls_between(cuda):
    from oscar_amd import ops

    c = cases.make_case([700, 33], [3, 1])
    kc, vc = (torch.from_numpy(c[x]).view(torch.int8).to(cuda) for x in ("k8", "v8"))
    q, k, v = (torch.from_numpy(c[x]).bfloat16().to(cuda) for x in "qkv")
    bt, slopes = torch.from_numpy(c["bt"]).to(cuda), slopes_of(6).to(cuda)
    plan = ops.plan_decode(c["qsl"], c["seqs"], has_new=True, num_kv_heads=1, group=6, head_dim=256, device=cuda)
    out, lse = torch.zeros(4, 6, 256, device=cuda), torch.zeros(4, 6, device=cuda)
    fresh = torch.zeros(4, 6, 256, device=cuda, dtype=torch.bfloat16)

    def call(o, l_, f):
        ops.attention_decode(q, k, v, kc, vc, bt, plan, c["scale"], head_dim=256, out_rot=o, lse=l_, soft_cap=9.0,
                             alibi_slopes=slopes)
        ops.attention_prefill(q, k, v, c["scale"], head_dim=256, out=f, soft_cap=9.0, alibi_slopes=slopes)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        call(out, lse, fresh)
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=side):
            call(out, lse, fresh)
    for _ in range(3):
        q.mul_(-1)
        graph.replay()
        want = [torch.zeros_like(x) for x in (out, lse, fresh)]
        call(*want)
        torch.cuda.synchronize()
        for a, b in zip((out, lse, fresh), want):
            assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("cap,steep", [(0.0, 0.0), (9.0, 1.0)])
def test_captured_calls_keep_their_workspaces(cuda, cap, steep):
    """A captured decode and a captured split prefill: calls that need larger workspaces run
    on the capture stream afterwards, memory is allocated and filled, and the graph is replayed
    on another stream beside such calls."""
    from oscar_amd import ops

    score = dict(soft_cap=cap, alibi_slopes=slopes_of(6, steep).to(cuda) if steep else None)
    gen = torch.Generator(device=cuda).manual_seed(4)

    def calls(histories, chunks, tokens):
        # (items of one tile each, whose sums have one order)
        c = cases.make_case(histories, chunks)
        plan = ops.plan_decode(c["qsl"], c["seqs"], has_new=True, num_kv_heads=1, group=6, head_dim=256, device=cuda,
                               target_items=400)
        kc, vc = (torch.from_numpy(c[x]).view(torch.int8).to(cuda) for x in ("k8", "v8"))
        q, k, v = (torch.from_numpy(c[x]).bfloat16().to(cuda) for x in "qkv")
        rows = [torch.randn(tokens, h, 256, generator=gen, device=cuda).bfloat16() for h in (6, 1, 1)]
        bt, n = torch.from_numpy(c["bt"]).to(cuda), sum(chunks)
        outs = (torch.zeros(n, 6, 256, device=cuda), torch.zeros(n, 6, device=cuda),
                torch.zeros(tokens, 6, 256, device=cuda, dtype=torch.bfloat16))

        def run():
            ops.attention_decode(q, k, v, kc, vc, bt, plan, c["scale"], head_dim=256, out_rot=outs[0], lse=outs[1], **score)
            ops.attention_prefill(*rows, c["scale"], head_dim=256, out=outs[2], **score)
        return run, outs, plan.partial_bytes

    small, outs, few = calls([700, 33], [3, 1], 900)
    large, others, many = calls([5000], [4], 4000)
    assert many > max(few, 1 << 20)  # (a shared workspace has a megabyte at least)
    small()
    large()
    want, beside = [x.clone() for x in outs], [x.clone() for x in others]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        small()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            small()
    for step in range(3):
        for x in (*outs, *others):
            x.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            large()
            fillers = [torch.full((1 << 20,), 7.0, device=cuda) for _ in range(8)]
            large()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((*outs, *others), (*want, *beside))), step
        assert all((x == 7.0).all() for x in fillers)
