"""The operators together, as a serving loop runs them (head norms, the write, scored
attention, its weights, eviction, the next step), and as torch operators."""
import math
import re

import numpy as np
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import oscar_amd.torch_ops  # noqa: F401  (registers the operators)
from oracle import cases
from oracle.attention import read_history
from test_scored_attention import REL_TOL, reference, slopes_of

CAP, SCALE, D, HQ, HK, BS = 30.0, 256 ** -0.5, 256, 12, 2, 128


def test_torch_operators_are_registered_and_give_shapes():
    mutated = {"accumulate_weights": {"weights"}, "evict": {"k_cache", "v_cache", "owner"}, "norm_rope": set()}
    for name, want in mutated.items():
        schema = str(getattr(torch.ops.oscar_amd, name).default._schema)
        assert set(re.findall(r"Tensor\(a\d+!\)\?? (\w+)", schema)) == want, schema
    with FakeTensorMode():
        q = torch.empty(5, 6, 256, dtype=torch.bfloat16, device="cuda")
        a, b = torch.ops.oscar_amd.norm_rope(q, q[:, :1], torch.empty(5, dtype=torch.int64, device="cuda"),
                                             torch.empty(9, 64, device="cuda"))
        assert a.shape == q.shape and b.shape == (5, 1, 256) and a.dtype == q.dtype
        w, kc = torch.empty(1, 1, 300, device="cuda"), torch.empty(8, 128, 1, 256, dtype=torch.int8, device="cuda")
        bt = torch.empty(1, 8, dtype=torch.int32, device="cuda")
        out = torch.ops.oscar_amd.evict(w, kc, kc.clone(), bt, [300], [1], None, None, None, 256)
        assert out.shape == w.shape
        assert torch.ops.oscar_amd.accumulate_weights(q, None, kc, kc, bt, [0, 5], [300], 1.0, w[0], w, 256) is None
        o, lse = torch.ops.oscar_amd.attention_decode(q, None, None, kc, kc, bt, [0, 5], [300], 0.1, 256, soft_cap=3.0)
        assert o.shape == (5, 6, 256) and lse.shape == (5, 6)


@pytest.mark.gpu
def test_torch_operators_match_the_wrappers(cuda):
    from oscar_amd import ops

    c = cases.make_case([700, 300], [3, 2])
    q, k, v = (torch.from_numpy(c[x]).bfloat16().to(cuda) for x in "qkv")
    kc, vc = (torch.from_numpy(c[x]).view(torch.int8).to(cuda) for x in ("k8", "v8"))
    stage, bt = tuple(torch.from_numpy(a).to(cuda) for a in c["stage"]), torch.from_numpy(c["bt"]).to(cuda)
    slopes, qsl, seqs = slopes_of(6).to(cuda), c["qsl"], c["seqs"]
    plan = ops.plan_decode(qsl, seqs, has_new=True, num_kv_heads=1, group=6, head_dim=D, device=cuda)
    out, lse = ops.attention_decode(q, k, v, kc, vc, bt, plan, SCALE, stage, head_dim=D, soft_cap=CAP, alibi_slopes=slopes)
    got = torch.ops.oscar_amd.attention_decode(q, k, v, kc, vc, bt, qsl, seqs, SCALE, D, *stage, soft_cap=CAP, alibi_slopes=slopes)
    assert (got[0] - out).abs().max() <= 1e-2 and (got[1] - lse).abs().max() <= 1e-4  # (another plan's order)
    a, b = torch.zeros(2, 1, 800, device=cuda), torch.zeros(2, 1, 800, device=cuda)
    # a decode plan serves as the batch's lists
    ops.accumulate_weights(q, k, kc, vc, bt, plan, SCALE, lse, a, stage, head_dim=D, soft_cap=CAP, alibi_slopes=slopes)
    torch.ops.oscar_amd.accumulate_weights(q, k, kc, vc, bt, qsl, seqs, SCALE, lse, b, D, *stage, soft_cap=CAP, alibi_slopes=slopes)
    assert torch.equal(a, b)
    caches = [(kc.clone(), vc.clone(), stage[2].clone()) for _ in range(2)]
    ep = ops.plan_evict(seqs, [2, 1], block_size=BS, sink_tokens=0, recent_tokens=50, device=cuda)
    w1 = ops.evict(ep, a, caches[0][0], caches[0][1], bt, head_dim=D, stage=(*stage[:2], caches[0][2]))
    w2 = torch.ops.oscar_amd.evict(a, caches[1][0], caches[1][1], bt, seqs, [2, 1], *stage[:2], caches[1][2], D, 0, 50)
    assert torch.equal(w1, w2) and all(torch.equal(x, y) for x, y in zip(*caches))


@pytest.mark.gpu
@pytest.mark.parametrize("cap,steep", [(0.0, 0.0), (20.0, 1.0)])
@pytest.mark.parametrize("n", [1, 33, 700, 2500])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_fresh_prompt_and_its_weights(cuda, n, dtype, cap, steep):
    """The LSE of a fresh prefill (within 4e-4 of the formula's) with the prompt's own rows: every
    query gives one in all, to within that LSE, the weights' own products (3e-4) and their 1e-4."""
    from oscar_amd import ops

    gen = torch.Generator().manual_seed(n)
    q, k, v = (torch.randn(n, h, D, generator=gen).to(dtype) for h in (HQ, HK, HK))
    slopes = torch.tensor([steep * 2.0 ** (-8.0 * (h + 1) / HQ) for h in range(HQ)]) if steep else None
    score = dict(soft_cap=cap, alibi_slopes=None if slopes is None else slopes.to(cuda))
    lse = torch.full((n, HQ), 77.0, device=cuda)
    ops.attention_prefill(q.to(cuda), k.to(cuda), v.to(cuda), SCALE, head_dim=D, lse=lse, **score)
    _, want, _ = reference(q.float(), k.float(), v.float(), 0, SCALE, cap, slopes, 1)
    assert (lse.double().cpu() - want).abs().max() <= 4e-4
    kc = torch.zeros(1, BS, HK, D, dtype=torch.int8, device=cuda)
    table = torch.zeros(1, -(-n // BS), dtype=torch.int32, device=cuda)
    weights = torch.zeros(1, HK, n, device=cuda)
    ops.accumulate_weights(q.to(cuda), k.to(cuda), kc, kc, table, ops.plan_weights([0, n], [n], has_new=True, device=cuda), SCALE,
                           lse, weights, head_dim=D, **score)
    assert (weights.double().sum(-1) / (n * HQ / HK) - 1).abs().max() <= 8e-4
    assert (weights >= 0).all()


@pytest.mark.gpu
def test_pages_past_four_gigabytes(cuda):
    """The same pages at the front of a small cache and at the end of one of 4.3 GB a side: the
    same bits from attention, weights and eviction."""
    from oscar_amd import ops

    c = cases.make_case([1500, 700], [3, 1], window=False)
    q, k, v = (torch.from_numpy(c[x]).bfloat16().to(cuda) for x in "qkv")
    small = [torch.from_numpy(c[x]).view(torch.int8).to(cuda) for x in ("k8", "v8")]
    bt = torch.from_numpy(c["bt"]).to(cuda)
    pages, blocks = small[0].shape[0], (1 << 32) // small[0][0].numel() + 1000
    shift = blocks - pages
    large = [torch.empty(blocks, *x.shape[1:], dtype=torch.int8, device=cuda) for x in small]
    assert shift * large[0][0].numel() > 1 << 32
    for a, b in zip(large, small):
        a[shift:] = b
    plan = ops.plan_decode(c["qsl"], c["seqs"], has_new=True, num_kv_heads=1, group=6, head_dim=256, device=cuda)
    drop = ops.plan_evict([1500, 700], [6, 2], block_size=128, sink_tokens=7, device=cuda)

    def run(caches, table):
        out, lse = ops.attention_decode(q, k, v, *caches, table, plan, c["scale"], head_dim=256, soft_cap=20.0)
        w = ops.accumulate_weights(q, k, *caches, table, plan, c["scale"], lse, torch.zeros(2, 1, 1503, device=cuda), head_dim=256,
                                   soft_cap=20.0)
        return out, lse, w, ops.evict(drop, w, *caches, table, head_dim=256)

    want, got = run(small, bt), run(large, bt + shift)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    assert all(torch.equal(a[shift:], b) for a, b in zip(large, small))


@pytest.mark.gpu
def test_a_serving_loop(cuda):
    """Two requests: prompts, decode steps whose weights add up, an eviction, and a step over
    what is left.  Each attention is checked against a 64-bit evaluation of the cache as it
    then is; each row's weights sum to its heads' queries; the tokens of least weight go."""
    from oscar_amd import ops

    gen = torch.Generator(device=cuda).manual_seed(11)
    blocks, cols = 48, 16
    kc, vc = (torch.zeros(blocks, BS, HK, D, dtype=torch.int8, device=cuda) for _ in range(2))
    table = torch.randperm(blocks, generator=torch.Generator().manual_seed(2))[:2 * cols].view(2, cols).int().to(cuda)
    rows = 20
    stage = (torch.zeros(rows, BS, HK, D, device=cuda), torch.zeros(rows, BS, HK, D, device=cuda),
             torch.full((rows, BS), -1, dtype=torch.int64, device=cuda))
    rk, rv = (torch.from_numpy(cases.hadamard_rotation(D, s)).to(cuda) for s in (1, 2))
    angle = torch.arange(4096, dtype=torch.float64)[:, None] * 1e4 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64)
    cos_sin = torch.cat([angle.cos(), angle.sin()], 1).float().to(cuda)
    gain = torch.ones(D, device=cuda).bfloat16()
    weights = torch.zeros(2, HK, cols * BS, device=cuda)
    lengths, positions = [0, 0], [0, 0]  # cached tokens; tokens seen

    def step(counts):
        nonlocal weights
        qsl, n = [0, counts[0], sum(counts)], sum(counts)
        qkv = torch.randn(n, (HQ + 2 * HK) * D, generator=gen, device=cuda).bfloat16()
        pos = torch.cat([torch.arange(p, p + c) for p, c in zip(positions, counts)]).to(cuda)
        q, k = ops.norm_rope(qkv[:, :HQ * D].view(n, HQ, D), qkv[:, HQ * D:(HQ + HK) * D].view(n, HK, D), pos, cos_sin,
                             q_weight=gain * 2, k_weight=gain)
        v = qkv[:, (HQ + HK) * D:].view(n, HK, D).contiguous()
        seqs = [a + c for a, c in zip(lengths, counts)]
        host = table.cpu().numpy()
        at = np.concatenate([host[r, np.arange(a, b) // BS].astype(np.int64) * BS + np.arange(a, b) % BS
                             for r, (a, b) in enumerate(zip(lengths, seqs))])
        qr, kr, vr = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
        before = [x.clone() for x in (kc, vc, *stage)]
        ops.store(k, v, kc, vc, torch.from_numpy(at).to(cuda), head_dim=D, rk=rk, rv=rv, stage=stage, stage_mode=2,
                  qsl_dev=torch.tensor(qsl, dtype=torch.int32, device=cuda),
                  seqs_dev=torch.tensor(seqs, dtype=torch.int32, device=cuda), num_reqs=2, recent_tokens=128,
                  sink_tokens_eff=0, query=q, query_rot=qr, key_rot=kr, value_rot=vr)
        plan = ops.plan_decode(qsl, seqs, has_new=True, num_kv_heads=HK, group=HQ // HK, head_dim=D, device=cuda, window=(0, 128))
        out, lse = ops.attention_decode(qr, kr, vr, kc, vc, table, plan, SCALE, stage, head_dim=D, soft_cap=CAP)
        old = weights.clone()
        ops.accumulate_weights(qr, kr, kc, vc, table, plan, SCALE, lse, weights, stage, head_dim=D, soft_cap=CAP)
        # the window as the read sees it is the one after the write
        seen = tuple(x.cpu().numpy() for x in stage)
        k8, v8 = (x.view(torch.uint8).cpu().numpy() for x in (kc, vc))
        for r, (a, b) in enumerate(zip(qsl, qsl[1:])):
            hk_, hv = read_history(k8, v8, host[r], 0, lengths[r], HK, D, seen, "bf16")
            keys, values = np.concatenate([hk_, kr[a:b].float().cpu()]), np.concatenate([hv, vr[a:b].float().cpu()])
            want, want_lse, size = reference(qr[a:b].float().cpu(), keys, values, lengths[r], SCALE, CAP, None, lengths[r] + 1)
            assert ((out[a:b].double().cpu() - want).abs() <= REL_TOL * size + 1e-5).all()
            assert (lse[a:b].double().cpu() - want_lse).abs().max() <= 4e-4
            # every query gives each of its heads' keys one in all (the LSE is within 4e-4, a weight within 1e-4)
            added = (weights - old)[r].double().sum(-1)
            assert (added / (counts[r] * HQ / HK) - 1).abs().max() <= 1e-3
        assert not torch.equal(before[0], kc)
        lengths[:], positions[:] = seqs, [p + c for p, c in zip(positions, counts)]

    step([1500, 700])
    step([3, 1])
    step([1, 4])
    plan = ops.plan_evict(lengths, [6, 2], block_size=BS, sink_tokens=4, recent_tokens=128, device=cuda)
    kept_least, gone_most = [], []
    for r, (length, many) in enumerate(zip(lengths, (6, 2))):
        tail = (length - 128) // BS * BS
        for h in range(HK):
            w = weights[r, h, 4:tail].sort().values
            gone_most.append(w[many * BS - 1].item())
            kept_least.append(w[many * BS].item())
    total = weights.sum(-1)
    new = ops.evict(plan, weights, kc, vc, table, head_dim=D, stage=stage)
    for i, (r, h) in enumerate((r, h) for r in range(2) for h in range(HK)):
        end = (lengths[r] - 128) // BS * BS - (6, 2)[r] * BS
        assert new[r, h, 4:end].min().item() == kept_least[i] >= gone_most[i]
        assert (new[r, h, plan.seq_lens[r]:] == 0).all()
        assert torch.equal(new[r, h, end:plan.seq_lens[r]], weights[r, h, end + (6, 2)[r] * BS:lengths[r]])
    assert (new.sum(-1) < total).all()
    weights, table = new, plan.table(table)
    lengths = list(plan.seq_lens)
    step([2, 3])
    step([150, 1])  # over the end of a page, into one that was freed or a later one
    assert math.isfinite(weights.sum().item())
