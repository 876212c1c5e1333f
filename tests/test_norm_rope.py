"""Head norms with the position rotation (ops.norm_rope): refusals on the CPU, values against
a 64-bit evaluation on the GPU.

Tolerance: the kernel computes in fp32 and rounds once.  A sum of squares takes at most 13
roundings (8 in a lane, 5 between lanes), its mean, eps, root and reciprocal 4 more (half of
the sum's error remains under the root), the two products and the rotation 5: below 2^-19 of
|a| + |b| of the rotated pair (of |y| where nothing turns).  The output's rounding adds half
a step of the value.
"""
import ctypes as C

import pytest
import torch

from oscar_amd import _lib

HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def reference(x, weight, positions, cos_sin, eps, offset, interleaved):
    """(y, the magnitude |a| + |b| that an error is relative to), in 64 bits."""
    x, r, half = x.double(), cos_sin.shape[1], cos_sin.shape[1] // 2
    y = x / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    y = y * (1.0 if weight is None else weight.double() + offset)
    table = cos_sin.double()[positions.long()][:, None]
    cos, sin = table[..., :half], table[..., half:]
    first, second = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, half), slice(half, r))
    a, b = y[..., first].clone(), y[..., second].clone()
    size = y.abs()
    size[..., first] = size[..., second] = a.abs() + b.abs()
    y[..., first], y[..., second] = a * cos - b * sin, b * cos + a * sin
    return y, size


def check(got, want, size):
    tol = HALF_STEP[got.dtype] * want.abs() + 2.0 ** -19 * size
    if got.dtype == torch.float16:
        tol = tol + 2.0 ** -25  # half a step of a subnormal
    assert (got.double() - want).abs().le(tol).all(), (got.double() - want).abs().sub(tol).max()


def table(rows, r, dtype=torch.float32, device="cpu"):
    inv = 1e4 ** (-torch.arange(0, r, 2, dtype=torch.float64) / r)
    angle = torch.arange(rows, dtype=torch.float64)[:, None] * inv
    return torch.cat([angle.cos(), angle.sin()], 1).to(dtype).to(device)


# ------------------------------------------------------------------ refusals (no launch)
def args(**changes):
    """Arguments that pass every check but launch nothing on their own: addresses are never read."""
    a = _lib.NormRopeArgs()
    fixed = dict(q=1 << 12, q_stride_token=1536, num_q_heads=6, k=2 << 12, k_stride_token=256, num_kv_heads=1, num_tokens=3,
                 head_dim=256, dtype=_lib.OSCAR_BF16, eps=1e-6, positions=3 << 12, cos_sin=4 << 12, cos_sin_dtype=0,
                 cos_sin_rows=10, rotary_dim=64, q_out=5 << 12, q_out_stride_token=1536, k_out=6 << 12,
                 k_out_stride_token=256)
    for name, value in {**fixed, **changes}.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("changes,message", [
    (dict(head_dim=192), "head_dim 192 unsupported"),
    (dict(num_tokens=-1), "negative size"),
    (dict(dtype=3), "types must be"),
    (dict(cos_sin_dtype=-1), "types must be"),
    (dict(q_weight=7 << 12, weight_dtype=5), "types must be"),
    (dict(eps=-1.0), "eps"),
    (dict(eps=float("nan")), "eps"),
    (dict(rotary_dim=0), "rotary_dim"),
    (dict(rotary_dim=24), "rotary_dim"),
    (dict(rotary_dim=272), "rotary_dim"),
    (dict(num_tokens=1 << 29), "too many rows"),
    (dict(q=None), "missing pointer"),
    (dict(k_out=None), "missing pointer"),
    (dict(positions=None), "missing pointer"),
    (dict(cos_sin_rows=0), "missing pointer"),
    (dict(q=(1 << 12) + 8), "aligned"),
    (dict(k_stride_token=257), "aligned"),
    (dict(cos_sin=(4 << 12) + 4), "aligned"),
    (dict(q_out_stride_token=0), "overlap"),
    (dict(k_out_stride_token=128), "overlap"),
])
def test_refusals(changes, message):
    lib = _lib.load()
    assert lib.oscarop_norm_rope_v1(C.byref(args(**changes)), None) == -22
    assert message in lib.oscar_last_error().decode()


@pytest.mark.parametrize("changes", [dict(num_tokens=1 << 45, num_q_heads=1 << 18, num_kv_heads=1 << 18), dict(num_tokens=1 << 61, num_q_heads=7),
                                     dict(num_q_heads=1 << 62, num_kv_heads=1 << 62), dict(num_q_heads=(1 << 63) - 1)])
def test_sizes_whose_product_wraps_around_are_refused(changes):
    lib = _lib.load()
    assert lib.oscarop_norm_rope_v1(C.byref(args(**changes)), None) == -22
    assert "too many rows" in lib.oscar_last_error().decode()


def test_empty_calls_succeed_without_a_launch():
    lib = _lib.load()
    assert lib.oscarop_norm_rope_v1(C.byref(args(num_tokens=0, q=None, positions=None)), None) == 0
    assert lib.oscarop_norm_rope_v1(C.byref(args(num_q_heads=0, num_kv_heads=0)), None) == 0
    assert lib.oscarop_norm_rope_v1(None, None) == -22


def test_wrapper_refusals():
    from oscar_amd import ops

    q, pos = torch.zeros(2, 2, 128), torch.zeros(2, dtype=torch.int64)
    with pytest.raises(ValueError, match="queries or keys"):
        ops.norm_rope(None, None, pos, table(4, 32))
    with pytest.raises(RuntimeError, match="device tensors"):
        ops.norm_rope(q, None, pos, table(4, 32))


# ------------------------------------------------------------------ values
CASES = [
    # tokens, hq, hk, d, dtype, rotary, interleaved, offset, weights, cos dtype
    (1, 6, 1, 256, torch.bfloat16, 64, False, 1.0, "same", torch.float32),
    (17, 6, 1, 256, torch.bfloat16, 256, False, 0.0, "fp32", torch.bfloat16),
    (33, 12, 2, 256, torch.float16, 96, True, 0.0, "none", torch.float16),
    (5, 16, 2, 128, torch.float16, 128, False, 1.0, "same", torch.float32),
    (301, 3, 5, 128, torch.float32, 16, True, 0.0, "same", torch.float32),
    (129, 1, 1, 128, torch.float32, 48, False, 0.0, "none", torch.bfloat16),
    (4099, 7, 3, 256, torch.bfloat16, 32, True, 1.0, "fp32", torch.float32),
    # four heads per lane group (rows of 40 MB and more), seven and nine heads of a token
    (12001, 5, 2, 256, torch.float16, 64, False, 0.0, "same", torch.float32),
    (9999, 8, 1, 128, torch.float32, 128, True, 0.0, "fp32", torch.float16),
]


@pytest.mark.gpu
@pytest.mark.parametrize("n,hq,hk,d,dtype,rotary,interleaved,offset,weights,cos_dtype", CASES)
@pytest.mark.parametrize("in_place", [False, True])
def test_values(cuda, n, hq, hk, d, dtype, rotary, interleaved, offset, weights, cos_dtype, in_place):
    from oscar_amd import ops

    gen = torch.Generator(device=cuda).manual_seed(n + d)
    row = torch.randn(n, (hq + 2 * hk) * d, generator=gen, device=cuda).to(dtype)
    row[:, ::29] *= 7
    q, k = row[:, :hq * d].view(n, hq, d), row[:, hq * d:(hq + hk) * d].view(n, hk, d)
    tail = row[:, (hq + hk) * d:].clone()
    wtype = torch.float32 if weights == "fp32" else dtype
    qw, kw = (None if weights == "none" else torch.randn(d, generator=gen, device=cuda).to(wtype) for _ in "qk")
    cos_sin = table(500, rotary, cos_dtype, cuda)
    positions = torch.randint(0, 500, (n,), generator=gen, device=cuda)
    positions = positions.int() if n % 2 else positions
    want = [reference(x, w, positions, cos_sin, 1e-5, offset, interleaved) for x, w in ((q, qw), (k, kw))]
    out = dict(q_out=q, k_out=k) if in_place else {}
    got = ops.norm_rope(q, k, positions, cos_sin, q_weight=qw, k_weight=kw, eps=1e-5, weight_offset=offset,
                        interleaved=interleaved, **out)
    for x, (y, size) in zip(got, want):
        check(x, y, size)
    assert torch.equal(row[:, (hq + hk) * d:], tail)  # the values beside them stay


@pytest.mark.gpu
def test_edges(cuda):
    """Positions outside the table, zero rows, infinities, one side only, odd strides."""
    from oscar_amd import ops

    d, cos_sin = 128, table(10, 64, device=cuda)
    x = torch.randn(6, 2, d, device=cuda)
    x[1] = 0
    x[2, 0, 5] = float("inf")
    positions = torch.tensor([0, 9, 3, 10, -1, 1 << 40], device=cuda)
    q, k = ops.norm_rope(x, None, positions, cos_sin, eps=0.0)
    assert k is None
    assert q[3:].isnan().all() and q[2, 0].isnan().any() and q[1].isnan().all()
    want, size = reference(x[:1], None, positions[:1], cos_sin, 0.0, 0.0, False)
    check(q[:1], want, size)
    _, k = ops.norm_rope(None, x, positions.clamp(0, 9), cos_sin)
    assert (k[1] == 0).all() and not k[3:].isnan().any()
    # transposed heads, a misaligned view, a broadcast row: read as they are
    for view in (x.transpose(0, 1).contiguous().transpose(0, 1), torch.cat([x.flatten()[:1], x.flatten()])[1:].view(6, 2, d),
                 x[:1].expand(6, 2, d)):
        got, _ = ops.norm_rope(view, None, positions.clamp(0, 9), cos_sin)
        want, size = reference(view, None, positions.clamp(0, 9), cos_sin, 1e-6, 0.0, False)
        finite = want.isfinite()
        check(torch.where(finite, got, 0), torch.where(finite, want, 0), torch.where(finite, size, 0))
    empty, _ = ops.norm_rope(x[:0], None, positions[:0], cos_sin)
    assert empty.shape == (0, 2, d)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [3, 9001])
@pytest.mark.parametrize("gain", ["neither", "q", "k"])
def test_a_missing_gain_takes_no_offset(cuda, n, gain):
    """Norms without a gain beside ones whose weights are stored around zero (offset 1)."""
    from oscar_amd import ops

    gen = torch.Generator(device=cuda).manual_seed(n)
    q, k = (torch.randn(n, h, 128, generator=gen, device=cuda) for h in (5, 3))
    w = torch.randn(128, generator=gen, device=cuda)
    qw, kw = (w if gain == side else None for side in "qk")
    cs, positions = table(50, 64, device=cuda), torch.randint(0, 50, (n,), generator=gen, device=cuda)
    got = ops.norm_rope(q, k, positions, cs, q_weight=qw, k_weight=kw, eps=1e-5, weight_offset=1.0)
    for x, y, weight in zip(got, (q, k), (qw, kw)):
        check(x, *reference(y, weight, positions, cs, 1e-5, 1.0, False))


@pytest.mark.gpu
def test_wrapper_refusals_on_the_device(cuda):
    from oscar_amd import ops

    q, pos, cs = torch.zeros(4, 2, 128, device=cuda), torch.zeros(4, dtype=torch.int64, device=cuda), table(4, 32, device=cuda)
    for kw in (dict(positions=pos[:3]), dict(positions=pos.float()), dict(cos_sin=cs[:, :24]), dict(k=q.half()),
               dict(k=q[:3]), dict(q=q[..., :64]), dict(q_weight=pos[:4]), dict(q_out=q.half()),
               dict(q_out=q.transpose(0, 1).contiguous().transpose(0, 1)), dict(q_out=q[:1].expand(4, 2, 128)),
               dict(q_weight=torch.ones(128, device=cuda), k_weight=torch.ones(128, device=cuda).half())):
        with pytest.raises(ValueError):
            ops.norm_rope(**{**dict(q=q, k=q, positions=pos, cos_sin=cs), **kw})
    with pytest.raises(RuntimeError):
        ops.norm_rope(q, None, pos.cpu(), cs)


@pytest.mark.gpu
def test_captured_and_on_another_stream(cuda):
    from oscar_amd import ops

    x = torch.randn(9, 3, 256, device=cuda).bfloat16()
    pos, cs, out = torch.arange(9, device=cuda), table(32, 64, device=cuda), torch.empty_like(x)
    want, _ = ops.norm_rope(x, None, pos, cs)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, _ = ops.norm_rope(x, None, pos, cs)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.norm_rope(x, None, pos, cs, q_out=out)
    for step in range(3):
        pos.add_(1)
        graph.replay()
        want, _ = ops.norm_rope(x, None, pos, cs)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
