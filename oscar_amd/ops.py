"""Torch-facing wrappers around the C ABI (include/oscar_amd.h).

PyTorch is used for device memory and streams only; every computation runs in
liboscar_amd.so.  All functions raise when the library is missing or a launch
fails; there is no CPU fallback.
"""
from __future__ import annotations

import ctypes as C
import math
import struct
from dataclasses import dataclass

import numpy as np
import torch

from . import _lib
from ._lib import (GROUP_INTS, OSCAR_BF16, OSCAR_F16, OSCAR_F32, STAGE_INVALIDATE, STAGE_NONE,
                   STAGE_WRITE, WORK_INTS)

_DTYPES = {torch.float32: OSCAR_F32, torch.float16: OSCAR_F16, torch.bfloat16: OSCAR_BF16}


def dtype_code(dtype: torch.dtype) -> int:
    return _DTYPES[dtype]


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


# the current stream's raw handle without building a Stream object (2 us a call); a torch
# built without a GPU has none, and imports this module all the same
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream(device: torch.device) -> int:
    return _raw_stream(device.index if device.index is not None else torch.cuda.current_device())


def _require_cuda(*tensors) -> None:
    for t in tensors:
        if t is not None and t.device.type != "cuda":
            raise RuntimeError("OSCAR HIP ops need device tensors (no CPU fallback)")


_get_device = getattr(torch._C, "_cuda_getDevice", None)  # the current device's index, as above


def _device_index(*tensors) -> int:
    """The index of the device that all the tensors given (None: none) are on."""
    index = None
    for t in tensors:
        if t is not None:
            i = t.get_device()
            if i != index:
                if i < 0:
                    raise RuntimeError("OSCAR HIP ops need device tensors (no CPU fallback)")
                if index is not None:
                    raise ValueError(f"OSCAR HIP ops need all tensors on one device, got {index} and {i}")
                index = i
    return index


def _launch(name: str, index: int, *args) -> None:
    """Call the entry point `name` on the device's current stream, with the device made the
    current one (the library launches there)."""
    call = getattr(_lib.load(), name)
    if index == _get_device():
        status = call(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            status = call(*args, _raw_stream(index))
    if status:
        _lib.check(status, name)


_CACHE = struct.Struct("=QQ10q").pack  # _lib.Cache's fields


def cache_struct(k_cache: torch.Tensor, v_cache: torch.Tensor, head_dim: int) -> _lib.Cache:
    """Byte view of a packed cache pair [num_blocks, block_size, Hk, D] (int8 or bf16).  The
    kernels take the blocks, tokens and heads of K for both, so the two must have the same,
    and their slots room for the constants (K's first 32 bytes) and the codes."""
    if k_cache.ndim != 4 or v_cache.ndim != 4 or not k_cache.is_contiguous() or not v_cache.is_contiguous():
        raise ValueError("OSCAR requires contiguous [blocks, tokens, heads, bytes] caches")
    blocks, tokens, heads, width = k_cache.shape
    v_blocks, v_tokens, v_heads, v_width = v_cache.shape
    k2, v2 = width * k_cache.element_size(), v_width * v_cache.element_size()
    if v_blocks != blocks or v_tokens != tokens or v_heads != heads:
        raise ValueError(f"OSCAR requires K and V caches of the same blocks, tokens and heads, got "
                         f"{list(k_cache.shape[:3])} and {list(v_cache.shape[:3])}")
    if k2 < 32 + head_dim // 4 or v2 < head_dim // 4:
        raise ValueError(f"OSCAR slots of head_dim {head_dim} take {32 + head_dim // 4} bytes of K and {head_dim // 4} of V, "
                         f"the caches have {k2} and {v2}")
    return _lib.Cache.from_buffer_copy(_CACHE(k_cache.data_ptr(), v_cache.data_ptr(), blocks, tokens, heads, head_dim,
                                              tokens * heads * k2, heads * k2, k2, tokens * heads * v2, heads * v2, v2))


def staging_struct(stage, k_cache: torch.Tensor | None = None, head_dim: int | None = None) -> _lib.Staging | None:
    """The FP32 window arena (stage_k, stage_v, owner) as a C struct.  With the cache
    given, its geometry is checked against it (streaming_attention.py:55-65): owner
    [rows, block_size], values [rows, block_size, Hk, D], rows >= 1, all contiguous."""
    if stage is None:
        return None
    sk, sv, owner = stage
    if sk.dtype != torch.float32 or sv.dtype != torch.float32 or owner.dtype != torch.int64:
        raise ValueError("staging arena must be fp32 values and int64 owner tags")
    if not (sk.is_contiguous() and sv.is_contiguous() and owner.is_contiguous()):
        raise ValueError("Streaming staging tensors must be contiguous")
    if k_cache is not None:
        rows = owner.shape[0] if owner.ndim == 2 else 0
        want = (rows, k_cache.shape[1], k_cache.shape[2], head_dim)
        if rows < 1 or owner.shape != want[:2] or sk.shape != want or sv.shape != want:
            raise ValueError("Invalid streaming staging geometry")
    return _lib.Staging(sk.data_ptr(), sv.data_ptr(), owner.data_ptr(), owner.shape[0])


def upload(parts, device) -> list:
    """Host integer arrays (int32 / int64) to the device in ONE non-blocking copy.

    The arrays are packed at 8-byte aligned offsets into one pinned host buffer (torch's
    caching host allocator keeps the block until the copy has run, so the host never
    waits for the stream); the returned device tensors are views of one device buffer."""
    arrays = [np.ascontiguousarray(p) for p in parts]
    offsets, total = [], 0
    for a in arrays:
        if a.dtype not in (np.int32, np.int64):
            raise TypeError("upload() takes int32 or int64 arrays")
        offsets.append(total)
        total += (a.nbytes + 7) & ~7
    host = torch.empty(max(total, 8), dtype=torch.uint8, pin_memory=True)
    view = host.numpy()
    for a, o in zip(arrays, offsets):
        view[o:o + a.nbytes] = a.view(np.uint8)
    dev = host.to(device, non_blocking=True)
    out = []
    for a, o in zip(arrays, offsets):
        dt = torch.int32 if a.dtype == np.int32 else torch.int64
        out.append(dev[o:o + a.nbytes].view(dt) if a.size else torch.empty(0, dtype=dt, device=device))
    return out


class DeviceScratch:
    """Scratch of one (device, stream): last-writer claim tables, the claim epoch, the
    small store's arrival counters and the growable workspaces of the store, the decode,
    the prefill and the native step (captured decodes and prefills have their own, see
    _call_workspace).  Work enqueued on different streams gets different
    scratch, so concurrent calls never share these buffers (each is allocated while its
    stream is current, so torch's allocator orders its reuse on that stream)."""

    _by_device: dict = {}

    def __init__(self, device: torch.device):
        self.device = device
        self.step_ws = torch.empty(0, dtype=torch.uint8, device=device)
        # claim epoch lives on the device so that captured graphs replay with fresh epochs
        self.epoch_counter = torch.zeros(2, dtype=torch.int64, device=device)
        self.slot_claims = torch.zeros(0, dtype=torch.int64, device=device)
        self.seat_claims = torch.zeros(0, dtype=torch.int64, device=device)
        self.store_ws = torch.empty(0, dtype=torch.uint8, device=device)
        self.arrivals = torch.zeros(0, dtype=torch.int32, device=device)
        self.attn_ws = torch.empty(0, dtype=torch.uint8, device=device)
        self.prefill_ws = torch.empty(0, dtype=torch.uint8, device=device)

    @classmethod
    def get(cls, device: torch.device, stream: int | None = None) -> "DeviceScratch":
        """The scratch of `device` for `stream` (a raw HIP stream handle; default: the
        device's current stream, the one the caller's work goes to)."""
        index = device.index if device.index is not None else torch.cuda.current_device()
        if stream is None:
            stream = _raw_stream(index)
        key = (index, stream)
        if key not in cls._by_device:
            cls._by_device[key] = cls(torch.device("cuda", index))
        return cls._by_device[key]

    def claims(self, slots: int, seats: int):
        """Claim tables; growing one restarts both tables and the epoch from zero."""
        grow = self.slot_claims.numel() < slots or self.seat_claims.numel() < max(seats, 1)
        if grow:
            self.slot_claims = torch.zeros(max(slots, self.slot_claims.numel()), dtype=torch.int64,
                                           device=self.device)
            self.seat_claims = torch.zeros(max(seats, 1, self.seat_claims.numel()), dtype=torch.int64,
                                           device=self.device)
            self.epoch_counter.zero_()
        return self.slot_claims, self.seat_claims

    def store_workspace(self, nbytes: int) -> torch.Tensor:
        if self.store_ws.numel() < nbytes:
            self.store_ws = torch.empty(max(nbytes, 1 << 20), dtype=torch.uint8, device=self.device)
        return self.store_ws

    def store_arrivals(self, num_kv_heads: int) -> torch.Tensor:
        """Arrival counters of the one-launch store (calls of <= 64 tokens): zeroed
        once, and every call leaves them zero."""
        need = 2 * 64 * num_kv_heads
        if self.arrivals.numel() < need:
            self.arrivals = torch.zeros(need, dtype=torch.int32, device=self.device)
        return self.arrivals

    def prefill_workspace(self, nbytes: int) -> torch.Tensor:
        if self.prefill_ws.numel() < nbytes:
            self.prefill_ws = torch.empty(max(nbytes, 1 << 20), dtype=torch.uint8, device=self.device)
        return self.prefill_ws

    def attn_workspace(self, nbytes: int) -> torch.Tensor:
        if self.attn_ws.numel() < nbytes:
            self.attn_ws = torch.empty(max(nbytes, 1 << 20), dtype=torch.uint8, device=self.device)
        return self.attn_ws

    def step_workspace(self, nbytes: int) -> torch.Tensor:
        """The native decode step's workspace (rotated q / k / v, out_rot, LSE, item
        partials)."""
        if self.step_ws.numel() < max(nbytes, 1):  # never hand out an empty buffer
            self.step_ws = torch.empty(max(nbytes, 4 << 20), dtype=torch.uint8, device=self.device)
        return self.step_ws


# whether the current device's current stream captures a graph
_is_capturing = getattr(torch._C, "_cuda_isCurrentStreamCapturing", None)


def _call_workspace(index: int, kind: str, nbytes: int) -> torch.Tensor:
    """The workspace of one attention call on device `index` (kind: the DeviceScratch method):
    the stream's shared one, or, while the stream captures a graph, one of the call's own out of
    the graph's memory pool.  The graph keeps the address: the shared buffer may be replaced by
    a larger one, and be in use by its stream while the graph is replayed on another."""
    if index != _get_device():
        with torch.cuda.device(index):
            return _call_workspace(index, kind, nbytes)
    if _is_capturing():
        return torch.empty(max(nbytes, 1), dtype=torch.uint8, device=torch.device("cuda", index))
    scratch = DeviceScratch._by_device.get((index, _raw_stream(index)))
    if scratch is None:
        scratch = DeviceScratch.get(torch.device("cuda", index))
    return getattr(scratch, kind)(nbytes)


class DeviceContext:
    """The library's native context for one device (pinned + device metadata ring of the
    decode step, safe to share between streams: a ring slot is reused once the event
    recorded after its last reader has completed), created once per device and
    destroyed with the process."""

    _by_device: dict = {}

    def __init__(self, index: int):
        lib = _lib.load()
        ptr = C.c_void_p()
        _lib.check(lib.oscar_context_create_v1(index, C.byref(ptr)), "oscar_context_create_v1")
        self.ptr = ptr
        self.index = index

    @classmethod
    def get(cls, device: torch.device) -> "DeviceContext":
        index = device.index if device.index is not None else torch.cuda.current_device()
        ctx = cls._by_device.get(index)
        if ctx is None:
            ctx = cls._by_device[index] = cls(index)
        return ctx


LEAST_CAP, MOST_CAP = 2.0 ** -20, 1024.0  # the caps that the library takes


def score_struct(soft_cap, alibi_slopes, num_q_heads: int, device) -> _lib.Score | None:
    """The score function of an attention call as a C struct; None for the plain product."""
    if alibi_slopes is not None:
        if alibi_slopes.dtype != torch.float32 or alibi_slopes.shape != (num_q_heads,) \
                or not alibi_slopes.is_contiguous():
            raise ValueError(f"alibi_slopes must be a contiguous fp32 [{num_q_heads}] tensor")
        if alibi_slopes.device != device:
            raise ValueError(f"alibi_slopes are on {alibi_slopes.device}, the queries on {device}")
    if soft_cap != 0 and not LEAST_CAP <= soft_cap <= MOST_CAP:
        raise ValueError(f"soft_cap must lie in [2^-20, 1024], 0 for none, got {soft_cap}")
    if soft_cap == 0 and alibi_slopes is None:
        return None
    return _lib.Score(float(soft_cap), _ptr(alibi_slopes))


def decode_step(ctx: DeviceContext, args: "_lib.StepArgs", stream: int, scratch: DeviceScratch, score=None) -> int:
    """oscar_decode_step_v1 (oscarop_decode_step_v1 with a score function); grows the
    stream's step workspace and retries once when it is too small.  Returns 0, or
    STEP_NOT_DECODE when the batch needs the general path."""
    lib = _lib.load()
    if score is not None:
        return _scored_step(lib, ctx, args, stream, scratch, score)
    rc = lib.oscar_decode_step_v1(ctx.ptr, C.byref(args), C.c_void_p(stream))
    if rc == -28 and args.workspace_needed > args.workspace_bytes:
        ws = scratch.step_workspace(args.workspace_needed)
        args.workspace, args.workspace_bytes = ws.data_ptr(), ws.numel()
        rc = lib.oscar_decode_step_v1(ctx.ptr, C.byref(args), C.c_void_p(stream))
    if rc < 0:
        _lib.check(rc, "oscar_decode_step_v1")
    return rc


def _scored_step(lib, ctx, args, stream, scratch, score) -> int:
    for _ in range(2):
        rc = lib.oscarop_decode_step_v1(ctx.ptr, C.byref(args), C.byref(score), C.c_void_p(stream))
        if rc != -28 or args.workspace_needed <= args.workspace_bytes:
            break
        ws = scratch.step_workspace(args.workspace_needed)
        args.workspace, args.workspace_bytes = ws.data_ptr(), ws.numel()
    if rc < 0:
        _lib.check(rc, "oscarop_decode_step_v1")
    return rc


# ------------------------------------------------------------------------ store
def store(key, value, k_cache, v_cache, slot_mapping, **kw):
    """Rotate + clip + INT2 quantize + scatter (+ staging window) in one C call.

    key/value [N, Hk, D] (bf16/fp16/fp32), slot_mapping [N] int64 (negative = skip).
    rk/rv fp32 [D, D] or None for identity.  Optional query [N, Hq, D] and
    *_rot outputs receive the unclipped rotated values in the input dtype.  Keyword
    arguments as store_args.
    """
    args = store_args(key, value, k_cache, v_cache, slot_mapping, **kw)
    if args is not None:
        _lib.check(_lib.load().oscar_store_v1(C.byref(args[0]), C.c_void_p(_stream(key.device))), "oscar_store_v1")


def store_args(key, value, k_cache, v_cache, slot_mapping, *, head_dim, rk=None, rv=None,
               k_clip=0.0, v_clip=0.0, stage=None, stage_mode=STAGE_NONE, qsl_dev=None,
               seqs_dev=None, num_reqs=0, recent_tokens=0, sink_tokens_eff=0, query=None,
               query_rot=None, key_rot=None, value_rot=None):
    """The C arguments of a store (None for an empty call) and the tensors they point
    into, for oscar_store_v1 (store) or oscar_decode_write_v1 (attention_decode's
    `store`)."""
    _require_cuda(key, value, k_cache, v_cache, slot_mapping)
    n = slot_mapping.shape[0]
    if n == 0:
        return None
    lib = _lib.load()
    dev = key.device
    hk = k_cache.shape[2]
    if key.dtype not in _DTYPES or value.dtype != key.dtype:
        raise ValueError("key/value must share a float dtype")
    key = key[:n].reshape(n, hk, head_dim)
    value = value[:n].reshape(n, hk, head_dim)
    if key.stride(2) != 1 or key.stride(1) != head_dim or value.stride(2) != 1 or value.stride(1) != head_dim:
        key, value = key.contiguous(), value.contiguous()
    slot_mapping = slot_mapping.to(device=dev, dtype=torch.int64).contiguous()
    scratch = DeviceScratch.get(dev)
    cache = cache_struct(k_cache, v_cache, head_dim)
    st = staging_struct(stage, k_cache, head_dim)
    seats = 0 if st is None else st.rows * cache.block_size
    slot_claims, seat_claims = scratch.claims(cache.num_blocks * cache.block_size, seats)
    a = _lib.StoreArgs()
    a.key, a.value = key.data_ptr(), value.data_ptr()
    a.kv_dtype = _DTYPES[key.dtype]
    a.num_tokens = n
    a.key_stride_token, a.value_stride_token = key.stride(0), value.stride(0)
    if query is not None:
        query = query[:n]
        if query.stride(-1) != 1 or query.stride(-2) != head_dim:
            query = query.contiguous()
        a.query, a.num_q_heads, a.query_stride_token = query.data_ptr(), query.shape[1], query.stride(0)
    for name, r in (("rk", rk), ("rv", rv)):
        if r is not None:
            if r.dtype != torch.float32 or not r.is_contiguous() or r.shape != (head_dim, head_dim):
                raise ValueError(f"{name} must be a contiguous fp32 [{head_dim}, {head_dim}] tensor")
            setattr(a, name, r.data_ptr())
    a.k_clip_ratio, a.v_clip_ratio = float(k_clip), float(v_clip)
    a.slot_mapping = slot_mapping.data_ptr()
    a.cache = cache
    a.stage_mode = stage_mode if st is not None else STAGE_NONE
    if st is not None:
        a.staging = st
    if stage_mode == STAGE_WRITE:
        a.query_start_loc, a.seq_lens = qsl_dev.data_ptr(), seqs_dev.data_ptr()
        a.num_reqs, a.recent_tokens, a.sink_tokens_eff = num_reqs, recent_tokens, sink_tokens_eff
    for name, t in (("query_rot", query_rot), ("key_rot", key_rot), ("value_rot", value_rot)):
        if t is not None:
            if not t.is_contiguous() or t.dtype != key.dtype:
                raise ValueError(f"{name} must be contiguous in the key dtype")
            setattr(a, name, t.data_ptr())
    a.slot_claims, a.seat_claims = slot_claims.data_ptr(), seat_claims.data_ptr()
    a.epoch_counter = scratch.epoch_counter.data_ptr()
    if n >= 1 << 24:
        raise ValueError("oscar store: at most 2^24 tokens per call")
    need = lib.oscar_store_workspace_bytes_v1(n, hk, head_dim)
    ws = scratch.store_workspace(need)
    a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
    a.arrivals = scratch.store_arrivals(hk).data_ptr()
    return a, (key, value, slot_mapping, query, st, ws)


# ------------------------------------------------------------------------ rotate
def rotate(x: torch.Tensor, r: torch.Tensor, *, transpose=False, out_dtype=None, out=None):
    """x [..., D] @ R (or @ R^T) with MFMA hi/lo products; returns out_dtype (default x dtype)."""
    _require_cuda(x, r)
    d = x.shape[-1]
    rows = x.numel() // d
    x2 = x.reshape(rows, d)
    if x2.stride(1) != 1:
        x2 = x2.contiguous()
    out_dtype = out_dtype or x.dtype
    if out is None:
        out = torch.empty(*x.shape[:-1], d, dtype=out_dtype, device=x.device)
    o2 = out.reshape(rows, d)
    r = r.contiguous()
    a = _lib.RotateArgs(x2.data_ptr(), _DTYPES[x2.dtype], rows, x2.stride(0), r.data_ptr(), int(bool(transpose)),
                        o2.data_ptr(), _DTYPES[out_dtype], o2.stride(0), d)
    status = _lib.load().oscar_rotate_v1(C.byref(a), _stream(x.device))
    if status:
        _lib.check(status, "oscar_rotate_v1")
    return out


# ------------------------------------------------------------------------ head norms and rotation
def _aligned(x: torch.Tensor) -> torch.Tensor:
    """x contiguous and 16-byte aligned."""
    x = x.contiguous()
    return x if x.data_ptr() % 16 == 0 else x.clone()


def _row_stride(x: torch.Tensor, address: int, heads: int, d: int) -> int | None:
    """The token stride of x [N, heads, d] if the kernel reads it as it lies: heads next to
    each other, rows 16-byte aligned."""
    if address % 16:
        return None
    if x.is_contiguous():
        return heads * d
    s0, s1, s2 = x.stride()
    if s2 != 1 or heads > 1 and s1 != d or s0 * x.element_size() % 16:
        return None
    return s0


def norm_rope(q, k, positions, cos_sin, *, q_weight=None, k_weight=None, eps=1e-6, weight_offset=0.0,
              interleaved=False, q_out=None, k_out=None):
    """RMS norm of every query and key head, then the position rotation, in one launch.

    q [N, Hq, D] and k [N, Hk, D] of one type (bf16 / fp16 / fp32; either may be None), as
    views of the projection's rows if they are.  positions [N] int32 or int64; cos_sin
    [P, R]: row p holds the R / 2 cosines of position p, then its sines (R a multiple of
    16, at most D; values past R are only normed).  Per row of D values
    y = x / sqrt(mean(x^2) + eps) * (weight + weight_offset), weights [D] or None (no
    gain, whatever the offset); pairs (i, i + R / 2), or (2 i, 2 i + 1) if interleaved, turn by the angles.
    fp32 throughout, rounded once.  A position outside the table gives NaN rows.

    Returns (q_out, k_out): new tensors, or the ones given; q_out=q and k_out=k work in
    place.
    """
    x = k if q is None else q
    if x is None:
        raise ValueError("norm_rope needs queries or keys")
    index = _device_index(q, k, positions, cos_sin, q_weight, k_weight, q_out, k_out)
    dtype = x.dtype
    code = _DTYPES.get(dtype)
    if x.ndim != 3:
        raise ValueError("q and k must be [tokens, heads, 128 or 256]")
    n, _, d = x.shape
    if d != 256 and d != 128:
        raise ValueError("q and k must be [tokens, heads, 128 or 256]")
    if code is None or k is not x and k is not None and (k.dtype != dtype or k.ndim != 3 or k.shape[::2] != (n, d)):
        raise ValueError("q and k must share a float dtype, the token count and the head width")
    wide = positions.dtype == torch.int64
    if not wide and positions.dtype != torch.int32 or positions.shape != (n,):
        raise ValueError("positions must be [tokens] int32 or int64")
    rows, rotary = cos_sin.shape if cos_sin.ndim == 2 else (0, 0)
    cs_code = _DTYPES.get(cos_sin.dtype)
    if cs_code is None or rotary % 16 or not 16 <= rotary <= d:
        raise ValueError("cos_sin must be a float [positions, R] table, R a multiple of 16 up to the head width")
    positions, cos_sin, wtype, sides = positions.contiguous(), _aligned(cos_sin), None, []
    for name, y, weight, out in (("q", q, q_weight, q_out), ("k", k, k_weight, k_out)):
        if y is None:
            sides.append((None, 0, 0, None, None, None, 0, None))
            continue
        heads, address = y.shape[1], y.data_ptr()
        stride = _row_stride(y, address, heads, d)
        if stride is None:
            y = y.clone(memory_format=torch.contiguous_format)
            stride, address = heads * d, y.data_ptr()
        if out is None:
            out = torch.empty(n, heads, d, dtype=dtype, device=y.device)
            out_address, out_stride = out.data_ptr(), heads * d
        else:
            out_address = out.data_ptr()
            out_stride = _row_stride(out, out_address, heads, d) if out.dtype == dtype and out.shape == y.shape else None
            if out_stride is None:
                raise ValueError(f"{name}_out must have {name}'s shape and type, its heads next to each other and "
                                 "16-byte aligned rows")
        gain = None
        if weight is not None:
            if wtype is None:
                wtype = weight.dtype
            if weight.dtype != wtype or weight.shape != (d,) or wtype not in _DTYPES:
                raise ValueError("the norm weights must be [head width] of one float dtype")
            weight = _aligned(weight)
            gain = weight.data_ptr()
        sides.append((address, stride, heads, gain, out, out_address, out_stride, (y, weight)))
    (qp, qs, hq, qw, q_out, qo, qos, _), (kp, ks, hk, kw, k_out, ko, kos, _) = sides
    a = _lib.NormRopeArgs(qp, qs, hq, kp, ks, hk, n, d, code, qw, kw, OSCAR_F32 if wtype is None else _DTYPES[wtype],
                          weight_offset, eps, positions.data_ptr(), wide, cos_sin.data_ptr(), cs_code,
                          bool(interleaved), rows, rotary, qo, qos, ko, kos)
    _launch("oscarop_norm_rope_v1", index, C.byref(a))
    return q_out, k_out


# ------------------------------------------------------------------------ decode attention
@dataclass
class DecodePlan:
    """A split-K plan: host records (items, groups) and, once uploaded, their device copies."""
    host_items: np.ndarray   # int32 [num_items * WORK_INTS]
    host_groups: np.ndarray  # int32 [num_groups * GROUP_INTS]
    host_qsl: list
    host_seqs: list
    has_new: bool
    num_items: int
    num_groups: int
    partial_bytes: int
    max_group_items: int
    items: torch.Tensor | None = None   # device int32 copies
    groups: torch.Tensor | None = None
    qsl: torch.Tensor | None = None
    seqs: torch.Tensor | None = None

    def host_parts(self) -> list:
        """The arrays the kernels read, in upload() order (items, groups, qsl, seqs)."""
        return [self.host_items, self.host_groups, np.asarray(self.host_qsl, np.int32),
                np.asarray(self.host_seqs or [0], np.int32)]

    def adopt(self, device_parts: list) -> "DecodePlan":
        self.items, self.groups, self.qsl, self.seqs = device_parts
        return self


def plan_decode(qsl: list, seqs: list, *, has_new: bool, num_kv_heads: int, group: int,
                head_dim: int, device, target_items: int | None = None,
                chunk_tokens: int = 8192, window: tuple = (0, 0), upload_now: bool = True) -> DecodePlan:
    """Split-K plan (host): items of whole 32-token tiles, balanced over the CUs.

    window = (sink_tokens, recent_tokens) of the FP32 staging window, a balance hint
    (the expected window tiles go to items of their own); (0, 0) = no window.
    upload_now=False leaves the device copies to the caller (one combined upload()).
    """
    lib = _lib.load()
    nreq = len(seqs)
    qa = (C.c_int32 * (nreq + 1))(*qsl)
    sa = (C.c_int32 * max(nreq, 1))(*seqs)
    if target_items is None:
        target_items = cu_count(device)
    plan = _lib.Plan()
    sink, recent = (int(x) for x in window)
    # one call with room for any plan the target allows (at most 3 ranges per group,
    # at most 256 tiles per item); a second, exact call only if that was too small
    sub = max(1, 32 // group)  # query tokens per sub-request (32 rows per kv head)
    ngroups = num_kv_heads * sum(-(-(b - a) // sub) for a, b in zip(qsl, qsl[1:]) if b > a)
    guess = max(target_items, 1) + 3 * ngroups + sum(-(-s // 8192) for s in seqs) * num_kv_heads
    items = np.zeros(max(guess, 1) * WORK_INTS, np.int32)
    groups = np.zeros(max(ngroups, 1) * GROUP_INTS, np.int32)
    i_ptr = items.ctypes.data_as(C.POINTER(C.c_int32))
    g_ptr = groups.ctypes.data_as(C.POINTER(C.c_int32))
    n = lib.oscar_attn_plan_v1(qa, sa, nreq, int(has_new), num_kv_heads, group, head_dim,
                               chunk_tokens, target_items, sink, recent, i_ptr, guess,
                               g_ptr, max(ngroups, 1), C.byref(plan))
    if n == -28:
        items = np.zeros(max(plan.num_items, 1) * WORK_INTS, np.int32)
        i_ptr = items.ctypes.data_as(C.POINTER(C.c_int32))
        n = lib.oscar_attn_plan_v1(qa, sa, nreq, int(has_new), num_kv_heads, group, head_dim,
                                   chunk_tokens, target_items, sink, recent, i_ptr, plan.num_items,
                                   g_ptr, max(ngroups, 1), C.byref(plan))
    if n < 0:
        _lib.check(n, "oscar_attn_plan_v1")
    p = DecodePlan(items[: plan.num_items * WORK_INTS], groups[: plan.num_groups * GROUP_INTS],
                   list(qsl), list(seqs), bool(has_new), plan.num_items, plan.num_groups,
                   plan.partial_bytes, plan.max_group_items)
    if upload_now:
        p.adopt(upload(p.host_parts(), device))
    return p


_CU_COUNT: dict = {}


def cu_count(device) -> int:
    dev = torch.device(device)
    key = dev.index if dev.index is not None else torch.cuda.current_device()
    if key not in _CU_COUNT:
        _CU_COUNT[key] = torch.cuda.get_device_properties(key).multi_processor_count
    return _CU_COUNT[key]


def _plan_sizes(plan, block_size: int) -> tuple:
    """Of a plan's requests with queries: (pages of the longest history, longest length, most
    queries), worked out again only when the plan's lists or the page size are others."""
    key = (block_size, plan.has_new, tuple(plan.host_qsl), tuple(plan.host_seqs))
    known = getattr(plan, "_sizes", None)
    if known is not None and known[0] == key:
        return known[1]
    pages = longest = most = 0
    for a, b, seq in zip(plan.host_qsl, plan.host_qsl[1:], plan.host_seqs):
        if b > a:
            pages = max(pages, -(-(seq - (b - a) if plan.has_new else seq) // block_size))
            longest, most = max(longest, seq), max(most, b - a)
    sizes = pages, longest, most
    plan._sizes = key, sizes
    return sizes


def _covers(plan: DecodePlan, n: int) -> bool:
    """The plan's requests tile the rows [0, n)."""
    qsl = plan.host_qsl
    return qsl[0] == 0 and qsl[-1] == n and all(a <= b for a, b in zip(qsl, qsl[1:]))


def _check_table(table: torch.Tensor, plan: DecodePlan, block_size: int) -> None:
    """streaming_attention.py:48-53: the block table must cover every history."""
    if table.ndim != 2 or table.shape[0] < len(plan.host_seqs):
        raise ValueError("Missing request block-table rows")
    if _plan_sizes(plan, block_size)[0] > table.shape[1]:
        raise ValueError("Block table cannot cover the history")


def _rows_apart(table: torch.Tensor) -> torch.Tensor:
    """A block table as the entry points take it: int32, columns next to each other, rows not
    on top of each other (one row broadcast to all requests, a single row out of a column)."""
    if table.dtype != torch.int32:
        table = table.to(torch.int32)
    if table.ndim == 2:
        row, column = table.stride()
        if column != 1 or row < table.shape[1]:
            table = table.clone(memory_format=torch.contiguous_format)
    return table


def attention_decode(q, k_new, v_new, k_cache, v_cache, block_table, plan: DecodePlan, scale,
                     stage=None, *, head_dim, out_rot=None, lse=None, phases=0, static_scratch=False,
                     store=None, soft_cap=0.0, alibi_slopes=None):
    """Rotated-domain attention over INT2 history (+ current chunk): (out_rot fp32, lse fp32).

    q (and k_new / v_new) are bf16 or fp16; history values are rounded q_dtype(fp16(x)).
    static_scratch: call oscar_attn_decode_static_v1 (item partials in the library's
    static device array, no workspace).  store: store_args(...) of the step's write, whose
    rotated outputs are q / k_new / v_new: one oscar_decode_write_v1 call runs the store
    and the decode (a small store's quantization then rides in the merge launch).
    soft_cap, alibi_slopes [Hq] fp32: a score s (scaled) of key t for a query at position p
    becomes soft_cap tanh(s / soft_cap) + alibi_slopes[h] (t - p); 0 and None leave it, a cap
    lies in [2^-20, 1024] (a score keeps 2^-22 of it).  Positions are places in the cache: after
    an eviction a token that moved counts from the place it moved into."""
    _require_cuda(q, k_cache, v_cache, block_table)
    if store is not None and static_scratch:
        raise ValueError("store= goes with the workspace decode only")
    score = score_struct(soft_cap, alibi_slopes, q.shape[1], q.device)
    if score is not None and (store is not None or static_scratch):
        raise ValueError("soft_cap and alibi_slopes go with the plain workspace decode")
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError("OSCAR HIP attention requires bf16 or fp16 queries")
    n, hq, _ = q.shape
    dev = q.device
    if out_rot is None or lse is None:
        # rows of no request stay zero (lse -inf); the merge writes every row of a request
        all_rows = phases == 0 and plan.num_items > 0 and _covers(plan, n)
        if out_rot is None:
            out_rot = (torch.empty if all_rows else torch.zeros)(n, hq, head_dim, dtype=torch.float32, device=dev)
        if lse is None:
            lse = torch.empty(n, hq, dtype=torch.float32, device=dev)
            if not all_rows:
                lse.fill_(-math.inf)
    if plan.num_items == 0 or n == 0:
        if store is not None:
            _lib.check(_lib.load().oscar_store_v1(C.byref(store[0]), C.c_void_p(_stream(dev))), "oscar_store_v1")
        return out_rot, lse
    if q.stride(2) != 1 or q.stride(1) != head_dim:
        q = q.contiguous()
    if (k_new is None) != (v_new is None):
        raise ValueError("Both new K and V must be supplied together")
    if k_new is not None:
        if k_new.dtype != q.dtype or v_new.dtype != q.dtype:
            raise ValueError("Current K/V must match the query dtype")
        k_new, v_new = k_new.contiguous(), v_new.contiguous()
    table = block_table
    if table.get_device() != q.get_device():
        table = table.to(device=dev, dtype=torch.int32)
    table = _rows_apart(table)
    if plan.has_new != (k_new is not None):
        raise ValueError("plan and call disagree on the presence of current K/V")
    if plan.items is None:
        raise ValueError("the decode plan has not been uploaded")
    _check_table(table, plan, k_cache.shape[1])
    st = staging_struct(stage, k_cache, head_dim)
    ws = None if static_scratch else _call_workspace(q.get_device(), "attn_workspace", plan.partial_bytes)
    has_new = k_new is not None
    a = _lib.AttnArgs(q.data_ptr(), n, hq, q.stride(0), _ptr(k_new), _ptr(v_new), k_new.stride(0) if has_new else 0,
                      cache_struct(k_cache, v_cache, head_dim), table.data_ptr(), table.stride(0), plan.qsl.data_ptr(),
                      plan.seqs.data_ptr(), plan.seqs.numel(), None if st is None else C.pointer(st), scale,
                      plan.items.data_ptr(), plan.num_items, plan.groups.data_ptr(), plan.num_groups, _ptr(ws),
                      0 if ws is None else ws.numel(),
                      plan.max_group_items, out_rot.data_ptr(), lse.data_ptr(), phases, _DTYPES[q.dtype], *table.shape)
    lib, stream = _lib.load(), _stream(dev)
    if score is not None:
        _launch("oscarop_attn_decode_v1", q.get_device(), C.byref(a), C.byref(score))
    elif store is not None:
        _lib.check(lib.oscar_decode_write_v1(C.byref(store[0]), C.byref(a), stream), "oscar_decode_write_v1")
    else:
        entry = "oscar_attn_decode_static_v1" if static_scratch else "oscar_attn_decode_v1"
        _lib.check(getattr(lib, entry)(C.byref(a), stream), entry)
    return out_rot, lse


# ------------------------------------------------------------------------ prefill
def attention_prefill(q, k, v, scale, *, head_dim, history=0, k_cache=None, v_cache=None,
                      block_table_row=None, stage=None, out=None, lse=None, split=True, soft_cap=0.0,
                      alibi_slopes=None):
    """Causal GQA prefill of one request.

    q/k/v are bf16 or fp16 (history values rounded q_dtype(fp16(x))).
    history == 0: original-domain fresh-only prefill, returns [n, Hq, D] in q's dtype.
    history > 0: rotated continuation over the packed history, returns fp32 out_rot
    (and fills lse [n, Hq] when given).
    split: cut the query tiles' key ranges into balanced chunks (a larger workspace for
    their partials and one merge launch); False runs one workgroup per query tile.
    soft_cap, alibi_slopes: as in attention_decode.
    """
    _require_cuda(q, k, v)
    score = score_struct(soft_cap, alibi_slopes, q.shape[1], q.device)
    if q.dtype not in (torch.bfloat16, torch.float16) or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError("OSCAR HIP prefill requires bf16 or fp16 q/k/v of one dtype")
    n, hq, _ = q.shape
    hk = k.shape[1]
    q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    if out is None:
        out = torch.empty(n, hq, head_dim, dtype=q.dtype if history == 0 else torch.float32,
                          device=q.device)
    a = _lib.PrefillArgs()
    a.q, a.q_stride_token, a.k, a.v, a.kv_stride_token = q.data_ptr(), q.stride(0), k.data_ptr(), v.data_ptr(), k.stride(0)
    a.num_tokens, a.num_q_heads, a.num_kv_heads, a.head_dim = n, hq, hk, head_dim
    a.history = history
    keep = []
    if history > 0:
        a.cache = cache_struct(k_cache, v_cache, head_dim)
        row = block_table_row.to(device=q.device, dtype=torch.int32).contiguous()
        if math.ceil(history / k_cache.shape[1]) > row.numel():
            raise ValueError("Block table cannot cover the history")
        keep.append(row)
        a.block_table_row, a.block_table_cols = row.data_ptr(), row.numel()
        st = staging_struct(stage, k_cache, head_dim)
        if st is not None:
            keep.append(st)
            a.staging = C.pointer(st)
    a.scale = float(scale)
    a.out, a.out_stride_token = out.data_ptr(), out.stride(0)
    a.q_dtype = _DTYPES[q.dtype]
    if lse is not None:
        a.lse = lse.data_ptr()
    lib = _lib.load()
    # the history values plus the partials of the balanced split (0 for calls too small
    # to split and without history)
    need = lib.oscar_prefill_workspace_bytes_v2(history, n, hq, hk, head_dim)
    if need < 0:
        raise ValueError("OSCAR HIP prefill: unsupported sizes")
    if not split:
        need = lib.oscar_prefill_workspace_bytes_v1(history, hk, head_dim)
    if need > 0:
        # the size asked for, not the shared buffer's (which an earlier call may have
        # grown past v1's size: the call would then split)
        ws = _call_workspace(q.get_device(), "prefill_workspace", need)
        a.workspace, a.workspace_bytes = ws.data_ptr(), need
    if score is not None:
        _launch("oscarop_attn_prefill_v1", q.get_device(), C.byref(a), C.byref(score))
        return out
    _lib.check(lib.oscar_attn_prefill_v1(C.byref(a), C.c_void_p(_stream(q.device))), "oscar_attn_prefill_v1")
    return out


# ------------------------------------------------------------------------ accumulated weights
@dataclass
class WeightsPlan:
    """The requests of a batch, on the host and on the device, as accumulate_weights takes
    them (a DecodePlan of the same batch serves as well)."""
    host_qsl: list
    host_seqs: list
    has_new: bool
    qsl: torch.Tensor    # device int32
    seqs: torch.Tensor


def _request_lists(qsl, seqs, has_new) -> tuple[list, list]:
    qsl, seqs = [int(x) for x in qsl], [int(x) for x in seqs]
    if len(qsl) != len(seqs) + 1 or qsl[0] < 0 or any(b < a for a, b in zip(qsl, qsl[1:])):
        raise ValueError("query starts must be one more than the lengths and must not decrease")
    if any(s < 0 or has_new and s < b - a for a, b, s in zip(qsl, qsl[1:], seqs)):
        raise ValueError("Sequence length must cover its query chunk")
    return qsl, seqs


def plan_weights(qsl, seqs, *, has_new: bool, device) -> WeightsPlan:
    """The lists of a batch (query starts, lengths) for accumulate_weights, uploaded once for
    all layers."""
    qsl, seqs = _request_lists(qsl, seqs, has_new)
    dev = upload([np.asarray(qsl, np.int32), np.asarray(seqs or [0], np.int32)], device)
    return WeightsPlan(qsl, seqs, bool(has_new), *dev)


def accumulate_weights(q, k_new, k_cache, v_cache, block_table, plan, scale, lse, weights, stage=None, *, head_dim,
                       soft_cap=0.0, alibi_slopes=None):
    """Add to weights [requests, Hk, columns] (fp32) the attention weight that each token of
    each request received: weights[r, h, t] += sum over r's queries and the query heads of
    KV head h of exp(score - lse).

    q, k_new, the caches, block_table, scale, stage, soft_cap and alibi_slopes as
    attention_decode took them for this batch, lse [n, Hq] (fp32) as it returned it (a row
    with -inf adds nothing).  After a fresh prompt's attention_prefill(lse=...), history 0:
    its unrotated q and k.  plan: plan_weights(...) or the batch's plan_decode(...).  Request
    r is row r of block_table and of weights; weights is updated in place and returned: the
    same bits for calls of the same sizes (requests, heads, longest length, most queries,
    columns), equal to fp32 roundings for others.
    """
    if plan.qsl is None:
        raise ValueError("the plan has not been uploaded")
    index = _device_index(q, k_new, k_cache, v_cache, block_table, lse, weights, plan.qsl, plan.seqs, *(stage or ()))
    score = score_struct(soft_cap, alibi_slopes, q.shape[1], q.device)
    code = _DTYPES.get(q.dtype)
    if code is None or code == OSCAR_F32:
        raise ValueError("OSCAR HIP attention requires bf16 or fp16 queries")
    if q.ndim != 3 or q.shape[2] != head_dim:
        raise ValueError("q must be [tokens, heads, head_dim]")
    n, hq, _ = q.shape
    hk, reqs, bs = k_cache.shape[2], len(plan.host_seqs), k_cache.shape[1]
    if plan.has_new != (k_new is not None):
        raise ValueError("plan and call disagree on the presence of current K")
    if plan.host_qsl[-1] > n:
        raise ValueError("the plan has more queries than the call")
    if k_new is not None:
        if k_new.dtype != q.dtype or k_new.shape[1:] != (hk, head_dim) or k_new.shape[0] < plan.host_qsl[-1]:
            raise ValueError("Current K must match the queries' type and the cache's heads")
        k_new = k_new.contiguous()
    if lse.dtype != torch.float32 or lse.shape != (n, hq):
        raise ValueError("lse must be fp32 [tokens, query heads]")
    _, longest, most = _plan_sizes(plan, bs)
    head_stride, request_stride = _weight_strides("weights", weights, reqs, hk, longest)
    if reqs == 0 or n == 0 or longest == 0:
        return weights
    table = _rows_apart(block_table)
    _check_table(table, plan, bs)
    if q.stride(2) != 1 or q.stride(1) != head_dim:
        q = q.contiguous()
    st = staging_struct(stage, k_cache, head_dim)
    lse = lse.contiguous()
    rows = n if k_new is None else min(n, k_new.shape[0])  # what a plan's lists on the device may reach
    a = _lib.WeightsArgs(q.data_ptr(), rows, hq, q.stride(0), _ptr(k_new), 0 if k_new is None else k_new.stride(0),
                         cache_struct(k_cache, v_cache, head_dim), table.data_ptr(), table.stride(0), *table.shape,
                         plan.qsl.data_ptr(), plan.seqs.data_ptr(), reqs, code, longest, most,
                         None if st is None else C.pointer(st), scale, lse.data_ptr(), weights.data_ptr(), request_stride,
                         head_stride, weights.shape[2], None, 0)
    need = _lib.load().oscarop_attn_weights_workspace_bytes_v1(C.byref(a))
    if need > 0:
        ws = torch.empty(need, dtype=torch.uint8, device=q.device)  # a captured call keeps its own
        a.workspace, a.workspace_bytes = ws.data_ptr(), need
    _launch("oscarop_attn_weights_v1", index, C.byref(a), None if score is None else C.byref(score))
    return weights


def _weight_strides(name: str, w: torch.Tensor, reqs: int, hk: int, longest: int) -> tuple:
    """(head, request) strides of weights for at least reqs requests of up to `longest` tokens."""
    if w.dtype != torch.float32 or w.ndim != 3 or w.shape[0] < reqs or w.shape[1] != hk \
            or w.stride(2) != 1 and w.shape[2] > 1:
        raise ValueError(f"{name} must be fp32 [requests, KV heads, columns], columns next to each other")
    if longest > w.shape[2]:
        raise ValueError(f"{name} has {w.shape[2]} columns for {longest} tokens")
    head = w.stride(1) if hk > 1 else w.shape[2]
    return head, w.stride(0) if reqs > 1 else hk * head


# ------------------------------------------------------------------------ eviction
@dataclass
class EvictPlan:
    """How many pages each request of a batch gives up, for all layers of a model.

    seq_lens: the lengths afterwards.  freed[r]: the columns (first, last + 1) of request r's
    row of table(...) that hold its free pages."""
    seq_lens: list
    freed: list
    lengths: list        # before
    longest: int         # of them
    max_drop: int        # tokens
    block_size: int
    requests: torch.Tensor   # device int32 [requests, 4]: length, sink, tail, dropped tokens

    def table(self, block_table: torch.Tensor) -> torch.Tensor:
        """The block table after the last layer's evict: each request's kept pages in their
        order, then its free ones."""
        bs, many = self.block_size, len(self.lengths)
        if block_table.ndim != 2 or block_table.shape[0] < many:
            raise ValueError("Missing request block-table rows")
        if -(-self.longest // bs) > block_table.shape[1]:
            raise ValueError("Block table cannot cover the history")
        length, _, tail, drop = self.requests.to(torch.int64).t()[..., None]
        pages, end, gone = -(-length // bs), (tail - drop) // bs, drop // bs
        col = torch.arange(block_table.shape[1], device=block_table.device)
        source = torch.where(col < end, col, torch.where(col < pages - gone, col + gone,
                                                         torch.where(col < pages, col - pages + gone + end, col)))
        out = block_table.clone()
        out[:many] = torch.gather(block_table[:many], 1, source)
        return out


def plan_evict(seq_lens, drop_pages, *, block_size: int, sink_tokens: int = 0, recent_tokens: int = 0, device) -> EvictPlan:
    """Plan to take drop_pages[r] whole pages out of request r of length seq_lens[r] (host
    lists; 0: the request keeps all).  The first sink_tokens and the last recent_tokens stay,
    the latter with all of their pages; a request that has too little between them is refused."""
    lengths, pages = [int(x) for x in seq_lens], [int(x) for x in drop_pages]
    if len(lengths) != len(pages):
        raise ValueError("one page count for each length")
    if block_size < 1 or sink_tokens < 0 or recent_tokens < 0:
        raise ValueError("block size, sink and recent tokens must not be negative")
    records, freed = [], []
    for r, (length, many) in enumerate(zip(lengths, pages)):
        if length < 0 or many < 0:
            raise ValueError(f"request {r}: negative length or page count")
        tail = max(length - recent_tokens, 0) // block_size * block_size
        if many and tail - sink_tokens < many * block_size:
            raise ValueError(f"request {r}: {many} pages of {block_size} to drop, {max(tail - sink_tokens, 0)} tokens "
                             "between its first and its last ones")
        drop = many * block_size
        records.append([length, sink_tokens, tail, drop] if many else [length, 0, 0, 0])
        freed.append((-(-length // block_size) - many, -(-length // block_size)))
    dev, = upload([np.asarray(records, np.int32).reshape(-1)], device)
    return EvictPlan([n - q[3] for n, q in zip(lengths, records)], freed, lengths, max(lengths, default=0), max((q[3] for q in records), default=0),
                     int(block_size), dev.view(-1, 4))


def evict(plan: EvictPlan, weights, k_cache, v_cache, block_table, *, head_dim, stage=None, weights_out=None):
    """Drop the tokens of least accumulated weight from one layer's cache, whole pages at a
    time; returns the weights by new position ([requests, Hk, columns], zero from the new
    length on; weights_out if given, which must not overlap weights).

    plan: plan_evict(...) of the batch.  Per request and KV head the plan's tokens of least
    weight between the first and the last ones go (equal weights: the later token first; NaN
    counts as the largest); the kept tokens of the last pages before the recent ones move
    into their places (keys of attention have no order; with alibi_slopes they have one: a
    token that moved then counts from its new place, those before the new end are nearer by
    the dropped tokens).  A place that is written loses its FP32 window copy.
    The caches and the owner tags of `stage` change in place, block_table does not: after the
    last layer plan.table(block_table) is the new one, plan.seq_lens the new lengths.  The
    pages between must be the request's own.
    """
    index = _device_index(weights, k_cache, v_cache, block_table, weights_out, plan.requests, *(stage or ()))
    cache = cache_struct(k_cache, v_cache, head_dim)
    reqs, hk, bs, longest = len(plan.lengths), cache.num_kv_heads, cache.block_size, plan.longest
    if plan.block_size != bs:
        raise ValueError(f"the plan is for pages of {plan.block_size} tokens, the cache has {bs}")
    if weights_out is None:
        weights_out = torch.empty(weights.shape, dtype=torch.float32, device=weights.device)
    head, request = _weight_strides("weights", weights, reqs, hk, longest)
    out_head, out_request = _weight_strides("weights_out", weights_out, reqs, hk, longest)
    if weights.shape != weights_out.shape:
        raise ValueError("weights_out must have the shape of weights")
    if reqs < weights.shape[0]:
        weights_out[reqs:].copy_(weights[reqs:])
    if reqs == 0 or weights.shape[2] == 0:
        return weights_out
    table = _rows_apart(block_table)
    if table.ndim != 2 or table.shape[0] < reqs:
        raise ValueError("Missing request block-table rows")
    if -(-longest // bs) > table.shape[1]:
        raise ValueError("Block table cannot cover the history")
    st = staging_struct(stage, k_cache, head_dim)
    need = _lib.load().oscarop_evict_workspace_bytes_v1(reqs, hk, plan.max_drop)
    ws = torch.empty(max(need, 0), dtype=torch.uint8, device=weights.device)  # a captured call keeps its own
    a = _lib.EvictArgs(weights.data_ptr(), request, head, weights.shape[2], weights_out.data_ptr(), out_request, out_head,
                       cache, table.data_ptr(), table.stride(0), *table.shape, plan.requests.data_ptr(), reqs, 0,
                       plan.max_drop, None if st is None else C.pointer(st), ws.data_ptr(), ws.numel())
    _launch("oscarop_evict_v1", index, C.byref(a))
    return weights_out
