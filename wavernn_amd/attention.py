"""Self-attention of the forward models' transformer blocks (models/common_layers.py:148-185), forward and backward, and the
learned relative position bias by buckets that it applies without a dense mask.

``attention(q, k, v, ...)`` is the part of ``nn.MultiheadAttention`` between its projections; ``forward_models.FFTBlock`` calls
it with the attention path ``'fused'``.  ``RelativePositionBias`` holds the table of a position bias: called, it gives the dense
``[heads, q_len, k_len]`` tensor that ``nn.MultiheadAttention`` takes as an additive mask; given to ``attention`` as ``bias_table`` it
never becomes one.  The kernels run in libwrnn_mi355.so (include/wrnn_mi355.h states the formulas); there is no CPU fallback.

Types: float32 and bfloat16.  All sums, maxima and exponentials are held in 32 bits; in bfloat16 the probabilities and the scores'
gradients are rounded where they enter a matrix product.  The same inputs give the same bits, gradients included.
"""
from __future__ import annotations

import ctypes as C
import functools
import math
import struct
from typing import Optional

import torch
import torch.nn as nn
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib

_DTYPES = {torch.float32: 0, torch.bfloat16: 1}   # WRNN_FLOAT32, WRNN_BFLOAT16
MAX_DISTANCE, MAX_BUCKETS, MAX_HEAD_DIM = 1024, 256, 256


@functools.lru_cache(maxsize=64)
def _edges(num_buckets: int, max_distance: int, bidirectional: bool):
    """(edges as a list, the same as a host int32 array).  A distance d at or above E = side / 2 goes to bucket
    E + floor(log(d / E) / log(max_distance / E) * (side - E)); edge k is the first d with d^n E^k >= max_distance^k E^n, n = side - E,
    found in whole numbers because the logarithms come out a hair low or high where a border falls on a whole distance."""
    side = num_buckets // 2 if bidirectional else num_buckets
    if not 2 <= num_buckets <= MAX_BUCKETS or (bidirectional and (num_buckets % 2 or side < 2)):
        raise ValueError(f"num_buckets must be in 2..{MAX_BUCKETS}, and even and at least 4 with two sides, got {num_buckets}")
    if not side // 2 < max_distance <= MAX_DISTANCE:
        raise ValueError(f"max_distance must be in {side // 2 + 1}..{MAX_DISTANCE}, got {max_distance}")
    e = side // 2
    n = side - e
    edges, d = [], e
    for k in range(1, n):
        while d ** n * e ** k < max_distance ** k * e ** n:
            d += 1
        edges.append(d)
    return edges, (C.c_int32 * max(1, len(edges)))(*edges)


def bucket_edges(num_buckets: int = 32, max_distance: int = 128, bidirectional: bool = True) -> list:
    """The distances at which each bucket above the exact ones begins (``bucket_edges`` of the C ABI)."""
    return list(_edges(num_buckets, max_distance, bidirectional)[0])


def _on_gpu(t: torch.Tensor, what: str) -> None:
    if t.device.type != 'cuda':
        raise RuntimeError(f"wavernn_amd.{what} runs only on an MI355X (HIP) device; there is no CPU fallback")


def has_tangents(*tensors: Optional[torch.Tensor]) -> bool:
    """Whether there is a dual tensor of forward-mode differentiation among them."""
    return forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def _no_tangents(*tensors: Optional[torch.Tensor]) -> None:
    """A dual tensor asks for no gradient and would come through without its tangent."""
    if has_tangents(*tensors):
        raise RuntimeError("wavernn_amd.attention has no forward-mode derivatives")


def _rows(t: torch.Tensor) -> torch.Tensor:
    """The kernels take any strides of batch, head and position; rows are contiguous, hold whole fours of elements (16 bytes at
    least) and start on the bytes of four.  A copy, padded with zeros, where that does not hold."""
    s, n = t.stride(), t.shape
    if (s[3] == 1 and not n[3] % 4 and (n[3] > 4 or t.element_size() == 4) and not t.data_ptr() % (4 * t.element_size()) and s[2] < 1 << 22
            and not ((s[0] % 4 and n[0] != 1) or (s[1] % 4 and n[1] != 1) or (s[2] % 4 and n[2] != 1))):
        return t
    pad = max(-n[3] % 4, 16 // t.element_size() - n[3])
    # (pad keeps the order of a tensor whose heads lie innermost)
    return nn.functional.pad(t, (0, pad)).contiguous() if pad else t.clone(memory_format=torch.contiguous_format)


@functools.lru_cache(maxsize=1024)
def _dense(shape, stride):
    """Strides of a dense tensor of that shape whose batch / head / position order in memory is the given strides': the projections
    around attention then need no copy."""
    order = sorted(range(3), key=lambda i: (-stride[i], i))
    out, n = [0, 0, 0, 1], shape[3]
    for i in reversed(order):
        out[i] = n
        n *= max(shape[i], 1)
    return tuple(out)


def _empty_like(t: torch.Tensor) -> torch.Tensor:
    return torch.empty_strided(t.shape, _dense(t.shape, t.stride()), dtype=t.dtype, device=t.device)


# wrnn_attention_desc and wrnn_attention_grads as bytes: a call's time on the host is mostly the filling of these
_DESC = struct.Struct("11i f 3P 9q P q 4P")
_GRADS = struct.Struct("7P 15q")


def _ptr(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


class _Desc(bytes):
    """A wrnn_attention_desc, with the array of bucket edges whose address it holds: the cache of rules may drop its own reference at any time."""
    edges = None


def _desc(q, k, v, table, key_mask, key_lens, q_start, causal, scale, max_distance, bidirectional):
    B, H, Tq, D = q.shape
    buckets, edges = 0, None
    if table is not None:
        buckets = table.shape[0]
        edges = _edges(buckets, max_distance, bidirectional)[1]
    desc = _Desc(_DESC.pack(_DTYPES[q.dtype], B, H, k.shape[1], Tq, k.shape[2], D, causal, buckets, max_distance, bidirectional, scale,
                            q.data_ptr(), k.data_ptr(), v.data_ptr(), *q.stride()[:3], *k.stride()[:3], *v.stride()[:3], _ptr(key_mask),
                            0 if key_mask is None else key_mask.stride(0), _ptr(key_lens), _ptr(q_start), _ptr(table),
                            0 if edges is None else C.addressof(edges)))
    desc.edges = edges
    return desc


class _on:
    """The tensor's device as the current one for a library call; nothing to do where it is already."""
    __slots__ = ("guard",)

    def __init__(self, device: torch.device):
        self.guard = None if device.index == torch.cuda.current_device() else torch.cuda.device(device)

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()

    def __exit__(self, *e):
        if self.guard is not None:
            self.guard.__exit__(*e)


def _stream(device: torch.device) -> int:
    return torch._C._cuda_getCurrentRawStream(device.index)    # current_stream(device).cuda_stream without the object: 2 us a call


def _space(size: int, device: torch.device) -> Optional[torch.Tensor]:
    return torch.empty(size, dtype=torch.uint8, device=device) if size else None


def _forward(desc, q, lse, stats):
    lib = _lib.load()
    out = _empty_like(q)
    size = lib.wrnn_attention_workspace_bytes(desc)
    space = _space(size, q.device)
    if lib.wrnn_attention_forward_stats(desc, out.data_ptr(), _lib.I64x3(*out.stride()[:3]), _ptr(lse), _ptr(stats), _ptr(space), size,
                                        _stream(q.device)):
        _lib.check(1, "wrnn_attention_forward_stats")
    return out


class _Attention(torch.autograd.Function):

    @staticmethod
    def forward(ctx, q, k, v, table, key_mask, key_lens, q_start, causal, scale, max_distance, bidirectional, want_lse):
        with _on(q.device):
            lse = torch.empty(q.shape[:3], dtype=torch.float32, device=q.device) if want_lse else None
            stats = torch.empty(2, *q.shape[:3], dtype=torch.float32, device=q.device)
            desc = _desc(q, k, v, table, key_mask, key_lens, q_start, causal, scale, max_distance, bidirectional)
            out = _forward(desc, q, lse, stats)
        ctx.rule = (causal, scale, max_distance, bidirectional)
        ctx.save_for_backward(q, k, v, table, key_mask, key_lens, q_start, out, stats)
        if want_lse:
            ctx.mark_non_differentiable(lse)
        ctx.set_materialize_grads(False)    # lse gets none: no tensor of zeros for it
        return out, lse

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, _):
        if dout is None:    # nothing that was computed from out passed a gradient on
            return (None,) * 12
        q, k, v, table, key_mask, key_lens, q_start, out, stats = ctx.saved_tensors
        want_table = table is not None and ctx.needs_input_grad[3]
        B, H, Tq, _ = q.shape
        if not (B and H and Tq):
            return (torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v), torch.zeros_like(table) if want_table else None) + (None,) * 8
        lib = _lib.load()
        with _on(q.device):
            # saved-tensor hooks (offloading, checkpointing) hand other tensors back than were saved, in other places and strides
            q, k, v, out, dout = _rows(q), _rows(k), _rows(v), _rows(out), _rows(dout)
            if key_mask is not None and key_mask.stride(1) != 1:
                key_mask = key_mask.contiguous()
            stats, table, key_lens, q_start = (None if t is None else t.contiguous() for t in (stats, table, key_lens, q_start))
            desc = _desc(q, k, v, table, key_mask, key_lens, q_start, *ctx.rule)
            dq, dk, dv, dtable = _empty_like(q), None, None, None
            if ctx.needs_input_grad[1] or ctx.needs_input_grad[2]:
                dk, dv = _empty_like(k), _empty_like(v)
            if want_table:
                dtable = torch.empty_like(table)
            zero = (0, 0, 0)
            grads = _GRADS.pack(out.data_ptr(), 0, dout.data_ptr(), dq.data_ptr(), _ptr(dk), _ptr(dv), _ptr(dtable), *out.stride()[:3],
                                *dout.stride()[:3], *dq.stride()[:3], *(zero if dk is None else dk.stride()[:3]),
                                *(zero if dv is None else dv.stride()[:3]))
            size = lib.wrnn_attention_backward_workspace_bytes(desc)
            space = _space(size, q.device)
            if lib.wrnn_attention_backward_stats(desc, grads, stats.data_ptr(), space.data_ptr(), size, _stream(q.device)):
                _lib.check(1, "wrnn_attention_backward_stats")
        return (dq, dk, dv, dtable) + (None,) * 8


def _whole(t: Optional[torch.Tensor], B: int, q: torch.Tensor, name: str) -> Optional[torch.Tensor]:
    if t is None:
        return None
    if t.dtype not in (torch.int32, torch.int64) or tuple(t.shape) != (B,) or t.device != q.device:
        raise ValueError(f"{name} must be an int32 or int64 tensor [{B}] on {q.device}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t.clamp(-(1 << 30), 1 << 30).to(torch.int32) if t.dtype == torch.int64 else t.contiguous()


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, key_mask: Optional[torch.Tensor] = None,
              key_lens: Optional[torch.Tensor] = None, q_start: Optional[torch.Tensor] = None, causal: bool = False,
              scale: Optional[float] = None, bias_table: Optional[torch.Tensor] = None, max_distance: int = 128,
              bidirectional: bool = True, return_lse: bool = False):
    """softmax(scale * q k^T + bias) v over the allowed keys; differentiable in q, k, v and bias_table.

    q [B, H, Tq, D], k and v [B, Hkv, Tk, D] with H a multiple of Hkv (head h reads key head h // (H // Hkv)), D up to 256, any
    strides.  The result has q's shape and its order in memory.

    key_mask [B, Tk] bool: True leaves a key out (``key_padding_mask`` of nn.MultiheadAttention).  key_lens [B]: keys at or past a
    row's length are left out.  causal: query i of row b sees keys up to position i + q_start[b]; q_start [B] defaults to Tk - Tq, the
    queries being the last positions.  A query that is left no key gives zeros and takes part in no gradient.  What lies at keys that are left
    out for a whole row is never used, NaN and infinities included.  (An infinity at a key in use gives NaN where the formula in
    float32 would keep it.)
    scale: 1 / sqrt(D) by default.
    bias_table [num_buckets, H] (``RelativePositionBias.weight``) adds table[bucket(j - (i + q_start[b])), h]; max_distance and
    bidirectional are its rule.  -inf in a table leaves its distances out.
    Differentiable backward, once; forward-mode derivatives and the transforms of torch.func are refused.
    return_lse: also the log of each query's sum of exponentials, [B, H, Tq] float32, -inf for a query without keys (no gradient)."""
    _on_gpu(q, "attention")
    _no_tangents(q, k, v, bias_table)
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape or q.shape[0] != k.shape[0] or q.shape[3] != k.shape[3]:
        raise ValueError(f"expected q [B,H,Tq,D] and k, v [B,Hkv,Tk,D], got {tuple(q.shape)}, {tuple(k.shape)} and {tuple(v.shape)}")
    if q.dtype not in _DTYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError(f"attention takes float32 or bfloat16, the same for q, k and v, got {q.dtype}, {k.dtype} and {v.dtype}")
    dev = q.device
    if k.device != dev or v.device != dev:
        raise RuntimeError("q, k and v must be on the same device")
    B, H, Tq, D = q.shape
    if not 1 <= D <= MAX_HEAD_DIM:
        raise ValueError(f"head dimension {D} is outside 1..{MAX_HEAD_DIM}")
    if k.shape[1] == 0 or H % k.shape[1]:
        raise ValueError(f"{H} heads do not share {k.shape[1]} key heads evenly")
    if key_mask is not None:
        if key_mask.dtype != torch.bool or tuple(key_mask.shape) != (B, k.shape[2]) or key_mask.device != dev:
            raise ValueError(f"key_mask must be a bool tensor [{B}, {k.shape[2]}] on {dev}, got {key_mask.dtype} {tuple(key_mask.shape)} "
                             f"on {key_mask.device}")
        if key_mask.stride(1) != 1 and key_mask.shape[1] > 1:
            key_mask = key_mask.contiguous()
    key_lens, q_start = _whole(key_lens, B, q, "key_lens"), _whole(q_start, B, q, "q_start")
    if bias_table is not None:
        if bias_table.dim() != 2 or bias_table.shape[1] != H or bias_table.device != dev or bias_table.dtype not in _DTYPES:
            raise ValueError(f"bias_table must be a float32 or bfloat16 tensor [num_buckets, {H}] on {dev}, got {bias_table.dtype} "
                             f"{tuple(bias_table.shape)} on {bias_table.device}")
        bias_table = bias_table.float().contiguous()
        _edges(bias_table.shape[0], max_distance, bidirectional)   # checks the rule
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    q, k, v = _rows(q), _rows(k), _rows(v)
    out, lse = _run(q, k, v, bias_table, key_mask, key_lens, q_start, causal, scale, max_distance, bidirectional, return_lse)
    out = out if out.shape[3] == D else out[..., :D]
    return (out, lse) if return_lse else out


def _run(q, k, v, bias_table, key_mask, key_lens, q_start, causal, scale, max_distance, bidirectional, want_lse):
    # (a trace records the function, not what the library does inside)
    if torch.jit.is_tracing() or torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad
                                                              or (bias_table is not None and bias_table.requires_grad)):
        return _Attention.apply(q, k, v, bias_table, key_mask, key_lens, q_start, causal, scale, max_distance, bidirectional, want_lse)
    with _on(q.device):
        lse = torch.empty(q.shape[:3], dtype=torch.float32, device=q.device) if want_lse else None
        out = _forward(_desc(q, k, v, bias_table, key_mask, key_lens, q_start, causal, scale, max_distance, bidirectional), q, lse, None)
    return out, lse


class _RelativeBias(torch.autograd.Function):

    @staticmethod
    def forward(ctx, table, q_len, k_len, start, max_distance, bidirectional):
        ctx.rule = (table.shape[1], q_len, k_len, start, table.shape[0], max_distance, bidirectional)
        lib = _lib.load()
        with _on(table.device):
            out = torch.empty(table.shape[1], q_len, k_len, dtype=table.dtype, device=table.device)
            _lib.check(lib.wrnn_relative_bias_forward(table.data_ptr(), _DTYPES[table.dtype], *ctx.rule, _edges(table.shape[0], max_distance, bidirectional)[1],
                                                      out.data_ptr(), _stream(table.device)),
                       "wrnn_relative_bias_forward")
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        H, q_len, k_len, _, buckets, max_distance, bidirectional = ctx.rule
        if not (H and q_len and k_len):
            return (dout.new_zeros(buckets, H),) + (None,) * 5
        lib = _lib.load()
        with _on(dout.device):
            dout = dout.contiguous()
            dtable = torch.empty(buckets, H, dtype=dout.dtype, device=dout.device)
            size = lib.wrnn_relative_bias_workspace_bytes(H, q_len, k_len, buckets, max_distance)
            space = torch.empty(size, dtype=torch.uint8, device=dout.device)
            _lib.check(lib.wrnn_relative_bias_backward(dout.data_ptr(), _DTYPES[dout.dtype], *ctx.rule, _edges(buckets, max_distance, bidirectional)[1],
                                                       dtable.data_ptr(), space.data_ptr(), size,
                                                       _stream(dout.device)), "wrnn_relative_bias_backward")
        return (dtable,) + (None,) * 5


def relative_position_bias(table: torch.Tensor, q_len: int, k_len: int, *, q_start: Optional[int] = None, max_distance: int = 128,
                           bidirectional: bool = True) -> torch.Tensor:
    """table [num_buckets, H] -> [H, q_len, k_len] of the table's type: table[bucket(j - (i + q_start)), h]; q_start defaults to
    k_len - q_len.  Differentiable in the table."""
    q_len, k_len = int(q_len), int(k_len)
    start = k_len - q_len if q_start is None else int(q_start)
    if q_len < 0 or k_len < 0:
        raise ValueError(f"negative length ({q_len}, {k_len})")
    if max(q_len, k_len) > 1 << 28 or abs(start) > 1 << 29:
        raise ValueError(f"lengths are at most 2^28 and q_start is within +-2^29, got {q_len}, {k_len} and {start}")
    _on_gpu(table, "relative_position_bias")
    if table.dim() != 2 or table.dtype not in _DTYPES:
        raise TypeError(f"expected a float32 or bfloat16 table [num_buckets, heads], got {table.dtype} {tuple(table.shape)}")
    _edges(table.shape[0], max_distance, bidirectional)
    return _RelativeBias.apply(table.contiguous(), q_len, k_len, start, max_distance, bool(bidirectional))


class RelativePositionBias(nn.Module):
    """A learned bias on attention scores by the distance from query to key: exact buckets near, logarithmic ones up to
    ``max_distance``, one for everything beyond; with ``bidirectional`` half of them for keys behind the query.  Build extension, not
    in the reference."""

    def __init__(self, heads: int, num_buckets: int = 32, max_distance: int = 128, bidirectional: bool = True):
        super().__init__()
        _edges(num_buckets, max_distance, bidirectional)
        self.max_distance, self.bidirectional = max_distance, bidirectional
        self.weight = nn.Parameter(torch.empty(num_buckets, heads).normal_(std=0.02))

    def forward(self, q_len: int, k_len: int, q_start: Optional[int] = None) -> torch.Tensor:
        return relative_position_bias(self.weight, q_len, k_len, q_start=q_start, max_distance=self.max_distance,
                                      bidirectional=self.bidirectional)

    def extra_repr(self) -> str:
        return f"heads={self.weight.shape[1]}, num_buckets={self.weight.shape[0]}, max_distance={self.max_distance}, bidirectional={self.bidirectional}"
