"""Attention of the language models: sliding window with first tokens that stay visible, and learned relative position buckets.

``window_attention`` serves the causal stacks (prompts, parts of a prompt behind a cache, single tokens over a cache, training; the learned
sink logits are those of serenitymojo/models/text_encoder/gpt_oss_encoder.mojo:14-44), ``relative_attention`` the bidirectional encoders
whose layers add a learned bias for buckets of relative positions (serenitymojo/models/text_encoder/t5_encoder.mojo).

bf16 tensors with heads of 64 or 128 on a GPU run the kernels of ``csrc/text_attention*.cu``, forward and backward; other types, other
head widths and the CPU run the torch statements of ``ops.reference``. Keys and values that no query sees are not read: they may hold anything.
"""
from __future__ import annotations

import functools
import math
from typing import Optional, Union

import torch

from . import native, reference as ref

_NO_WINDOW = 1 << 30
#: what the kernels take, and their torch statements beyond: sequences and heads (a grid's extent), scales (normal fp32, times log2(e) too)
_MOST_BLOCKS, _LEAST_SCALE, _MOST_SCALE = 65535, 2.0 ** -126, 2.0 ** 127
#: by head width, the buckets that the kernels' tables hold and the distance at which the last one may begin; beyond them the torch statement runs
MAX_BUCKETS, MAX_NEAR = {64: 64, 128: 32}, {64: 512, 128: 240}


def prefix_lengths(mask: torch.Tensor) -> Optional[torch.Tensor]:
    """``kv_len`` (int32 [B]) for a padding mask [B, S] whose rows are ones and then zeros; None for any other mask. Reads one value from the device."""
    kept = mask != 0
    lengths = kept.sum(1, dtype=torch.int32)
    prefix = kept == (torch.arange(mask.shape[1], device=mask.device)[None, :] < lengths[:, None])
    return lengths if bool(prefix.all()) else None


def _check(name, q, k, v, kv_len, out):
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape:
        raise ValueError(f"{name}: q [B, Sq, H, Dh], k and v [B, Skv, Hkv, Dh]")
    if k.shape[0] != q.shape[0] or k.shape[3] != q.shape[3] or k.shape[2] == 0 or q.shape[2] % k.shape[2]:
        raise ValueError(f"{name}: k and v need q's batch and head width, and a number of heads that divides q's")
    if not (q.dtype == k.dtype == v.dtype) or not q.is_floating_point():
        raise ValueError(f"{name}: q, k and v of one floating type")
    if not (q.device == k.device == v.device):
        raise ValueError(f"{name}: q, k and v on one device")
    _per_sequence(name, "kv_len", kv_len, q)
    if out is not None and (out.shape != q.shape or out.dtype != q.dtype or out.device != q.device):
        raise ValueError(f"{name}: out must have q's shape, type and device")


def _per_sequence(name, what, t, q):
    if t is not None and (t.dtype != torch.int32 or t.shape != q.shape[:1] or t.device != q.device):
        raise ValueError(f"{name}: {what} must be int32 [B] on q's device")


def _kernels(q, k, v, scale, param, kv_len, q_start, out) -> bool:
    """Whether the kernels cover the call. They check shapes, types and devices themselves, which costs a short call less."""
    if not q.is_cuda or q.dtype is not torch.bfloat16 or q.dim() != 4 or not (scale is None or _LEAST_SCALE <= scale <= _MOST_SCALE):
        return False
    sequences, _, heads, width = q.shape
    if sequences > _MOST_BLOCKS or heads > _MOST_BLOCKS or (width != 64 and width != 128) or (param is not None and param.dtype is not torch.bfloat16 and param.dtype is not torch.float32):
        return False
    return native.use_native(q) and native.direct(*[t for t in (q, k, v, param, kv_len, q_start, out) if t is not None])


def _wants_grad(q, k, v, param) -> bool:
    return torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or (param is not None and param.requires_grad))


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: Optional[int] = None, sinks: int = 0,
                     scale: Optional[float] = None, kv_len: Optional[torch.Tensor] = None, q_start: Union[int, torch.Tensor] = 0,
                     sink_logits: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal grouped-query attention with a sliding window: q [B, Sq, H, Dh], k / v [B, Skv, Hkv, Dh] (any strides) -> [B, Sq, H, Dh].

    Query row i stands at position ``p = q_start + i`` (``q_start`` an int, or int32 [B]; 0 for a whole prompt, ``kv_len - Sq`` for the last
    tokens of a cache) and sees key j when ``j <= p``, ``p - j < window`` or ``j < sinks`` (``window`` None: all earlier keys), and
    ``j < kv_len[b]`` (int32 [B]). Query head h reads key / value head ``h // (H // Hkv)``. ``sink_logits`` [H] take part in each row's softmax
    and carry no value. A row that sees no key is zero and has no gradient. Differentiable in q, k, v and sink_logits, once.
    """
    name = "window_attention"
    if window is None:
        window = _NO_WINDOW
    elif type(window) is not int or window < 1:
        raise ValueError(f"{name}: window must be a positive int or None")
    elif window > _NO_WINDOW:
        window = _NO_WINDOW
    if type(sinks) is not int or sinks < 0:
        raise ValueError(f"{name}: sinks must be an int of at least 0")
    if sinks > _NO_WINDOW:
        sinks = _NO_WINDOW
    start, starts = 0, None
    if isinstance(q_start, torch.Tensor):
        starts = q_start
    elif type(q_start) is not int:
        raise ValueError(f"{name}: q_start must be an int or int32 [B]")
    elif q_start:
        start = max(min(q_start, _NO_WINDOW), -_NO_WINDOW)
    if scale is not None:
        scale = float(scale)
    kernels = _kernels(q, k, v, scale, sink_logits, kv_len, starts, out)
    if kernels:
        if not _wants_grad(q, k, v, sink_logits):
            return native.ops().window_attention(q, k, v, window, sinks, scale, kv_len, start, starts, sink_logits, out)
        o = native.ops().text_attention(q, k, v, sink_logits, scale, window, sinks, kv_len, start, starts, [])
        if out is None:
            return o
    _check(name, q, k, v, kv_len, out)
    _per_sequence(name, "q_start", starts, q)
    if sink_logits is not None and (sink_logits.shape != q.shape[2:3] or not sink_logits.is_floating_point() or sink_logits.device != q.device):
        raise ValueError(f"{name}: sink_logits must be [H] on q's device")
    if not kernels:
        o = ref.window_attention(q, k, v, window if window < _NO_WINDOW else None, sinks, scale, kv_len, starts if starts is not None else start, sink_logits)
    return out.copy_(o) if out is not None else o


@functools.lru_cache(maxsize=64)
def _buckets(num_buckets: int, max_distance: int):
    single, borders = ref.bucket_borders(num_buckets, max_distance)
    return [num_buckets, single, *borders]


def relative_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, max_distance: int = 128, scale: float = 1.0,
                       kv_len: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Bidirectional attention with a learned bias: q [B, Sq, H, Dh], k / v [B, Skv, H, Dh] (any strides) -> [B, Sq, H, Dh].

    ``table`` [num_buckets, H] (an even number, at least 4; the weight of the encoders' ``relative_attention_bias``) is added to the score of query i and
    key j at the bucket of j - i: half of the buckets per direction, single distances first, then distances that grow by equal factors up to
    ``max_distance``. ``kv_len`` (int32 [B]) hides the keys from there on. No ``scale`` by default, as these encoders are trained. An entry of -inf
    switches a bucket off; a row that sees no key is zero and has no gradient. Differentiable in q, k, v and table, once.
    """
    name = "relative_attention"
    if table.dim() != 2 or table.shape[0] < 4 or table.shape[0] % 2:
        raise ValueError(f"{name}: table must be [num_buckets, H], num_buckets even and at least 4")
    if type(max_distance) is not int or max_distance <= table.shape[0] // 4:
        raise ValueError(f"{name}: max_distance must be an int beyond the distances that have a bucket each ({table.shape[0] // 4})")
    scale = float(scale)
    buckets = _buckets(table.shape[0], max_distance)
    kernels = _kernels(q, k, v, scale, table, kv_len, None, out) and table.shape[0] <= MAX_BUCKETS[q.shape[3]] and buckets[-1] <= MAX_NEAR[q.shape[3]]
    if kernels:
        if not _wants_grad(q, k, v, table):
            return native.ops().relative_attention(q, k, v, table, buckets, scale, kv_len, out)
        o = native.ops().text_attention(q, k, v, table, scale, _NO_WINDOW, 0, kv_len, 0, None, buckets)
        if out is None:
            return o
    _check(name, q, k, v, kv_len, out)
    if k.shape[2] != q.shape[2]:
        raise ValueError(f"{name}: q, k and v with the same heads")
    if table.shape[1] != q.shape[2] or not table.is_floating_point() or table.device != q.device:
        raise ValueError(f"{name}: table must be [num_buckets, H] on q's device")
    if not kernels:
        o = ref.relative_attention(q, k, v, table, max_distance, scale, kv_len)
    return out.copy_(o) if out is not None else o


def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor, window: Optional[int] = None, scale: Optional[float] = None,
                     sink_logits: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal grouped-query attention of sequences that lie one behind the other: q [T, H, Dh], k / v [T, Hkv, Dh] (any strides) -> [T, H, Dh].

    Sequence b has the rows cu_seqlens[b] .. cu_seqlens[b + 1] (int32 [B + 1], not falling, on the tensors' device; a length may be zero), and its row i sees its rows
    j with ``j <= i`` and ``i - j < window`` (None: all earlier ones). Query head h reads key / value head ``h // (H // Hkv)``; ``sink_logits`` [H] take part in each row's
    softmax and carry no value. What other sequences hold does not count, NaN neither; rows of no sequence are not read, their output is zero and has no gradient.
    Ends outside the rows or falling ones are an error on the CPU; the kernels hold ends within the rows, and where they fall no sequence is seen: all is zero, and
    ``ops.check_status`` reports it.
    Differentiable in q, k, v and sink_logits, once; with a gradient wanted, sequences of up to 256 rows and windows of up to 128 are rounded less, for it is a difference of nearly equal terms.
    """
    name = "packed_attention"
    if window is None:
        window = _NO_WINDOW
    elif type(window) is not int or window < 1:
        raise ValueError(f"{name}: window must be a positive int or None")
    elif window > _NO_WINDOW:
        window = _NO_WINDOW
    if scale is not None:
        scale = float(scale)
    if (q.is_cuda and q.dtype is torch.bfloat16 and q.dim() == 3 and q.shape[2] in (64, 128) and q.shape[0] < _NO_WINDOW and q.shape[1] <= _MOST_BLOCKS and cu_seqlens.numel() <= _MOST_BLOCKS
            and (scale is None or _LEAST_SCALE <= scale <= _MOST_SCALE) and (sink_logits is None or sink_logits.dtype in (torch.bfloat16, torch.float32)) and native.use_native(q)
            and native.direct(q, k, v, cu_seqlens, sink_logits)):
        if not _wants_grad(q, k, v, sink_logits):
            return native.ops().packed_attention_fwd(q, k, v, cu_seqlens, window, scale, sink_logits)
        return native.ops().packed_attention(q, k, v, sink_logits, cu_seqlens, window, scale)
    if q.dim() != 3 or k.dim() != 3 or k.shape != v.shape:
        raise ValueError(f"{name}: q [T, H, Dh], k and v [T, Hkv, Dh]")
    if cu_seqlens.dim() != 1 or cu_seqlens.shape[0] < 1 or cu_seqlens.dtype != torch.int32 or cu_seqlens.device != q.device:
        raise ValueError(f"{name}: cu_seqlens must be int32 [B + 1] on q's device")
    _check(name, q[None], k[None], v[None], None, None)
    if sink_logits is not None and (sink_logits.shape != q.shape[1:2] or not sink_logits.is_floating_point() or sink_logits.device != q.device):
        raise ValueError(f"{name}: sink_logits must be [H] on q's device")
    return ref.packed_attention(q, k, v, cu_seqlens, window if window < _NO_WINDOW else None, scale, sink_logits)
