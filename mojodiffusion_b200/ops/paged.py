"""Keys and values of many sequences in pages, and attention over them: what a batch of prompts of different lengths is served from.

A pool [pages, Hkv, P, Dh] holds P positions of one sequence per page; ``block_table`` [B, width] (int32) names the pages of each sequence in order. Pages
are bf16, or 8 bits: e4m3 values in units of a power of two per page and key head, kept as a byte (e8m0, 2^(byte - 127)) in ``k_scale`` /
``v_scale`` [pages, Hkv] (uint8). e4m3 keeps three bits behind the point at any size, so such a unit costs no precision; when later tokens of a
page need a larger one, what the page holds is brought to it.

``paged_append`` brings new keys and values there, normalised per head and rotated on the way, and rotates the queries of the same tokens; ``paged_attention``
reads them, for one token or a few of each sequence or for parts of prompts (the cached decoding of serenitymojo/llm/decoder.mojo:1-150 and
serenitymojo/llm/sqa.mojo:1-116, for a batch of sequences of different lengths).

bf16 tensors with heads of 64 or 128 and pages of 16, 32, 64 or 128 positions run the kernels of ``csrc/paged*.cu`` on a GPU; other types and sizes and the CPU run the torch
statements of ``ops.reference``. A page number outside the pool, or a position without a page, is an error on the CPU; the kernels skip it and report it
(``ops.check_status``). So they do with ends of sequences that fall or lie outside the rows: there the largest end so far counts, and none passes the last one. Neither operator has a gradient.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from . import native, reference as ref

_SIZES = (16, 32, 64, 128)


def _check_pages(name, x, k_pages, v_pages, block_table, k_scale, v_scale, B):
    if k_pages.dim() != 4 or k_pages.shape != v_pages.shape or k_pages.dtype != v_pages.dtype or min(k_pages.shape) == 0:
        raise ValueError(f"{name}: k_pages and v_pages must be [pages, Hkv, P, Dh] of one type")
    N, G, P, D = k_pages.shape
    for t in (k_pages, v_pages):
        if t.stride(3) != 1 or (P > 1 and t.stride(2) != D):
            raise ValueError(f"{name}: the [P, Dh] block of a page and head must be contiguous")
    if x.shape[-1] != D:
        raise ValueError(f"{name}: the pages have another head width")
    if k_pages.dtype == torch.float8_e4m3fn:
        for s in (k_scale, v_scale):
            if s is None or s.shape != (N, G) or s.dtype != torch.uint8 or s.device != x.device:
                raise ValueError(f"{name}: pages of 8 bits need k_scale and v_scale, uint8 [pages, Hkv]")
    elif k_scale is not None or v_scale is not None or k_pages.dtype != x.dtype:
        raise ValueError(f"{name}: pages of the tensors' own type without scales, or float8_e4m3fn with them")
    if block_table.dim() != 2 or block_table.shape[0] != B or block_table.dtype != torch.int32:
        raise ValueError(f"{name}: block_table must be int32 [B, width]")
    for t in (k_pages, v_pages, block_table):
        if t.device != x.device:
            raise ValueError(f"{name}: all tensors on one device")


def _no_gradient(name, *tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise ValueError(f"{name} has no gradient: call it under torch.no_grad(), or on detached tensors")


def _kernels(x, k_pages, *others) -> bool:
    """Whether the kernels cover the call. They check shapes, types and devices themselves, which costs a short call less."""
    if not x.is_cuda or x.dtype is not torch.bfloat16 or k_pages.dim() != 4 or x.shape[-1] not in (64, 128) or k_pages.shape[2] not in _SIZES:
        return False
    return native.use_native(x) and native.direct(x, k_pages, *others)


def paged_append(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor, start: torch.Tensor,
                 cos: torch.Tensor, sin: torch.Tensor, cu_seqlens: Optional[torch.Tensor] = None, k_scale: Optional[torch.Tensor] = None,
                 v_scale: Optional[torch.Tensor] = None, q: Optional[torch.Tensor] = None, q_norm: Optional[torch.Tensor] = None,
                 k_norm: Optional[torch.Tensor] = None, eps: float = 1e-6, keys: bool = False) -> Union[None, torch.Tensor, Tuple[Optional[torch.Tensor], torch.Tensor]]:
    """Keys and values of new tokens into the pages, in place; the rotated queries [T, H, Dh] of the same tokens where ``q`` is given (else None). With ``keys`` a pair:
    these and the normalised, rotated keys [T, Hkv, Dh] in k's type, for the attention of whole prompts.

    k, v [T, Hkv, Dh] and q [T, H, Dh] (any strides) hold the sequences' new rows one behind the other: sequence b has the rows
    cu_seqlens[b] .. cu_seqlens[b + 1] (int32 [B + 1], not falling; None: one row each, T = B), which take the positions start[b], start[b] + 1, ... (int32 [B]).
    Per head: root-mean-square norm with the weight ``q_norm`` / ``k_norm`` [Dh] where given (``eps`` inside the root), then the halves (a, b) become
    (a cos - b sin, b cos + a sin) with row p of ``cos`` / ``sin`` [positions, Dh / 2] (fp32) for position p; values stay as they are. All in fp32, rounded once.
    A page that gets its first token takes its scales anew, whatever it held before. Infinities in k or v become NaN in 8 bits and do not count for the scale.
    Rows of no sequence are not read, and zero in the results. A page that tokens go to must belong to one sequence.
    """
    if _kernels(k, k_pages, v, q, v_pages, block_table, start, cos, sin, cu_seqlens, k_scale, v_scale, q_norm, k_norm):
        found = native.ops().paged_append(k, v, k_pages, v_pages, block_table, start, cos, sin, cu_seqlens, k_scale, v_scale, q, q_norm, k_norm, eps, keys)
        return found if keys else found[0]
    name = "paged_append"
    if k.dim() != 3 or k.shape != v.shape or k.dtype != v.dtype or not k.is_floating_point() or k.shape[1] == 0 or k.device != v.device:
        raise ValueError(f"{name}: k and v must be [T, Hkv, Dh] of one floating type on one device")
    T, G, D = k.shape
    B = start.shape[0] if start.dim() == 1 else -1
    if start.dtype != torch.int32 or B < 0 or start.device != k.device:
        raise ValueError(f"{name}: start must be int32 [B] on k's device")
    if cu_seqlens is None:
        if T != B:
            raise ValueError(f"{name}: without cu_seqlens every sequence has one row")
    elif cu_seqlens.dtype != torch.int32 or cu_seqlens.shape != (B + 1,) or cu_seqlens.device != k.device:
        raise ValueError(f"{name}: cu_seqlens must be int32 [B + 1] on k's device")
    _check_pages(name, k, k_pages, v_pages, block_table, k_scale, v_scale, B)
    if k_pages.shape[1] != G or D % 2:
        raise ValueError(f"{name}: the pages have other heads, or the head width is odd")
    if cos.dim() != 2 or cos.shape != sin.shape or cos.shape[1] != D // 2 or cos.dtype != torch.float32 or sin.dtype != torch.float32 or cos.device != k.device or sin.device != k.device:
        raise ValueError(f"{name}: cos and sin must be fp32 [positions, Dh / 2] on k's device")
    if q is not None and (q.dim() != 3 or q.shape[0] != T or q.shape[2] != D or q.shape[1] == 0 or q.shape[1] % G or q.dtype != k.dtype or q.device != k.device):
        raise ValueError(f"{name}: q must be [T, H, Dh] of k's type, with a number of heads that k's divides")
    for w in (q_norm, k_norm):
        if w is not None and (w.shape != (D,) or not w.is_floating_point() or w.device != k.device):
            raise ValueError(f"{name}: q_norm and k_norm must be [Dh] on k's device")
    if q is None and q_norm is not None:
        raise ValueError(f"{name}: q_norm without q")
    _no_gradient(name, k, v, q, q_norm, k_norm, k_pages, v_pages)
    with torch.no_grad():
        found = ref.paged_append(k, v, k_pages, v_pages, block_table, start, cos, sin, cu_seqlens, k_scale, v_scale, q, q_norm, k_norm, float(eps))
    return found if keys else found[0]


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor, kv_len: torch.Tensor,
                    scale: Optional[float] = None, k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None,
                    max_len: Optional[int] = None) -> torch.Tensor:
    """Causal grouped-query attention over the pages: q [B, Sq, H, Dh] (any strides) -> [B, Sq, H, Dh].

    The pages of sequence b hold ``kv_len[b]`` positions (int32 [B]), those of the queries among them: query row i stands at position kv_len[b] - Sq + i and sees
    the keys up to its own position. Query head h reads key head ``h // (H // Hkv)``. A row before the first position is zero. ``max_len`` (int): no sequence is longer, and
    what lies behind is not seen; parts of prompts take a workspace of this size (all that the table has room for by default). Slots behind a sequence's
    end are not read: they may hold anything. A value of infinity that a query sees gives NaN, and a value that is not finite may reach the other queries of its sequence in the same call.
    """
    if max_len is not None and (type(max_len) is not int or max_len < 0):
        raise ValueError("paged_attention: max_len must be an int of at least 0")
    if _kernels(q, k_pages, v_pages, block_table, kv_len, k_scale, v_scale):
        return native.ops().paged_attention(q, k_pages, v_pages, block_table, kv_len, scale, k_scale, v_scale, max_len)
    name = "paged_attention"
    if q.dim() != 4 or not q.is_floating_point() or q.shape[2] == 0:
        raise ValueError(f"{name}: q must be floating [B, Sq, H, Dh]")
    _check_pages(name, q, k_pages, v_pages, block_table, k_scale, v_scale, q.shape[0])
    if q.shape[2] % k_pages.shape[1]:
        raise ValueError(f"{name}: the pages need a number of heads that divides q's")
    if kv_len.dtype != torch.int32 or kv_len.shape != q.shape[:1] or kv_len.device != q.device:
        raise ValueError(f"{name}: kv_len must be int32 [B] on q's device")
    scale = q.shape[3] ** -0.5 if scale is None else float(scale)
    if not 2.0 ** -126 <= scale <= 2.0 ** 126:
        raise ValueError(f"{name}: scale must be positive, and normal in fp32")
    _no_gradient(name, q, k_pages, v_pages)
    with torch.no_grad():
        return ref.paged_attention(q, k_pages, v_pages, block_table, kv_len, scale, k_scale, v_scale, max_len)
