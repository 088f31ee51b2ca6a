"""Several sequences of different lengths at once: a pool of key / value pages for all layers of a decoder, and generation over it.

A sequence takes pages as it grows and gives them back when it ends, so that a batch of prompts needs no common length and no padding: prompts run packed one
behind the other (``ops.packed_attention``), their keys and values go to the pages on the way (``ops.paged_append``), and each step decodes one token of every
sequence over its pages (``ops.paged_attention``). Per sequence the behaviour is that of the cached decoder for one prompt (serenitymojo/llm/decoder.mojo:1-150), with
angles in fp32 instead of the model's type."""
from __future__ import annotations

from typing import Dict, List, Optional, Sequence

import torch

from .. import ops
from ..models.layers import own_parameters
from ..models.text.qwen3 import Qwen3Config, _Norm, scaled_inv_freq


class PagedKVCache:
    """``pages`` pages of ``page_size`` positions for every layer, in ``dtype``: the model's own type, or ``torch.float8_e4m3fn`` with a scale per page and key head.
    Sequences are numbers that the caller chooses. On a GPU a bf16 model with heads of 64 or 128 runs the kernels with pages of 16, 32, 64 or 128 positions; with other
    sizes the torch statements run, one sequence after the other, which takes many times as long."""

    def __init__(self, cfg: Qwen3Config, pages: int, dtype=torch.bfloat16, device=None, page_size: int = 64):
        if pages < 1 or page_size < 1:
            raise ValueError("PagedKVCache: at least one page of at least one position")
        L, G, D = cfg.num_hidden_layers, cfg.num_key_value_heads, cfg.head_dim
        self.cfg, self.page_size, self.device = cfg, page_size, torch.device(device if device is not None else "cpu")
        eight = dtype == torch.float8_e4m3fn
        self.k, self.v = (torch.zeros(L, pages, G, page_size, D, dtype=torch.uint8 if eight else dtype, device=device) for _ in range(2))
        if eight:
            self.k, self.v = self.k.view(dtype), self.v.view(dtype)
        self.k_scale, self.v_scale = (torch.ones(L, pages, G, dtype=torch.uint8, device=device) if eight else None for _ in range(2))
        self.free = list(range(pages))[::-1]
        self.pages: Dict[int, List[int]] = {}
        self.lengths: Dict[int, int] = {}
        self._angles = None

    def reserve(self, sequence: int, length: int) -> None:
        """Pages for ``length`` positions of a sequence in all (a new one starts empty)."""
        mine = self.pages.get(sequence, [])
        missing = -(-length // self.page_size) - len(mine)
        if missing > len(self.free):
            raise RuntimeError("KV cache is full")
        self.pages[sequence] = mine + [self.free.pop() for _ in range(missing)]
        self.lengths.setdefault(sequence, 0)

    def release(self, sequence: int) -> None:
        self.give_back(sequence, None)

    def give_back(self, sequence: int, kept: Optional[int]) -> None:
        """All pages of a sequence but the first ``kept``; None: the sequence itself ends."""
        pages = self.pages.pop(sequence)
        self.free += pages[kept or 0:][::-1]
        if kept is None:
            del self.lengths[sequence]
        else:
            self.pages[sequence] = pages[:kept]

    def table(self, sequences: Sequence[int]) -> torch.Tensor:
        """int32 [B, width]: the pages of the sequences. Places that a shorter sequence does not have name page 0 and are not read."""
        width = max([len(self.pages[s]) for s in sequences], default=0)
        return torch.tensor([self.pages[s] + [0] * (width - len(self.pages[s])) for s in sequences], dtype=torch.int32, device=self.device).reshape(len(sequences), width)

    def angles(self, positions: int):
        """cos and sin [at least ``positions``, head_dim / 2] in fp32, formed in 64 bits: angles of far positions have few bits left in 32. The tables grow by doubling, so that
        a sequence that gets longer token by token rarely waits for new ones."""
        if self._angles is None or self._angles[0].shape[0] < positions:
            inv = scaled_inv_freq(self.cfg.head_dim, self.cfg.rope_theta, self.cfg.rope_scaling).double()
            a = torch.arange(1 << (max(positions, 64) - 1).bit_length(), dtype=torch.float64)[:, None] * inv[None]
            self._angles = a.cos().float().to(self.device), a.sin().float().to(self.device)
        return self._angles

    def layer(self, i: int) -> dict:
        """The pages of a layer, as the operators take them."""
        return dict(k_pages=self.k[i], v_pages=self.v[i], k_scale=None if self.k_scale is None else self.k_scale[i], v_scale=None if self.v_scale is None else self.v_scale[i])


def _layers(enc, x, attend):
    """The decoder's layers over rows x [T, hidden]; ``attend(layer number, attention module, q, k, v, norm weights)`` -> [T, H, Dh]."""
    c = enc.cfg
    for i, l in enumerate(enc.model.layers):
        a = l.self_attn
        h = l.input_layernorm(x)
        q, k, v = (p(h).view(-1, n, c.head_dim) for p, n in ((a.q_proj, c.num_attention_heads), (a.k_proj, c.num_key_value_heads), (a.v_proj, c.num_key_value_heads)))
        norms = {}
        if c.qk_norm:
            own = [own_parameters(n, _Norm) for n in (a.q_norm, a.k_norm)]
            if None not in own and all("weight" in p for p in own) and a.q_norm.eps == a.k_norm.eps:
                norms = dict(q_norm=own[0]["weight"], k_norm=own[1]["weight"], eps=a.q_norm.eps)
            else:                                          # modules that a program hooked or replaced run themselves
                q, k = a.q_norm(q), a.k_norm(k)
        x = x + a.o_proj(attend(i, q, k, v, norms).reshape(x.shape[0], -1))
        x = x + l.mlp(l.post_attention_layernorm(x))
    return x


@torch.no_grad()
def paged_prefill(enc, cache: PagedKVCache, sequences: Sequence[int], prompts: Sequence[Sequence[int]]) -> torch.Tensor:
    """Whole prompts of new sequences, packed -> hidden state of the last token of each [B, hidden]. After an error the cache is as it was: no sequence has begun."""
    if any(len(p) == 0 for p in prompts) or any(cache.lengths.get(s, 0) for s in sequences) or len(set(sequences)) != len(sequences) or len(sequences) != len(prompts):
        raise ValueError("paged_prefill: a prompt of at least one token for each of several new sequences")
    held = {s: len(cache.pages[s]) for s in sequences if s in cache.pages}
    try:
        x = _prefill(enc, cache, sequences, prompts)
    except BaseException:
        for s in reversed(sequences):
            if s in cache.pages:
                cache.give_back(s, held.get(s))
        raise
    for s, p in zip(sequences, prompts):
        cache.lengths[s] = len(p)
    return x


def _prefill(enc, cache, sequences, prompts):
    dev = cache.device
    for s, p in zip(sequences, prompts):
        cache.reserve(s, len(p))
    ends = [0]
    for p in prompts:
        ends.append(ends[-1] + len(p))
    cu = torch.tensor(ends, dtype=torch.int32, device=dev)
    table, start = cache.table(sequences), torch.zeros(len(prompts), dtype=torch.int32, device=dev)
    cos, sin = cache.angles(max([len(p) for p in prompts], default=1))

    def attend(i, q, k, v, norms):
        q, k = ops.paged_append(k, v, block_table=table, start=start, cos=cos, sin=sin, cu_seqlens=cu, q=q, keys=True, **norms, **cache.layer(i))
        return ops.packed_attention(q, k, v, cu)

    x = _layers(enc, enc.model.embed_tokens(torch.tensor([t for p in prompts for t in p], dtype=torch.long, device=dev)), attend)
    return x[cu[1:].long() - 1]


@torch.no_grad()
def paged_step(enc, cache: PagedKVCache, sequences: Sequence[int], tokens: torch.Tensor) -> torch.Tensor:
    """The next token of each sequence, tokens [B] -> hidden [B, hidden]; every sequence grows by one."""
    if tokens.shape != (len(sequences),) or len(set(sequences)) != len(sequences):
        raise ValueError("paged_step: one token for each of several sequences")
    for s in sequences:
        cache.reserve(s, cache.lengths[s] + 1)
    start = torch.tensor([cache.lengths[s] for s in sequences], dtype=torch.int32, device=cache.device)
    kv_len, table, longest = start + 1, cache.table(sequences), max([cache.lengths[s] for s in sequences], default=0) + 1
    cos, sin = cache.angles(longest)

    def attend(i, q, k, v, norms):
        pages = cache.layer(i)
        q = ops.paged_append(k, v, block_table=table, start=start, cos=cos, sin=sin, q=q, **norms, **pages)
        return ops.paged_attention(q[:, None], block_table=table, kv_len=kv_len, max_len=longest, **pages)[:, 0]

    x = _layers(enc, enc.model.embed_tokens(tokens), attend)
    for s in sequences:
        cache.lengths[s] += 1
    return x
