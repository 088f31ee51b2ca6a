"""Prompt-expansion language model support: KV-cached incremental decode over the Qwen3 stack (:mod:`decoder`), the pages that batches of prompts of different
lengths are decoded from (:mod:`paged`), and the host-side token sampler (:mod:`sampler`)."""
from .decoder import KVCache, Qwen3Decoder, single_query_attention
from .paged import PagedKVCache, paged_prefill, paged_step
from .sampler import Rng, SamplerConfig, argmax, sample

__all__ = ["KVCache", "PagedKVCache", "Qwen3Decoder", "paged_prefill", "paged_step", "single_query_attention", "Rng", "SamplerConfig", "argmax", "sample"]
