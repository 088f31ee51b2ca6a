"""Ops: hand-written sm_100a kernels (GPU) with pure-torch fp32 references (CPU path and test oracle)."""
from . import native, reference
from .functional import *  # noqa: F401,F403
from .native import check_status
from .paged import paged_append, paged_attention
from .text_attention import packed_attention, prefix_lengths, relative_attention, window_attention
