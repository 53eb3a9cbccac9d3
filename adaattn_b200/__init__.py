"""adaattn_b200: the AdaAttn attention-forward path on B200 (sm_100a).

Public surface, mirroring hkevin01/AdaAttn's attention package:
``AdaAttention`` (module), ``PrecisionMode``, ``AttentionConfig`` and the error
types; ``analyze`` / ``attention_forward`` for [B, H, N, D] tensors; and
``adaattn_b200.kernels`` for the reference's kernel-level functions. Beside
them the serving side: ``PagedKVCache`` and its functions (attention of one new
token over a paged cache, the append, the page operations) and
``token_logprobs``.
"""

from .config import (AttentionConfig, AttentionError, KernelError, MemoryError,
                     NumericalError, PrecisionMode, ShapeError)
from .core import DecisionTable, analyze, attention_forward, attention_forward_host
from .attention import AdaAttention
from .paged import (PagedKVCache, compact_pages, copy_pages, fork_pages, free_pages, paged_append,
                    paged_attention, reserve_pages)
from .scoring import TokenLogprobs, token_logprobs

__all__ = [
    "AdaAttention", "AttentionConfig", "AttentionError", "KernelError", "MemoryError",
    "NumericalError", "PrecisionMode", "ShapeError", "DecisionTable", "analyze",
    "attention_forward",
    "attention_forward_host",
    "PagedKVCache", "paged_attention", "paged_append", "reserve_pages", "fork_pages", "copy_pages",
    "free_pages", "compact_pages", "TokenLogprobs", "token_logprobs",
]

__version__ = "0.1.0"
