"""Custom ops of the paged 4- or 8-bit key / value cache (no reference counterpart).

* ``torch.ops.gko.kv_cache_write(k, v, k_codes, v_codes, k_pairs, v_pairs, slots)`` quantises new keys
  and values into the cache, in place (``ops.kv_cache_write``).
* ``torch.ops.gko.kv_cache_read(k_codes, v_codes, k_pairs, v_pairs, block_table, cu_seqlens, tokens,
  head_dim) -> (k, v)`` reads cached sequences back for ``gko::fmha_varlen_fwd`` (``ops.kv_cache_read``).
* ``torch.ops.gko.fmha_cache_fwd(q, k_codes, ..., window, softcap, sinks) -> (out, lse)`` answers new
  tokens from the cache (``ops.fmha_cache_fwd``).

They are opaque to Dynamo, so a compiled decode step keeps them whole. No gradients: a cache is read
by inference only.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from .. import ops


def _ensure_op():
    have = lambda n: hasattr(torch.ops, "gko") and hasattr(torch.ops.gko, n)  # noqa: E731
    if not have("kv_cache_write"):

        @torch.library.custom_op("gko::kv_cache_write", mutates_args=("k_codes", "v_codes", "k_pairs", "v_pairs"))
        def kv_cache_write(k: torch.Tensor, v: torch.Tensor, k_codes: torch.Tensor, v_codes: torch.Tensor,
                           k_pairs: torch.Tensor, v_pairs: torch.Tensor, slots: torch.Tensor) -> None:
            ops.kv_cache_write(k, v, (k_codes, v_codes, k_pairs, v_pairs), slots)

        @kv_cache_write.register_fake
        def _(k, v, k_codes, v_codes, k_pairs, v_pairs, slots):
            return None

    if not have("kv_cache_read"):

        @torch.library.custom_op("gko::kv_cache_read", mutates_args=())
        def kv_cache_read(k_codes: torch.Tensor, v_codes: torch.Tensor, k_pairs: torch.Tensor, v_pairs: torch.Tensor,
                          block_table: torch.Tensor, cu_seqlens: torch.Tensor, tokens: int, head_dim: int
                          ) -> Tuple[torch.Tensor, torch.Tensor]:
            return ops.kv_cache_read((k_codes, v_codes, k_pairs, v_pairs), block_table, cu_seqlens, tokens, head_dim)

        @kv_cache_read.register_fake
        def _(k_codes, v_codes, k_pairs, v_pairs, block_table, cu_seqlens, tokens, head_dim):
            shape = (tokens, k_codes.size(1), head_dim)
            return k_pairs.new_empty(shape), v_pairs.new_empty(shape)

    if not have("fmha_cache_fwd"):

        @torch.library.custom_op("gko::fmha_cache_fwd", mutates_args=())
        def fmha_cache_fwd(q: torch.Tensor, k_codes: torch.Tensor, v_codes: torch.Tensor, k_pairs: torch.Tensor,
                           v_pairs: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
                           cu_seqlens_q: Optional[torch.Tensor], max_seqlen_q: int, max_seqlen_k: int, scale: float,
                           causal: int, window: int, softcap: float, sinks: int) -> Tuple[torch.Tensor, torch.Tensor]:
            return ops.fmha_cache_fwd(q, (k_codes, v_codes, k_pairs, v_pairs), block_table, seq_lens, cu_seqlens_q,
                                      max_seqlen_q, max_seqlen_k, scale, causal, window, softcap, sinks)

        @fmha_cache_fwd.register_fake
        def _(q, k_codes, v_codes, k_pairs, v_pairs, block_table, seq_lens, cu_seqlens_q, max_seqlen_q, max_seqlen_k,
              scale, causal, window, softcap, sinks):
            return q.new_empty(q.shape), q.new_empty((q.size(1), q.size(0)), dtype=torch.float32)


def register(backend=None):
    """Install the cache ops. ``backend`` is accepted and ignored."""
    _ensure_op()
