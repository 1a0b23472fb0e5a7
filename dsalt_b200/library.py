"""The operators registered with ``torch.library`` (namespace ``dsalt_b200``), so that
``torch.compile`` treats each as one opaque node with a shape function, as the reference
keeps its kernels opaque (``_dynamo_opaque``, ``dsalt/kernels/dsalt_triton_attn.py:330-336``)
— here without a graph break, so ``fullgraph=True`` compiles a model that contains them.

* ``torch.ops.dsalt_b200.window_signals``   → :func:`dsalt_b200.ops.window_signals`
* ``torch.ops.dsalt_b200.select_landmarks`` → :func:`dsalt_b200.ops.select_landmarks`
* ``torch.ops.dsalt_b200.dsalt_attention``  → :func:`dsalt_b200.ops.dsalt_attention`
* ``torch.ops.dsalt_b200.core_forward``     → :func:`dsalt_b200.ops.core_forward`

* ``torch.ops.dsalt_b200.append_cache`` / ``cache_attention`` / ``sample_tokens``
  → the functions of :mod:`dsalt_b200.serving` of these names (``sample_tokens`` with its settings as
  numbers and the log-probability)

``cu_list`` (the host copy of ``cu_seqlens``) is an ``int[]`` argument: the kernels size
their launches and workspaces from it, so a compiled graph is specialised on the packing.
The fake (meta) functions give the output shapes and dtypes; no real implementation runs
while tracing.
"""
from __future__ import annotations

from typing import List, Optional

import torch

from . import ops
from . import serving


def _n_sets(cu_list: List[int], mode: str, block: int) -> int:
    return len(cu_list) - 1 if mode == "global" else ops.n_block_sets(cu_list, block)


@torch.library.custom_op("dsalt_b200::window_signals", mutates_args=())
def window_signals(x: torch.Tensor, gate_weight: torch.Tensor, gate_bias: torch.Tensor, n_min: int, n_max: int,
                   v: torch.Tensor, head_dim: int, norm_round: bool,
                   logit: Optional[torch.Tensor]) -> List[torch.Tensor]:
    w, xn, vn = ops.window_signals(x, gate_weight, gate_bias, n_min, n_max, v, head_dim, norm_round, logit=logit)
    return [w, xn, vn]


@window_signals.register_fake
def _(x, gate_weight, gate_bias, n_min, n_max, v, head_dim, norm_round, logit):
    T = x.shape[0]
    n_kv = v.reshape(T, -1).shape[1] // head_dim
    return [x.new_empty(T, dtype=torch.int32), x.new_empty(T, dtype=torch.float32),
            x.new_empty(T, n_kv, dtype=torch.float32)]


@torch.library.custom_op("dsalt_b200::select_landmarks", mutates_args=())
def select_landmarks(xnorm: torch.Tensor, vnorm: torch.Tensor, w: torch.Tensor, alpha: torch.Tensor,
                     cu_seqlens: torch.Tensor, k_lmk: int, n_heads: int, mode: str, block: int,
                     cu_list: List[int]) -> torch.Tensor:
    return ops.select_landmarks(xnorm, vnorm, w, alpha, cu_seqlens, k_lmk, n_heads, mode, block, cu_list=cu_list)


@select_landmarks.register_fake
def _(xnorm, vnorm, w, alpha, cu_seqlens, k_lmk, n_heads, mode, block, cu_list):
    return xnorm.new_empty(n_heads, _n_sets(cu_list, mode, block), k_lmk, dtype=torch.int32)


@torch.library.custom_op("dsalt_b200::dsalt_attention", mutates_args=())
def dsalt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, lmk_indices: torch.Tensor,
                    lmk_bias: Optional[torch.Tensor], w_sizes: torch.Tensor, cu_seqlens: torch.Tensor, lmk_block: int,
                    cu_list: List[int], out_dtype: torch.dtype) -> torch.Tensor:
    return ops.dsalt_attention(q, k, v, lmk_indices, lmk_bias, w_sizes, cu_seqlens, lmk_block=lmk_block,
                               out_dtype=out_dtype, cu_list=cu_list)


@dsalt_attention.register_fake
def _(q, k, v, lmk_indices, lmk_bias, w_sizes, cu_seqlens, lmk_block, cu_list, out_dtype):
    return q.new_empty(q.shape, dtype=out_dtype)


@torch.library.custom_op("dsalt_b200::core_forward", mutates_args=())
def core_forward(x: torch.Tensor, gate_weight: torch.Tensor, gate_bias: torch.Tensor, n_min: int, n_max: int,
                 alpha: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_lmk: int,
                 cu_seqlens: torch.Tensor, mode: str, block: int, norm_round: bool, cu_list: List[int],
                 out_dtype: torch.dtype, logit: Optional[torch.Tensor]) -> torch.Tensor:
    return ops.core_forward(x, gate_weight, gate_bias, n_min, n_max, alpha, q, k, v, k_lmk, cu_seqlens, mode=mode,
                            block=block, norm_round=norm_round, out_dtype=out_dtype, cu_list=cu_list, logit=logit)


@core_forward.register_fake
def _(x, gate_weight, gate_bias, n_min, n_max, alpha, q, k, v, k_lmk, cu_seqlens, mode, block, norm_round, cu_list,
      out_dtype, logit):
    return q.new_empty(q.shape, dtype=out_dtype)


@torch.library.custom_op("dsalt_b200::append_cache", mutates_args=("k_cache", "v_cache", "k_scale", "v_scale"))
def append_cache(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                 v_scale: torch.Tensor, slots: torch.Tensor) -> None:
    serving.append_cache(k, v, k_cache, v_cache, k_scale, v_scale, slots)


@append_cache.register_fake
def _(k, v, k_cache, v_cache, k_scale, v_scale, slots):
    return None


@torch.library.custom_op("dsalt_b200::cache_attention", mutates_args=())
def cache_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                    v_scale: torch.Tensor, block_tables: torch.Tensor, seq_lens: torch.Tensor,
                    cu_q: Optional[torch.Tensor], w_sizes: Optional[torch.Tensor], lmk_indices: Optional[torch.Tensor],
                    lmk_bias: Optional[torch.Tensor], out_dtype: torch.dtype) -> torch.Tensor:
    return serving.cache_attention(q, k_cache, v_cache, k_scale, v_scale, block_tables, seq_lens, cu_q=cu_q,
                                   w_sizes=w_sizes, lmk_indices=lmk_indices, lmk_bias=lmk_bias, out_dtype=out_dtype)


@cache_attention.register_fake
def _(q, k_cache, v_cache, k_scale, v_scale, block_tables, seq_lens, cu_q, w_sizes, lmk_indices, lmk_bias, out_dtype):
    return q.new_empty(q.shape, dtype=out_dtype)


@torch.library.custom_op("dsalt_b200::sample_tokens", mutates_args=())
def sample_tokens(logits: torch.Tensor, u: torch.Tensor, temperature: float, top_k: int, top_p: float,
                  min_p: float) -> List[torch.Tensor]:
    return list(serving.sample_tokens(logits, u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p,
                                      return_logprob=True))


@sample_tokens.register_fake
def _(logits, u, temperature, top_k, top_p, min_p):
    return [logits.new_empty(logits.shape[0], dtype=torch.int64), logits.new_empty(logits.shape[0], dtype=torch.float32)]
