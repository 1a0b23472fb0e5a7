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

* ``torch.ops.dsalt_b200.qk_norm_rope`` / ``gated_ffn`` / ``pack8`` / ``unpack8``
  → the functions of :mod:`dsalt_b200.layers` of these names. The first two have gradients, formed by
  ``qk_norm_rope_backward`` and ``gated_ffn_backward``: a graph keeps their inputs alone, and the
  backward pass forms again what else it reads

``cu_list`` (the host copy of ``cu_seqlens``) is an ``int[]`` argument: the kernels size
their launches and workspaces from it, so a compiled graph is specialised on the packing.
The fake (meta) functions give the output shapes and dtypes; no real implementation runs
while tracing.
"""
from __future__ import annotations

from typing import List, Optional

import torch

from . import _lib as L
from . import layers
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


@torch.library.custom_op("dsalt_b200::qk_norm_rope", mutates_args=())
def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                 positions: Optional[torch.Tensor], q_weight: Optional[torch.Tensor], k_weight: Optional[torch.Tensor],
                 eps: float) -> List[torch.Tensor]:
    return list(layers.qk_norm_rope(q, k, cos, sin, positions=positions, q_weight=q_weight, k_weight=k_weight, eps=eps))


@qk_norm_rope.register_fake
def _(q, k, cos, sin, positions, q_weight, k_weight, eps):
    return [q.new_empty(q.shape), k.new_empty(k.shape)]


@torch.library.custom_op("dsalt_b200::qk_norm_rope_backward", mutates_args=())
def qk_norm_rope_backward(dq: torch.Tensor, dk: torch.Tensor, q: torch.Tensor, k: torch.Tensor, cos: torch.Tensor,
                          sin: torch.Tensor, positions: Optional[torch.Tensor], q_weight: Optional[torch.Tensor],
                          k_weight: Optional[torch.Tensor], eps: float) -> List[torch.Tensor]:
    return L.torch_layers().qk_norm_rope_grads(dq, dk, q, k, cos, sin, positions, q_weight, k_weight, eps)


@qk_norm_rope_backward.register_fake
def _(dq, dk, q, k, cos, sin, positions, q_weight, k_weight, eps):
    return [q.new_empty(q.shape), k.new_empty(k.shape),
            *(q.new_empty(0) if w is None else w.new_empty(w.shape) for w in (q_weight, k_weight))]


def _keep_heads(ctx, inputs, output):
    *tensors, ctx.eps = inputs
    ctx.save_for_backward(*tensors)


def _heads_backward(ctx, grads):
    q, k, cos, sin, positions, q_weight, k_weight = ctx.saved_tensors
    dq, dk = (torch.zeros_like(t) if d is None else d for d, t in zip(grads, (q, k)))
    dq, dk, dwq, dwk = torch.ops.dsalt_b200.qk_norm_rope_backward(dq, dk, q, k, cos, sin, positions, q_weight, k_weight, ctx.eps)
    return dq, dk, None, None, None, *((None, None) if q_weight is None else (dwq, dwk)), None


qk_norm_rope.register_autograd(_heads_backward, setup_context=_keep_heads)


@torch.library.custom_op("dsalt_b200::gated_ffn", mutates_args=())
def gated_ffn(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor,
              activation: str) -> torch.Tensor:
    return layers.gated_ffn(x, w_gate, w_up, w_down, activation=activation)


@gated_ffn.register_fake
def _(x, w_gate, w_up, w_down, activation):
    return x.new_empty(x.shape[:-1] + (w_down.shape[0],))


@torch.library.custom_op("dsalt_b200::gated_ffn_backward", mutates_args=())
def gated_ffn_backward(dy: torch.Tensor, x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor,
                       activation: str, wanted: List[bool]) -> List[torch.Tensor]:
    ts = x, w_gate, w_up, w_down
    cast = (t.to(dy.dtype) for t in ts)  # as autocast had them in the forward pass
    grads = L.torch_layers().gated_ffn_grads(dy, *cast, layers.ACTIVATIONS[activation], wanted)
    return [g.to(t.dtype) for g, t in zip(grads, ts)]


@gated_ffn_backward.register_fake
def _(dy, x, w_gate, w_up, w_down, activation, wanted):
    return [t.new_empty(t.shape if w else 0) for t, w in zip((x, w_gate, w_up, w_down), wanted)]


def _keep_ffn(ctx, inputs, output):
    *tensors, ctx.activation = inputs
    ctx.save_for_backward(*tensors)


def _ffn_backward(ctx, dy):
    wanted = list(ctx.needs_input_grad[:4])
    grads = torch.ops.dsalt_b200.gated_ffn_backward(dy, *ctx.saved_tensors, ctx.activation, wanted)
    return *(g if w else None for g, w in zip(grads, wanted)), None


gated_ffn.register_autograd(_ffn_backward, setup_context=_keep_ffn)


@torch.library.custom_op("dsalt_b200::pack8", mutates_args=())
def pack8(x: torch.Tensor) -> List[torch.Tensor]:
    return list(layers.pack8(x))


@pack8.register_fake
def _(x):
    return [x.new_empty(x.shape, dtype=torch.int8),
            x.new_empty(x.shape[:-1] + ((x.shape[-1] + layers.GROUP - 1) // layers.GROUP,), dtype=torch.uint8)]


@torch.library.custom_op("dsalt_b200::unpack8", mutates_args=())
def unpack8(codes: torch.Tensor, exps: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    return layers.unpack8(codes, exps, dtype)


@unpack8.register_fake
def _(codes, exps, dtype):
    return codes.new_empty(codes.shape, dtype=dtype)
