"""What a decoder block computes around its attention, over the C ABI, with gradients.

* :func:`qk_norm_rope`        — norm of each query and key head and the position rotation, one pass
* :func:`gated_ffn`           — ``(act(x Wgᵀ) · (x Wuᵀ)) Wdᵀ``: the activation and the product in the
  epilogue of the first matrix product, their gradients in that of the backward's first
* :func:`pack8` / :func:`unpack8` — activations in 8 bits, 32 values to a power-of-two scale;
  ``gated_ffn(keep="8bit")`` keeps its activations so between its forward and backward pass

The reference norms and rotates nothing but by elementwise torch operations
(``dsalt/kernels/window_utils.py:73-88``) and runs its block's MLP as three linear layers
(``dsalt/modules/dsalt_transformer.py``). As in :mod:`dsalt_b200.serving`, tensors must be CUDA
tensors of one device and every call launches on its current stream; none synchronises. Gradients are
those of one backward pass: second and forward-mode derivatives are refused. Checks,
outputs and autograd nodes are compiled (``csrc/torch_layers.cpp``): the calls are short.
"""
from __future__ import annotations

import torch

from . import _lib as L
from .ops import _DT

GROUP = 32  # values that share a scale
ACTIVATIONS = {"silu": L.ACT_SILU, "gelu": L.ACT_GELU}
KEEP = {"16bit": L.KEEP_INPUT, "8bit": L.KEEP_8BIT}


# --------------------------------------------------------------------------- 8 bits
def pack8(x):
    """``x [..., n]`` (bf16, fp16 or fp32) in 8 bits: ``(codes [..., n] int8, exps [..., ceil(n / 32)]
    uint8)``. 32 neighbouring values share the scale ``2^(exps - 127)``, chosen so that the largest
    lies in [64, 128) steps; a value is off by half a step at most (a whole one above 127 steps). A
    group with a NaN or an infinity reads as NaN as a whole. No gradient goes through it."""
    return L.torch_layers().pack8(x)


def unpack8(codes, exps, dtype=torch.bfloat16):
    """The values that :func:`pack8`'s ``codes`` and ``exps`` stand for, in ``dtype``."""
    if dtype not in _DT:
        raise TypeError(f"unsupported dtype {dtype}")
    return L.torch_layers().unpack8(codes, exps, _DT[dtype])


# --------------------------------------------------------------------------- heads
def qk_norm_rope(q, k, cos, sin, *, positions=None, q_weight=None, k_weight=None, eps: float = 1e-6):
    """Norm of each head and half-split rotation in one pass: ``(q', k')``, contiguous, in the
    input's dtype (fp32 in between, rounded once).

    ``q [T, H, D]``, ``k [T, H_kv, D]`` (any strides that leave 16-byte aligned rows, e.g. views of one
    projection; others are copied), ``D`` a multiple of 16 (fp32: 8) up to 256. ``q_weight, k_weight
    [D]``: ``n = w x / sqrt(mean(x²) + eps)``; without them no norm. ``cos, sin``: tables of
    :func:`dsalt_b200.module.build_rope_cache` (``[rows, D]``, whose second half repeats the first and is
    not read, or ``[rows, D/2]``); token ``t`` takes row ``positions[t]``, or row ``t``. A position outside
    the tables is taken as 0 and reported by :func:`dsalt_b200.device_status` (51). Differentiable in
    ``q``, ``k`` and the weights."""
    return L.torch_layers().qk_norm_rope(q, k, cos, sin, positions, q_weight, k_weight, eps)


# --------------------------------------------------------------------------- feed-forward
def autocast_all(*ts):
    """The tensors as a linear layer takes them: in autocast's dtype where that is on."""
    if torch.is_autocast_enabled("cuda") and ts[0].is_cuda:
        dt = torch.get_autocast_dtype("cuda")
        return tuple(t.to(dt) for t in ts)
    return ts


def gated_ffn(x, w_gate, w_up, w_down, *, activation: str = "silu", keep: str = "16bit"):
    """``(act(x Wgᵀ) · (x Wuᵀ)) Wdᵀ``: ``x [..., d_model]``, ``w_gate, w_up [d_ff, d_model]``, ``w_down [d_out,
    d_ff]`` → ``[..., d_out]`` in ``x``'s dtype. Sums are fp32; the product of gate and up is rounded to the
    dtype once, as the operand of the last product.

    ``activation`` is ``"silu"`` or ``"gelu"`` (by the error function). Differentiable in all four;
    ``keep`` says in what form the backward pass finds ``x``, ``x Wgᵀ`` and ``x Wuᵀ``: ``"16bit"``, ``x`` as it is
    and the others each with 16 significant bits, in three bytes (fp32 inputs: fp32), or ``"8bit"``, as
    :func:`pack8` holds them (a third of the memory; the gradients are then those at the held values, and a value
    that is not finite is one for its group of 32). bf16
    and fp16 run on the tensor cores where sizes are multiples of 8; fp32 and other sizes on the CUDA
    cores. Under autocast all four are cast first, as a linear layer's are."""
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}")
    if keep not in KEEP:
        raise ValueError(f"keep must be one of {sorted(KEEP)}")
    return L.torch_layers().gated_ffn(*autocast_all(x, w_gate, w_up, w_down), ACTIVATIONS[activation], KEEP[keep])
