"""What a decoder block computes around its attention, over the C ABI, with gradients.

* :func:`qk_norm_rope`        — norm of each query and key head and the position rotation, one pass
* :func:`gated_ffn`           — ``(act(x Wgᵀ) · (x Wuᵀ)) Wdᵀ``: the activation and the product in the
  epilogue of the first matrix product, their gradients in that of the backward's first
* :func:`pack8` / :func:`unpack8` — activations in 8 bits, 32 values to a power-of-two scale;
  ``gated_ffn(keep="8bit")`` keeps its activations so between its forward and backward pass

The reference norms and rotates nothing but by elementwise torch operations
(``dsalt/kernels/window_utils.py:73-88``) and runs its block's MLP as three linear layers
(``dsalt/modules/dsalt_transformer.py``). As in :mod:`dsalt_b200.serving`, tensors must be CUDA
tensors of one device and every call launches on its current stream; none synchronises.
"""
from __future__ import annotations

import functools

import torch

from . import _lib as L
from .ops import _dt, _ptr, _workspace
from .serving import _on_one_device, _rows, _run, _want

GROUP = 32  # values that share a scale
ACTIVATIONS = {"silu": L.ACT_SILU, "gelu": L.ACT_GELU}
KEEP = {"16bit": L.KEEP_INPUT, "8bit": L.KEEP_8BIT}


def _no_second_derivative() -> None:
    if torch.is_grad_enabled():  # only with create_graph=True
        raise RuntimeError("dsalt_b200 operators have no second derivative")


# --------------------------------------------------------------------------- 8 bits
def _matrix(x: torch.Tensor):
    """``x [..., n]`` as rows of consecutive values and their stride (a copy where its strides do not
    allow that)."""
    n = x.shape[-1]
    if x.is_contiguous():
        return (x if x.dim() == 2 else x.view(-1, n)), n
    if x.dim() != 2:
        x = x.reshape(-1, n)
    row, one = x.stride()
    if n > 1 and one != 1 or x.shape[0] > 1 and row < n:
        return x.contiguous(), n
    return x, (row if x.shape[0] > 1 else n)


def _pack(dev, x2, stride):
    rows, n = x2.shape
    codes = torch.empty((rows, n), dtype=torch.int8, device=dev)
    exps = torch.empty((rows, -(-n // GROUP)), dtype=torch.uint8, device=dev)
    _run(dev, "dsalt_pack8", x2.data_ptr(), _dt(x2), rows, n, stride, codes.data_ptr(), exps.data_ptr())
    return codes, exps


def pack8(x):
    """``x [..., n]`` (bf16, fp16 or fp32) in 8 bits: ``(codes [..., n] int8, exps [..., ceil(n / 32)]
    uint8)``. 32 neighbouring values share the scale ``2^(exps - 127)``, chosen so that the largest
    lies in [64, 128) steps; a value is off by half a step at most (a whole one above 127 steps). A
    group with a NaN or an infinity reads as NaN as a whole. No gradient goes through it."""
    dev = _on_one_device(x)
    if x.dim() < 1:
        raise ValueError("pack8 needs at least one axis")
    shape = x.shape
    if len(shape) == 2 and shape[1]:
        return _pack(dev, *_matrix(x))
    if x.numel() == 0:
        _dt(x)
        return (torch.empty(shape, dtype=torch.int8, device=dev),
                torch.empty(shape[:-1] + (-(-shape[-1] // GROUP),), dtype=torch.uint8, device=dev))
    codes, exps = _pack(dev, *_matrix(x.detach()))
    return codes.view(shape), exps.view(shape[:-1] + (-1,))


def unpack8(codes, exps, dtype=torch.bfloat16):
    """The values that :func:`pack8`'s ``codes`` and ``exps`` stand for, in ``dtype``."""
    dev = _on_one_device(codes, exps)
    if codes.dim() < 1:
        raise ValueError("codes need at least one axis")
    shape = codes.shape
    n = shape[-1]
    _want(codes, "codes", torch.int8, shape)
    _want(exps, "exps", torch.uint8, shape[:-1] + (-(-n // GROUP),))
    out = torch.empty(shape, dtype=dtype, device=dev)
    _run(dev, "dsalt_unpack8", codes.data_ptr(), exps.data_ptr(), codes.numel() // n if n else 0, n, out.data_ptr(),
         _dt(out))
    return out


# --------------------------------------------------------------------------- heads
def _table(t, D: int):
    """A table of angles as fp32 with 16-byte aligned rows, and their stride."""
    if t.dtype is not torch.float32:
        t = t.float()
    row, one = t.stride()
    several = t.shape[0] > 1
    if one != 1 or t.data_ptr() % 16 or several and (row % 4 or row < D // 2):
        t = t.clone(memory_format=torch.contiguous_format)
        row = t.stride(0)
    return t, (row if several else -(-D // 4) * 4)


def _rope_args(q, k, cos, sin, positions, q_weight, k_weight):
    """Checked arguments: ``(dev, T, H, H_kv, D, stride of the tables, cos, sin, positions, q_weight,
    k_weight)``."""
    if q.dim() != 3 or k.dim() != 3:
        raise ValueError("q must be [T, H, D] and k [T, H_kv, D]")
    dev = _on_one_device(q, k, cos, sin, positions, q_weight, k_weight)
    T, H, D = q.shape
    Tk, Hk, Dk = k.shape
    if Tk != T or Dk != D:
        raise ValueError(f"k must be [{T}, H_kv, {D}], got {tuple(k.shape)}")
    if k.dtype is not q.dtype:
        raise TypeError("q and k must share a dtype")
    if (q_weight is None) != (k_weight is None):
        raise ValueError("q_weight and k_weight go together")
    if q_weight is not None:
        _want(q_weight, "q_weight", q_weight.dtype, (D,))
        _want(k_weight, "k_weight", q_weight.dtype, (D,))
    if D % 2:
        raise ValueError(f"head_dim {D} is odd")
    if cos.dim() != 2 or cos.shape != sin.shape or cos.shape[1] not in (D, D // 2):
        raise ValueError(f"cos and sin must be [rows, {D}] or [rows, {D // 2}], both alike")
    cos, stride = _table(cos, D)
    sin, other = _table(sin, D)
    if other != stride:
        cos, sin = cos.contiguous(), sin.contiguous()
        stride = cos.stride(0)
    if positions is not None:
        if positions.shape != (T,) or positions.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"positions must be [{T}] whole numbers")
        if positions.dtype is not torch.int32 or not positions.is_contiguous():
            positions = positions.to(torch.int32).contiguous()
        if cos.shape[0] == 0 and T:
            raise ValueError("empty tables")
    elif cos.shape[0] < T:
        raise ValueError(f"tables of {cos.shape[0]} rows for {T} tokens")
    return dev, T, H, Hk, D, stride, cos, sin, positions, q_weight, k_weight


def _rope_forward(q, k, args, eps):
    dev, T, H, Hk, D, stride, cos, sin, positions, q_weight, k_weight = args
    qo = torch.empty((T, H, D), dtype=q.dtype, device=dev)
    ko = torch.empty((T, Hk, D), dtype=q.dtype, device=dev)
    q, q_token, q_head = _rows(q)
    k, k_token, k_head = _rows(k)
    _run(dev, "dsalt_qk_norm_rope", q.data_ptr(), k.data_ptr(), _dt(q), T, H, Hk, D, q_token, q_head, k_token, k_head,
         _ptr(q_weight), _ptr(k_weight), 0 if q_weight is None else _dt(q_weight), float(eps), cos.data_ptr(),
         sin.data_ptr(), max(cos.shape[0], 1), stride, _ptr(positions), qo.data_ptr(), ko.data_ptr())
    return qo, ko


class QKNormRopeFunction(torch.autograd.Function):
    """Autograd of :func:`qk_norm_rope`: ``q`` and ``k`` are kept as they came, the norms are formed
    again in the backward pass."""

    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, cos, sin, positions, eps):
        args = _rope_args(q, k, cos, sin, positions, q_weight, k_weight)
        ctx.save_for_backward(q, k, *args[6:])
        ctx.eps, ctx.table_stride = eps, args[5]
        return _rope_forward(q, k, args, eps)

    @staticmethod
    def backward(ctx, gq, gk):
        _no_second_derivative()
        q, k, cos, sin, positions, q_weight, k_weight = ctx.saved_tensors
        dev, (T, H, D), Hk = q.device, q.shape, k.shape[1]
        dq = torch.empty((T, H, D), dtype=q.dtype, device=dev)
        dk = torch.empty((T, Hk, D), dtype=q.dtype, device=dev)
        norm = q_weight is not None
        dwq, dwk = (torch.empty_like(q_weight), torch.empty_like(k_weight)) if norm else (None, None)
        ws = _workspace(_rope_workspace(D) if norm else 0, dev)
        q, q_token, q_head = _rows(q)
        k, k_token, k_head = _rows(k)
        gq, gq_token, gq_head = _rows(gq)
        gk, gk_token, gk_head = _rows(gk)
        _run(dev, "dsalt_qk_norm_rope_bwd", q.data_ptr(), k.data_ptr(), gq.data_ptr(), gk.data_ptr(), _dt(q), T, H, Hk, D,
             q_token, q_head, k_token, k_head, gq_token, gq_head, gk_token, gk_head, _ptr(q_weight), _ptr(k_weight),
             _dt(q_weight) if norm else 0, float(ctx.eps), cos.data_ptr(), sin.data_ptr(), max(cos.shape[0], 1),
             ctx.table_stride, _ptr(positions), dq.data_ptr(), dk.data_ptr(), _ptr(dwq), _ptr(dwk), ws.data_ptr(), ws.numel())
        return dq, dk, dwq, dwk, None, None, None, None


@functools.lru_cache(maxsize=64)
def _rope_workspace(D: int) -> int:
    return L.query("dsalt_qk_norm_rope_bwd_workspace_bytes", D)


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
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or q_weight is not None and q_weight.requires_grad
                                    or k_weight is not None and k_weight.requires_grad):
        return QKNormRopeFunction.apply(q, k, q_weight, k_weight, cos, sin, positions, eps)
    return _rope_forward(q, k, _rope_args(q, k, cos, sin, positions, q_weight, k_weight), eps)


# --------------------------------------------------------------------------- feed-forward
def _aligned(t, stride: int) -> bool:
    """Whether the rows of ``t`` are 16-byte aligned, or their length does not allow that anyway."""
    es = t.element_size()
    return t.shape[1] * es % 16 != 0 or t.data_ptr() % 16 == 0 and stride * es % 16 == 0


def _ffn_rows(x):
    x, stride = _matrix(x)
    if not _aligned(x, stride):
        x = x.clone(memory_format=torch.contiguous_format)
        stride = x.shape[1]
    return x, stride


def _ffn_args(x, w_gate, w_up, w_down, activation, keep):
    dev = _on_one_device(x, w_gate, w_up, w_down)
    if w_gate.dim() != 2 or w_down.dim() != 2 or x.dim() < 1:
        raise ValueError("x must be [..., d_model], w_gate and w_up [d_ff, d_model], w_down [d_out, d_ff]")
    F, d = w_gate.shape
    if x.shape[-1] != d or w_up.shape != w_gate.shape or w_down.shape[1] != F:
        raise ValueError(f"x {tuple(x.shape)}, w_gate {tuple(w_gate.shape)}, w_up {tuple(w_up.shape)} and w_down "
                         f"{tuple(w_down.shape)} do not fit together")
    if not (x.dtype is w_gate.dtype is w_up.dtype is w_down.dtype):
        raise TypeError("x and the weights must share a dtype")
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}")
    if keep not in KEEP:
        raise ValueError(f"keep must be one of {sorted(KEEP)}")
    _dt(x)
    return dev, d, F, w_down.shape[0]


@functools.lru_cache(maxsize=1024)
def _ffn_workspace(dt: int, T: int, d: int, F: int, d_out: int, keep: int) -> int:
    """Workspace bytes of a forward call, or (``keep`` not 0) of a backward one."""
    if keep:
        n = L.query("dsalt_gated_ffn_bwd_workspace_bytes", dt, T, d, F, d_out, keep)
    else:
        n = L.query("dsalt_gated_ffn_workspace_bytes", dt, T, d, F, d_out)
    return n


@functools.lru_cache(maxsize=256)
def _ffn_pitch(F: int) -> int:
    return L.query("dsalt_gated_ffn_pitch", F)


def _weight(w):
    if w.is_contiguous():
        return w if _aligned(w, w.shape[1]) else w.clone()
    return w.contiguous()


def _ffn_forward(x2, stride, w_gate, w_up, w_down, sizes, act, keep):
    """``(y, kept, exps)`` of rows ``x2``; nothing is kept with ``L.KEEP_NONE``."""
    dev, d, F, d_out = sizes
    T = x2.shape[0]
    dt = _dt(x2)
    y = torch.empty((T, d_out), dtype=x2.dtype, device=dev)
    kept = exps = None
    if keep:
        pitch = _ffn_pitch(F)
        coded = keep == L.KEEP_8BIT
        kept = torch.empty(2 if coded else 3, T, pitch, dtype=torch.int8 if coded else x2.dtype, device=dev)
        if coded or x2.dtype is not torch.float32:
            exps = torch.empty(2, pitch // GROUP, T, dtype=torch.uint8, device=dev)
    ws = torch.empty(_ffn_workspace(dt, T, d, F, d_out, 0), dtype=torch.uint8, device=dev)
    _run(dev, "dsalt_gated_ffn", x2.data_ptr(), dt, T, d, stride, w_gate.data_ptr(), w_up.data_ptr(),
         w_down.data_ptr(), F, d_out, act, keep, _ptr(kept), _ptr(exps), y.data_ptr(), ws.data_ptr(), ws.numel())
    return y, kept, exps


class GatedFFNFunction(torch.autograd.Function):
    """Autograd of :func:`gated_ffn`. Kept for the backward pass: ``x Wgᵀ`` and ``x Wuᵀ`` (written by
    the epilogue that forms them) and ``x``, the first two in 16 bits with a scale for 32 (of fp32 inputs in
    fp32), or all three in 8 bits. With 16 bits the rows that the last product read are kept too; with 8 they
    are formed again."""

    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, activation, keep):
        sizes = _ffn_args(x, w_gate, w_up, w_down, activation, keep)
        act, mode = ACTIVATIONS[activation], KEEP[keep]
        x2, stride = _ffn_rows(x)
        ws = _weight(w_gate), _weight(w_up), _weight(w_down)
        y, kept, exps = _ffn_forward(x2, stride, *ws, sizes, act, mode)
        x_exps = None
        if not (ctx.needs_input_grad[1] or ctx.needs_input_grad[2]):
            x2 = None  # only the weights' gradients read it
        elif mode == L.KEEP_8BIT and x2.numel():
            x2, x_exps = _pack(sizes[0], x2, stride)
        ctx.save_for_backward(x2, x_exps, kept, exps, *ws)
        ctx.act, ctx.mode, ctx.sizes, ctx.shape, ctx.stride = act, mode, sizes, x.shape, stride
        return y if x.dim() == 2 else y.view(*x.shape[:-1], sizes[3])

    @staticmethod
    def backward(ctx, dy):
        _no_second_derivative()
        x2, x_exps, kept, exps, w_gate, w_up, w_down = ctx.saved_tensors
        dev, d, F, d_out = ctx.sizes
        need_x, need_gate, need_up, need_down = ctx.needs_input_grad[:4]
        T = kept.shape[1]
        dy, dy_stride = _ffn_rows(dy.reshape(T, d_out))
        dx = torch.empty(T, d, dtype=w_gate.dtype, device=dev) if need_x else None
        both = need_gate or need_up
        dwg, dwu = (torch.empty_like(w_gate), torch.empty_like(w_up)) if both else (None, None)
        dwd = torch.empty_like(w_down) if need_down else None
        dt = _dt(w_gate)
        ws = _workspace(_ffn_workspace(dt, T, d, F, d_out, ctx.mode), dev)
        _run(dev, "dsalt_gated_ffn_bwd", dy.data_ptr(), dt, T, d, dy_stride, _ptr(x2), ctx.stride, _ptr(x_exps),
             w_gate.data_ptr(), w_up.data_ptr(), w_down.data_ptr(), F, d_out, ctx.act, ctx.mode, kept.data_ptr(),
             _ptr(exps), _ptr(dx), _ptr(dwg), _ptr(dwu), _ptr(dwd), ws.data_ptr(), ws.numel())
        return (dx.view(ctx.shape) if need_x else None, dwg if need_gate else None, dwu if need_up else None, dwd,
                None, None)


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
    and the others in 16 bits with a scale for 32 values (fp32 inputs: fp32), or ``"8bit"``, as
    :func:`pack8` holds them (a third of the memory; the gradients are then those at the held values). bf16 and fp16 run on the tensor cores where sizes are
    multiples of 8; fp32 and other sizes on the CUDA cores. Under autocast all four are cast first, as
    a linear layer's are."""
    x, w_gate, w_up, w_down = autocast_all(x, w_gate, w_up, w_down)
    if torch.is_grad_enabled() and (x.requires_grad or w_gate.requires_grad or w_up.requires_grad or w_down.requires_grad):
        return GatedFFNFunction.apply(x, w_gate, w_up, w_down, activation, keep)
    sizes = _ffn_args(x, w_gate, w_up, w_down, activation, keep)
    x2, stride = _ffn_rows(x)
    y, _, _ = _ffn_forward(x2, stride, _weight(w_gate), _weight(w_up), _weight(w_down), sizes, ACTIVATIONS[activation], L.KEEP_NONE)
    return y if x.dim() == 2 else y.view(*x.shape[:-1], sizes[3])
