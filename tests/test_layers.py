"""What a decoder block computes around its attention, without a GPU: the oracle against
independent statements of the same definitions and against differences, and the refusals of the C ABI and
of the torch-facing functions."""
import ctypes
import os

import pytest
import torch

from dsalt_b200 import _lib as L
from dsalt_b200 import layers as Y
from oracle import layers_oracle as O


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(L.LIB_PATH):
        from dsalt_b200 import build
        build.build()
    return L.load()


def normal(g, *shape):
    return torch.empty(*shape, dtype=torch.float64).normal_(generator=g)


# ------------------------------------------------------------------ the oracle itself
def test_oracle_pack_is_within_a_step_and_never_above_the_largest():
    g = torch.Generator().manual_seed(0)
    x = (normal(g, 40, 1000) * torch.exp2(torch.randint(-30, 30, (40, 1000), generator=g).double())).float().double()
    x[3] = 0
    x[4, :40] = 1e-40  # below the normal range of fp32
    x = x.float().double()
    codes, exps = O.pack(x)
    got = O.unpack(codes, exps)
    pad = torch.cat([x, x.new_zeros(40, 24)], 1).view(40, 32, 32)
    top = pad.abs().amax(-1)
    step = torch.exp2(exps.double() - 127)
    assert ((top < 128 * step) & ((top >= 64 * step) | (exps == 1))).all()
    top, step = (t.repeat_interleave(32, 1)[:, :1000] for t in (top, step))
    whole = x.abs() > 127 * step
    assert ((got - x).abs() <= torch.where(whole, step, step / 2)).all() and (got.abs() <= top + step / 2).all()
    assert (got.abs()[top >= 127 * step] <= top[top >= 127 * step]).all()


def test_oracle_pack_of_values_that_are_not_finite():
    x = torch.ones(2, 70, dtype=torch.float64)
    x[0, 33], x[1, 69] = float("nan"), float("-inf")
    codes, exps = O.pack(x)
    assert exps.tolist() == [[121, 255, 121], [121, 121, 255]]
    assert codes[0, 32:64].abs().sum() == 0 and torch.isnan(O.unpack(codes, exps)[0, 32:64]).all()
    assert torch.equal(O.unpack(codes, exps)[0, :32], x[0, :32])


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_oracle_ffn_gradients_are_those_of_autograd_and_of_differences(act):
    g = torch.Generator().manual_seed(1)
    x, wg, wu, wd, dy = normal(g, 7, 10), normal(g, 12, 10), normal(g, 12, 10), normal(g, 5, 12), normal(g, 7, 5)
    leaves = [t.clone().requires_grad_(True) for t in (x, wg, wu, wd)]
    F = torch.nn.functional
    a = getattr(F, act)(leaves[0] @ leaves[1].T) * (leaves[0] @ leaves[2].T)
    y = a @ leaves[3].T
    torch.testing.assert_close(O.ffn(x, wg, wu, wd, act), y.detach(), rtol=1e-12, atol=1e-12)
    grads = O.ffn_grad(x, wg, wu, wd, act, dy)
    for got, ref in zip(grads, torch.autograd.grad(y, leaves, dy)):
        torch.testing.assert_close(got, ref, rtol=1e-11, atol=1e-11)
    step = 1e-5
    for i, t in enumerate((x, wg, wu, wd)):
        v = normal(g, *t.shape)
        ends = [O.ffn(*[w + s * v if j == i else w for j, w in enumerate((x, wg, wu, wd))], act) for s in (step, -step)]
        slope = ((ends[0] - ends[1]) / (2 * step) * dy).sum()
        assert abs(slope - (grads[i] * v).sum()) <= 1e-6 * (1 + grads[i].abs().sum())


def test_oracle_rope_gradients_are_those_of_differences():
    g = torch.Generator().manual_seed(2)
    x, w, d, angle = normal(g, 5, 3, 16), normal(g, 16), normal(g, 5, 3, 16), normal(g, 5, 8)
    cos, sin, eps = angle.cos(), angle.sin(), 1e-3
    from dsalt_b200.module import apply_rotary_emb
    n = torch.nn.functional.rms_norm(x, (16,), w, eps)
    both = [torch.cat([t, t], 1)[:, None] for t in (cos, sin)]
    torch.testing.assert_close(O.rope(x, w, cos, sin, eps), apply_rotary_emb(n, n, *both)[0], rtol=1e-12, atol=1e-12)
    torch.testing.assert_close(O.rope(x, None, cos, sin, eps), apply_rotary_emb(x, x, *both)[0], rtol=1e-12, atol=1e-12)
    dx, dw = O.rope_grad(x, w, cos, sin, eps, d)
    step = 1e-5
    vx, vw = normal(g, 5, 3, 16), normal(g, 16)
    slope = ((O.rope(x + step * vx, w, cos, sin, eps) - O.rope(x - step * vx, w, cos, sin, eps)) * d).sum() / (2 * step)
    assert abs(slope - (dx * vx).sum()) <= 1e-7 * (1 + dx.abs().sum())
    slope = ((O.rope(x, w + step * vw, cos, sin, eps) - O.rope(x, w - step * vw, cos, sin, eps)) * d).sum() / (2 * step)
    assert abs(slope - (dw * vw).sum()) <= 1e-7 * (1 + dw.abs().sum())
    dx, dw = O.rope_grad(x, None, cos, sin, eps, d)
    assert dw is None
    torch.testing.assert_close((dx * vx).sum(), (O.rope(vx, None, cos, sin, eps) * d).sum(), rtol=1e-10, atol=1e-10)


# ------------------------------------------------------------------ refusals of the C ABI
FAKE = ctypes.c_void_p(4096)  # never dereferenced: every call below fails before device work
ODD = ctypes.c_void_p(4100)


def test_pack_arguments_are_rejected(lib):
    def pack(x=FAKE, dt=L.BF16, rows=4, cols=64, stride=64, codes=FAKE, exps=FAKE):
        return lib.dsalt_pack8(x, dt, rows, cols, stride, codes, exps, None)

    assert pack(dt=5) == L.ERR_INVALID and pack(rows=-1) == L.ERR_INVALID and pack(cols=-1) == L.ERR_INVALID
    assert pack(stride=63) == L.ERR_INVALID and b"overlap" in lib.dsalt_last_error()
    assert pack(cols=(1 << 30) + 1, stride=1 << 40) == L.ERR_UNSUPPORTED
    for name in ("x", "codes", "exps"):
        assert pack(**{name: None}) == L.ERR_INVALID and b"null pointer" in lib.dsalt_last_error()
    assert pack(rows=0, x=None) == L.OK and pack(cols=0, x=None) == L.OK

    def unpack(codes=FAKE, exps=FAKE, rows=4, cols=64, out=FAKE, dt=L.F16):
        return lib.dsalt_unpack8(codes, exps, rows, cols, out, dt, None)

    assert unpack(dt=-1) == L.ERR_INVALID and unpack(rows=-1) == L.ERR_INVALID
    for name in ("codes", "exps", "out"):
        assert unpack(**{name: None}) == L.ERR_INVALID
    assert unpack(rows=0, out=None) == L.OK


def test_rope_arguments_are_rejected(lib):
    def fwd(q=FAKE, dt=L.BF16, T=8, H=4, Hk=2, D=64, qt=256, qh=64, wq=FAKE, wk=FAKE, wdt=L.F32, eps=1e-6, cos=FAKE,
            rows=100, stride=64, pos=FAKE, qo=FAKE):
        return lib.dsalt_qk_norm_rope(q, FAKE, dt, T, H, Hk, D, qt, qh, 128, 64, wq, wk, wdt, eps, cos, FAKE, rows, stride,
                                      pos, qo, FAKE, None)

    assert fwd(dt=9) == L.ERR_INVALID and fwd(wdt=9) == L.ERR_INVALID
    assert fwd(T=-1) == L.ERR_INVALID and fwd(H=0) == L.ERR_INVALID and fwd(rows=0) == L.ERR_INVALID
    assert fwd(stride=28) == L.ERR_INVALID and fwd(stride=33) == L.ERR_INVALID and b"aligned" in lib.dsalt_last_error()
    assert fwd(D=72) == L.ERR_UNSUPPORTED and fwd(D=272, stride=272) == L.ERR_UNSUPPORTED
    assert fwd(D=68, dt=L.F32, stride=68) == L.ERR_UNSUPPORTED and fwd(H=5000) == L.ERR_UNSUPPORTED
    assert fwd(pos=None, rows=7) == L.ERR_INVALID and b"tables of 7 rows" in lib.dsalt_last_error()
    assert fwd(wq=None) == L.ERR_INVALID and fwd(eps=-1.0) == L.ERR_INVALID and fwd(eps=float("nan")) == L.ERR_INVALID
    assert fwd(q=None) == L.ERR_INVALID and fwd(qo=None) == L.ERR_INVALID and fwd(cos=None) == L.ERR_INVALID
    assert fwd(q=ODD) == L.ERR_INVALID and fwd(qt=257) == L.ERR_INVALID and fwd(qh=68) == L.ERR_INVALID
    assert fwd(T=0, q=None, cos=None) == L.OK

    need = lib.dsalt_qk_norm_rope_bwd_workspace_bytes(64)
    assert need > 0 and need % 256 == 0 and lib.dsalt_qk_norm_rope_bwd_workspace_bytes(0) == 0

    def bwd(T=8, D=64, d=FAKE, dt_stride=256, wq=FAKE, wk=FAKE, dwq=FAKE, ws=FAKE, n=need):
        return lib.dsalt_qk_norm_rope_bwd(FAKE, FAKE, d, FAKE, L.BF16, T, 4, 2, D, 256, 64, 128, 64, dt_stride, 64, 128, 64,
                                          wq, wk, L.F32, 1e-6, FAKE, FAKE, 100, 64, FAKE, FAKE, FAKE, dwq, FAKE, ws, n,
                                          None)

    assert bwd(D=8) == L.ERR_UNSUPPORTED and bwd(d=None) == L.ERR_INVALID and bwd(dt_stride=4) == L.ERR_INVALID
    assert bwd(dwq=None) == L.ERR_INVALID and bwd(ws=None) == L.ERR_INVALID and bwd(n=need - 1) == L.ERR_WORKSPACE
    assert bwd(wk=None) == L.ERR_INVALID


def test_ffn_arguments_are_rejected(lib):
    need = lib.dsalt_gated_ffn_workspace_bytes(L.BF16, 8, 64, 96, 64)
    assert need > 0 and need % 256 == 0
    assert lib.dsalt_gated_ffn_workspace_bytes(7, 8, 64, 96, 64) == 0
    assert [lib.dsalt_gated_ffn_pitch(n) for n in (0, 1, 32, 33)] == [0, 32, 32, 64]

    def fwd(x=FAKE, dt=L.BF16, T=8, d=64, stride=64, F=96, d_out=64, act=L.ACT_SILU, keep=L.KEEP_NONE, kept=None, exps=None,
            y=FAKE, ws=FAKE, n=need):
        return lib.dsalt_gated_ffn(x, dt, T, d, stride, FAKE, FAKE, FAKE, F, d_out, act, keep, kept, exps, y, ws, n, None)

    assert fwd(dt=3) == L.ERR_INVALID and fwd(T=-1) == L.ERR_INVALID and fwd(F=0) == L.ERR_INVALID
    assert fwd(d=0) == L.ERR_INVALID and fwd(d_out=0) == L.ERR_INVALID
    assert fwd(act=2) == L.ERR_INVALID and fwd(keep=3) == L.ERR_INVALID
    assert fwd(T=1 << 28) == L.ERR_UNSUPPORTED and fwd(F=(1 << 20) + 8) == L.ERR_UNSUPPORTED
    assert fwd(stride=56) == L.ERR_INVALID and b"overlap" in lib.dsalt_last_error()
    assert fwd(x=None) == L.ERR_INVALID and fwd(y=None) == L.ERR_INVALID and fwd(ws=None) == L.ERR_INVALID
    assert fwd(keep=L.KEEP_INPUT) == L.ERR_INVALID and fwd(keep=L.KEEP_8BIT, kept=FAKE) == L.ERR_INVALID
    assert fwd(keep=L.KEEP_INPUT, kept=FAKE) == L.ERR_INVALID  # codes of 16 bits have scales
    assert fwd(n=need - 1) == L.ERR_WORKSPACE
    assert fwd(ws=ODD) == L.ERR_INVALID and fwd(keep=L.KEEP_INPUT, kept=ODD, exps=FAKE) == L.ERR_INVALID
    assert fwd(x=ODD) == L.ERR_INVALID and fwd(y=ODD) == L.ERR_INVALID and b"aligned" in lib.dsalt_last_error()
    assert fwd(stride=68) == L.ERR_INVALID and b"aligned" in lib.dsalt_last_error()
    # what only the plain path takes needs more workspace
    assert lib.dsalt_gated_ffn_workspace_bytes(L.BF16, 8, 64, 100, 64) > need
    assert lib.dsalt_gated_ffn_workspace_bytes(L.F32, 8, 64, 96, 64) > need
    assert fwd(T=0, x=None, y=None, ws=None) == L.OK

    need_b = lib.dsalt_gated_ffn_bwd_workspace_bytes(L.BF16, 8, 64, 96, 64, L.KEEP_8BIT)
    assert need_b > lib.dsalt_gated_ffn_bwd_workspace_bytes(L.BF16, 8, 64, 96, 64, L.KEEP_INPUT) > 0

    def bwd(dy=FAKE, x=FAKE, x_exps=FAKE, keep=L.KEEP_8BIT, kept=FAKE, exps=FAKE, dwg=FAKE, dwu=FAKE, ws=FAKE, n=need_b,
            stride=64, dt=L.BF16):
        return lib.dsalt_gated_ffn_bwd(dy, dt, 8, 64, stride, x, 64, x_exps, FAKE, FAKE, FAKE, 96, 64, L.ACT_GELU, keep, kept,
                                       exps, FAKE, dwg, dwu, FAKE, ws, n, None)

    assert bwd(keep=L.KEEP_NONE) == L.ERR_INVALID and b"keep" in lib.dsalt_last_error()
    assert bwd(dwg=None) == L.ERR_INVALID and b"go together" in lib.dsalt_last_error()
    assert bwd(dy=None) == L.ERR_INVALID and bwd(x=None) == L.ERR_INVALID and bwd(x_exps=None) == L.ERR_INVALID
    assert bwd(kept=None) == L.ERR_INVALID and bwd(exps=None) == L.ERR_INVALID and bwd(ws=None) == L.ERR_INVALID
    assert bwd(dy=ODD) == L.ERR_INVALID and bwd(dwg=ODD) == L.ERR_INVALID and bwd(stride=68) == L.ERR_INVALID
    assert bwd(stride=8) == L.ERR_INVALID and bwd(n=need_b - 1) == L.ERR_WORKSPACE and bwd(dt=4) == L.ERR_INVALID


# ------------------------------------------------------------------ the torch-facing functions
def test_functions_refuse_cpu_tensors():
    x, w = torch.zeros(4, 64), torch.zeros(96, 64)
    with pytest.raises(RuntimeError, match="CUDA"):
        Y.pack8(x)
    with pytest.raises(RuntimeError, match="CUDA"):
        Y.unpack8(torch.zeros(4, 64, dtype=torch.int8), torch.zeros(4, 2, dtype=torch.uint8))
    with pytest.raises(RuntimeError, match="CUDA"):
        Y.gated_ffn(x, w, w, torch.zeros(64, 96))
    with pytest.raises(RuntimeError, match="CUDA"):
        Y.gated_ffn(x.requires_grad_(True), w, w, torch.zeros(64, 96))
    q, k, t = torch.zeros(4, 2, 64), torch.zeros(4, 1, 64), torch.zeros(4, 64)
    with pytest.raises(RuntimeError, match="CUDA"):
        Y.qk_norm_rope(q, k, t, t)


# ------------------------------------------------------------------ the decoder stack
def test_config_and_modules_offer_the_kinds():
    from dsalt_b200.model import DSALTConfig, DSALTLMHeadModel, SwiGLUFFN
    small = dict(vocab_size=100, d_model=64, n_layers=1, n_heads=2, n_min=4, n_max=16, k_lmk=4, max_seq_len=64)
    with pytest.raises(ValueError, match="ffn must be one of"):
        DSALTConfig(**small, ffn="other")
    with pytest.raises(ValueError, match="kind must be one of"):
        SwiGLUFFN(64, 128, kind="8bit")
    plain, new = (DSALTLMHeadModel.from_config(DSALTConfig(**small, **kw)) for kw in ({}, dict(qk_norm=True, ffn="fused")))
    keys = set(new.state_dict())
    assert keys - set(plain.state_dict()) == {"layers.0.attn.q_norm.weight", "layers.0.attn.k_norm.weight"}
    assert set(plain.state_dict()) <= keys and new.layers[0].ffn.kind == "fused"
    assert DSALTConfig.from_dict(DSALTConfig(**small, qk_norm=True, ffn="fused_8bit").to_dict()).ffn == "fused_8bit"


def test_registered_forms_have_shape_functions():
    import dsalt_b200  # noqa: F401
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        new = lambda *s, dt=torch.bfloat16: torch.empty(*s, dtype=dt, device="cuda")  # noqa: E731
        q, k = torch.ops.dsalt_b200.qk_norm_rope(new(9, 4, 64), new(9, 2, 64), new(20, 64), new(20, 64),
                                                 new(9, dt=torch.int32), new(64), new(64), 1e-6)
        assert (q.shape, k.shape, q.dtype) == ((9, 4, 64), (9, 2, 64), torch.bfloat16)
        y = torch.ops.dsalt_b200.gated_ffn(new(2, 9, 64), new(96, 64), new(96, 64), new(48, 96), "gelu")
        assert y.shape == (2, 9, 48) and y.dtype == torch.bfloat16
        codes, exps = torch.ops.dsalt_b200.pack8(new(5, 70))
        assert (codes.shape, codes.dtype, exps.shape, exps.dtype) == ((5, 70), torch.int8, (5, 3), torch.uint8)
        assert torch.ops.dsalt_b200.unpack8(codes, exps, torch.float16).dtype == torch.float16
