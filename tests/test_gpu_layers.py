"""Head norm and rotation, 8-bit activations and the gated feed-forward block on the GPU against
their float64 oracle (``oracle.layers_oracle``). Tolerances are sums of what each rounding can do:
half a step of the type where a value is rounded to it, and a stated share of the sum of magnitudes
where products are added up."""
import pytest
import torch

from oracle import layers_oracle as O

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


@pytest.fixture(scope="module")
def Y():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from dsalt_b200 import layers
    return layers


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape, dtype=torch.float32, scale=1.0):
    return torch.empty(*shape, device="cuda").normal_(0, scale, generator=g).to(dtype)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def assert_within(got, ref, tol, what):
    got = got.double()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    over = (got - ref).abs() - tol
    assert bool((over <= 0).all()), f"{what}: off by {float((got - ref).abs().max())}, {float(over.max())} too much"


def assert_no_status():
    from dsalt_b200 import ops
    assert ops.device_status() == 0


# ------------------------------------------------------------------ 8 bits
def same_pack(Y, x):
    codes, exps = Y.pack8(x)
    flat = x.double().reshape(-1, x.shape[-1])
    c, s = O.pack(flat)
    assert codes.dtype == torch.int8 and exps.dtype == torch.uint8
    assert codes.shape == x.shape and exps.shape == x.shape[:-1] + (-(-x.shape[-1] // 32),)
    assert torch.equal(codes.reshape(c.shape), c) and torch.equal(exps.reshape(s.shape), s)
    for dt in TYPES.values():
        got = Y.unpack8(codes, exps, dt)
        ref = O.unpack(c, s).to(dt).view(x.shape)
        assert got.dtype == dt and torch.equal(got.isnan(), ref.isnan())
        assert torch.equal(got.nan_to_num(7.0), ref.nan_to_num(7.0))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 32), (3, 31), (5, 33), (64, 48), (7, 1000), (33, 1024), (129, 4096),
                                       (2, 100001), (70001, 8)])
def test_pack_matches_the_oracle(Y, dtype, rows, cols):
    g = gen(rows * 7 + cols)
    x = normal(g, rows, cols) * torch.exp(normal(g, rows, cols))
    same_pack(Y, x.to(TYPES[dtype]))


@pytest.mark.parametrize("dtype", list(TYPES))
def test_pack_of_borders_zeros_and_values_that_are_not_finite(Y, dtype):
    dt = TYPES[dtype]
    info = torch.finfo(dt)
    x = torch.zeros(12, 64, device="cuda")
    x[0, :] = torch.arange(64, device="cuda") - 31.5           # ties
    x[1, 3] = info.max
    x[1, 40] = -info.max
    x[2, 5], x[2, 6] = info.smallest_normal, info.tiny / 2
    x[3, 0] = float("nan")
    x[4, 31], x[4, 32] = float("inf"), 1.0
    x[5, 63] = -float("inf")
    x[6, :] = 127.5
    x[7, :] = 127.0
    x[8, :32] = torch.linspace(-127.9, 127.9, 32)
    x[9, 7] = 2.0 ** -20
    x[10, :] = -0.0
    same_pack(Y, x.to(dt))
    if dt == torch.float32:  # far below and above what 16-bit types hold, and below the normal range
        y = torch.full((2, 40), 1e-45, device="cuda")
        y[0, 1], y[1, 1], y[1, 33] = 3e38, 2.0 ** -126, 1e-39
        same_pack(Y, y)


def test_pack_of_other_shapes_strides_and_streams(Y):
    g = gen(3)
    wide = normal(g, 40, 256)
    same_pack(Y, wide[:, 32:160])            # rows apart, 16-byte aligned
    same_pack(Y, wide[:, 33:160])            # odd start
    same_pack(Y, wide.t())                   # columns
    same_pack(Y, wide.view(5, 8, 256))
    same_pack(Y, wide[0])
    same_pack(Y, wide[:1].expand(6, 256))
    same_pack(Y, normal(g, 1, 1)[0, 0].view(1))
    codes, exps = Y.pack8(wide[:0])
    assert codes.shape == (0, 256) and exps.shape == (0, 8) and Y.unpack8(codes, exps).shape == (0, 256)
    codes, exps = Y.pack8(wide[:, :0])
    assert codes.shape == (40, 0) and exps.shape == (40, 0) and Y.unpack8(codes, exps).shape == (40, 0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = Y.unpack8(*Y.pack8(wide), torch.float32)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got.double(), O.held(wide.double()))


def test_pack_refusals(Y):
    x = torch.zeros(4, 64, device="cuda")
    with pytest.raises(TypeError):
        Y.pack8(x.double())
    with pytest.raises(TypeError):
        Y.pack8(x[:0].long())
    with pytest.raises(ValueError):
        Y.pack8(x[0, 0])
    codes, exps = Y.pack8(x)
    with pytest.raises(ValueError):
        Y.unpack8(codes, exps[:, :1])
    with pytest.raises(TypeError):
        Y.unpack8(exps, exps)
    with pytest.raises(TypeError):
        Y.unpack8(codes, exps, torch.int32)
    with pytest.raises(RuntimeError):
        Y.unpack8(codes, exps.cpu())


# ------------------------------------------------------------------ heads
def rope_tables(rows, D, base=10000.0):
    theta = base ** (-torch.arange(0, D, 2, device="cuda", dtype=torch.float64) / D)
    a = torch.outer(torch.arange(rows, device="cuda", dtype=torch.float64), theta)
    return [torch.cat([t, t], 1).float() for t in (a.cos(), a.sin())]


def rope_tolerance(ref, dtype, size):
    """Half a step for the result's rounding, 2^-19 of the largest for some twenty fp32 operations."""
    return half_step(dtype) * ref.abs() + 2.0 ** -19 * size


def check_rope(Y, q, k, wq, wk, cos, sin, positions, eps, seed=5):
    T, H, D = q.shape
    at = positions.long() if positions is not None else torch.arange(T, device="cuda")
    c, s = cos.double()[at, :D // 2], sin.double()[at, :D // 2]
    g = gen(seed)
    dt = q.dtype
    dq, dk = normal(g, *q.shape, dtype=dt), normal(g, *k.shape, dtype=dt)
    kw = dict(positions=positions, q_weight=wq, k_weight=wk, eps=eps)
    with torch.no_grad():
        plain = Y.qk_norm_rope(q, k, cos, sin, **kw)
    leaves = [t.detach().requires_grad_(True) for t in (q, k)]
    if wq is not None:
        leaves += [t.detach().requires_grad_(True) for t in (wq, wk)]
        kw.update(q_weight=leaves[2], k_weight=leaves[3])
    out = Y.qk_norm_rope(leaves[0], leaves[1], cos, sin, **kw)
    grads = torch.autograd.grad(out, leaves, (dq, dk))
    again = torch.autograd.grad(Y.qk_norm_rope(leaves[0], leaves[1], cos, sin, **kw), leaves, (dq, dk))
    assert all(torch.equal(a, b) for a, b in zip(grads, again))
    assert_no_status()
    for i, (x, w, d) in enumerate(((q, wq, dq), (k, wk, dk))):
        x64, w64 = x.double(), None if w is None else w.double()
        ref = O.rope(x64, w64, c, s, eps)
        size = ref.abs().amax(-1, keepdim=True)
        assert out[i].is_contiguous() and out[i].dtype == dt and torch.equal(out[i], plain[i])
        assert_within(out[i], ref, rope_tolerance(ref, dt, size), f"output {i}")
        dx, dw = O.rope_grad(x64, w64, c, s, eps, d.double())
        if w is None:
            assert_within(grads[i], dx, rope_tolerance(dx, dt, d.double().abs().amax(-1, keepdim=True) * 2), f"gradient {i}")
            continue
        r = 1 / torch.sqrt((x64 * x64).mean(-1, keepdim=True) + eps)
        # the gradient of x: terms of the size r |w d| and, through the mean, r |x r| mean|w d x r|
        wd = (d.double().abs().amax(-1, keepdim=True) * 2) * w64.abs().max()
        xr = (x64 * r).abs().amax(-1, keepdim=True)
        assert_within(grads[i], dx, rope_tolerance(dx, dt, r * wd * (1 + xr * xr)), f"gradient {i}")
        # the weight's: n products added up in fp32, each sum of at most n terms in some order
        terms = 2 * d.double().abs().amax(-1) * (x64 * r).abs().amax(-1)
        n = x.shape[0] * x.shape[1]
        tol = (2.0 ** -19 + min(n, 4096) * 2.0 ** -24) * terms.sum() + half_step(w.dtype) * dw.abs()
        assert_within(grads[2 + i], dw, tol, f"weight gradient {i}")


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("T,H,Hk,D,norm", [
    (1, 1, 1, 16, True), (1, 16, 2, 128, True), (64, 16, 2, 128, True), (7, 5, 1, 96, True), (333, 12, 12, 64, True),
    (1000, 6, 2, 64, False), (257, 4, 4, 256, True), (129, 3, 1, 48, False), (5000, 9, 3, 32, True), (31, 2, 2, 240, True)])
def test_rope_matches_the_oracle(Y, dtype, T, H, Hk, D, norm):
    g, dt = gen(T + D), TYPES[dtype]
    q, k = normal(g, T, H, D, dtype=dt), normal(g, T, Hk, D, dtype=dt, scale=3.0)
    cos, sin = rope_tables(T + 3, D)
    wq, wk = (torch.rand(D, device="cuda", generator=g) + 0.5 for _ in range(2)) if norm else (None, None)
    pos = torch.randint(0, T + 3, (T,), device="cuda", generator=g, dtype=torch.int32) if T % 2 else None
    check_rope(Y, q, k, wq, wk, cos, sin, pos, 1e-6)


def test_rope_of_views_tables_and_weights_of_other_forms(Y):
    g = gen(11)
    T, H, Hk, D = 37, 4, 2, 64
    qkv = normal(g, T, H + 2 * Hk, D, dtype=torch.bfloat16)
    cos, sin = rope_tables(100, D)
    wq, wk = (torch.rand(D, device="cuda", generator=g).bfloat16() + 0.5 for _ in range(2))
    pos = torch.randint(0, 100, (T,), device="cuda", generator=g)  # int64
    check_rope(Y, qkv[:, :H], qkv[:, H:H + Hk], wq, wk, cos, sin, pos, 1e-5)
    # tables of the first half alone, cut from a wider one
    check_rope(Y, qkv[:, :H], qkv[:, H:H + Hk], wq, wk, cos[:, :D // 2], sin[:, :D // 2], pos, 1e-5)
    odd = normal(g, T, H, D + 1, dtype=torch.bfloat16)[:, :, 1:]   # rows that no 16-byte load takes
    check_rope(Y, odd, qkv[:, H:H + Hk], None, None, cos, sin, pos, 1e-5)
    check_rope(Y, qkv[:, :H].transpose(0, 1).contiguous().transpose(0, 1), qkv[:, H:H + Hk], wq, wk, cos, sin, pos, 1e-5)
    # one token, one row of angles
    check_rope(Y, qkv[:1, :H], qkv[:1, H:H + Hk], wq, wk, cos[5:6], sin[5:6], None, 1e-5)


def test_rope_gradients_that_are_broadcast_or_missing(Y):
    g = gen(12)
    T, H, Hk, D = 19, 4, 2, 64
    q, k = normal(g, T, H, D).requires_grad_(True), normal(g, T, Hk, D).requires_grad_(True)
    w = (torch.rand(D, device="cuda", generator=g) + 0.5).requires_grad_(True)
    cos, sin = rope_tables(T, D)
    qo, ko = Y.qk_norm_rope(q, k, cos, sin, q_weight=w, k_weight=w)   # one weight for both
    (qo.sum() * 3).backward()                                         # the keys' output is not used
    c, s = cos.double()[:, :D // 2], sin.double()[:, :D // 2]
    dx, dw = O.rope_grad(q.detach().double(), w.detach().double(), c, s, 1e-6, torch.full((T, H, D), 3.0, device="cuda").double())
    torch.testing.assert_close(q.grad.double(), dx, rtol=1e-5, atol=1e-5)
    torch.testing.assert_close(w.grad.double(), dw, rtol=1e-5, atol=1e-4)
    assert k.grad.abs().max() == 0


def test_rope_of_no_tokens_and_zero_heads_and_values_that_are_not_finite(Y):
    cos, sin = rope_tables(8, 64)
    w = torch.ones(64, device="cuda", requires_grad=True)
    q, k = torch.zeros(0, 4, 64, device="cuda"), torch.zeros(0, 2, 64, device="cuda")
    qo, ko = Y.qk_norm_rope(q, k, cos, sin, q_weight=w, k_weight=w)
    assert qo.shape == (0, 4, 64) and ko.shape == (0, 2, 64)
    assert torch.autograd.grad(qo.sum() + ko.sum(), w)[0].abs().max() == 0
    q, k = torch.zeros(3, 4, 64, device="cuda"), torch.ones(3, 2, 64, device="cuda")
    q[1, 2, 5] = float("nan")
    q[2, 0, 0] = float("inf")
    with torch.no_grad():
        qo, ko = Y.qk_norm_rope(q, k, cos, sin, q_weight=w, k_weight=w)
    assert qo[0].abs().max() == 0 and qo[1, 2].isnan().all() and qo[1, :2].abs().max() == 0
    assert not torch.isfinite(qo[2, 0]).all() and torch.isfinite(qo[2, 1:]).all() and torch.isfinite(ko).all()


def test_rope_position_outside_the_tables_is_reported(Y):
    from dsalt_b200 import ops
    g = gen(13)
    q, k = normal(g, 3, 2, 64), normal(g, 3, 1, 64)
    cos, sin = rope_tables(8, 64)
    ref = Y.qk_norm_rope(q, k, cos, sin, positions=torch.tensor([0, 7, 0], device="cuda"))
    assert ops.device_status() == 0
    got = Y.qk_norm_rope(q, k, cos, sin, positions=torch.tensor([8, 7, -1], device="cuda"))
    assert ops.device_status() == 51 and ops.device_status() == 0
    assert all(torch.equal(a, b) for a, b in zip(got, ref))
    far = torch.tensor([1 << 32, 7, -(1 << 40)], device="cuda")   # not what 32 bits would make of them
    got = Y.qk_norm_rope(q, k, cos, sin, positions=far)
    assert ops.device_status() == 51 and all(torch.equal(a, b) for a, b in zip(got, ref))


def test_rope_refusals(Y):
    g = gen(14)
    q, k = normal(g, 3, 2, 64), normal(g, 3, 1, 64)
    cos, sin = rope_tables(8, 64)
    w = torch.ones(64, device="cuda")
    bad = [
        (ValueError, dict(q=q[0])), (ValueError, dict(k=k[:2])), (TypeError, dict(k=k.half())),
        (ValueError, dict(k=k[..., :32])), (ValueError, dict(q_weight=w)), (ValueError, dict(q_weight=w[:32], k_weight=w)),
        (TypeError, dict(q_weight=w, k_weight=w.half())), (TypeError, dict(q_weight=w.double(), k_weight=w.double())),
        (ValueError, dict(cos=cos[:, :48])), (ValueError, dict(cos=cos[:4])), (ValueError, dict(cos=cos[:2], sin=sin[:2])),
        (ValueError, dict(positions=torch.zeros(4, dtype=torch.int32, device="cuda"))),
        (ValueError, dict(positions=torch.zeros(3, device="cuda"))), (RuntimeError, dict(cos=cos.cpu())),
        (TypeError, dict(q=q.double(), k=k.double())),
    ]
    for error, change in bad:
        args = dict(dict(q=q, k=k, cos=cos, sin=sin), **change)
        with pytest.raises(error):
            Y.qk_norm_rope(**args)
    from dsalt_b200 import DsaltError
    for D in (40 + 4, 264):
        c, s = rope_tables(8, D)
        with pytest.raises(DsaltError):
            Y.qk_norm_rope(normal(g, 3, 2, D), normal(g, 3, 1, D), c, s)


# ------------------------------------------------------------------ feed-forward
def near(x, dev):
    """How far the 8-bit form of values within ``dev`` of ``x`` may be from that of ``x``: a step where a
    value lies within ``dev`` of a tie, two for the whole group where its largest lies within ``dev`` of a
    power of two."""
    _, exps = O.pack(x)
    step = torch.exp2(exps.double() - 127).repeat_interleave(32, 1)[:, :x.shape[1]]
    at = (x / step).abs()
    tie = ((at - torch.floor(at)) - 0.5).abs() * step <= dev
    top_at = at == torch.cat([at, at.new_zeros(at.shape[0], -at.shape[1] % 32)], 1).view(
        at.shape[0], -1, 32).amax(-1).repeat_interleave(32, 1)[:, :at.shape[1]]
    edge = top_at & (((at - 64) * step <= 2 * dev) | ((128 - at) * step <= 2 * dev))
    rows, n = x.shape
    edge = torch.cat([edge, edge.new_zeros(rows, -n % 32)], 1).view(rows, -1, 32).any(-1).repeat_interleave(32, 1)[:, :n]
    return torch.where(edge, 2 * step, torch.where(tie, step, torch.zeros_like(step)))


def check_ffn(Y, x, wg, wu, wd, act, keep, dy):
    dt, e = x.dtype, half_step(x.dtype)
    T, d = x.shape
    F, n_out = wg.shape[0], wd.shape[0]
    leaves = [t.detach().requires_grad_(True) for t in (x, wg, wu, wd)]
    with torch.no_grad():
        plain = Y.gated_ffn(x, wg, wu, wd, activation=act)
    y = Y.gated_ffn(*leaves, activation=act, keep=keep)
    grads = torch.autograd.grad(y, leaves, dy)
    again = torch.autograd.grad(Y.gated_ffn(*leaves, activation=act, keep=keep), leaves, dy)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))
    assert_no_status()
    X, G, U, D, dY = (t.detach().double() for t in (x, wg, wu, wd, dy))

    def summed(K):  # n additions in fp32, or in the tensor cores' accumulators
        return (K + 8) * 2.0 ** -23

    g, u = X @ G.T, X @ U.T
    p, dp = O.share(g, act)
    a, da = g * p, p + g * dp
    slope, bend = 1.13, 0.8  # bounds of |act'| and |act''|
    dev_g, dev_u = summed(d) * (X.abs() @ G.abs().T), summed(d) * (X.abs() @ U.abs().T)
    h = a * u
    dev_a = slope * dev_g + 2.0 ** -18 * (a.abs() + g.abs() * 2.0 ** -4)
    dev_h = dev_a * u.abs() + a.abs() * dev_u + dev_a * dev_u
    ref = h @ D.T
    held_h = e * (h.abs() + dev_h) + 2.0 ** -25 + dev_h   # rounded as an operand; fp16 below its normal range too
    tol = held_h @ D.abs().T + summed(F) * ((h.abs() + held_h) @ D.abs().T)
    assert y.dtype == dt
    assert_within(y, ref, tol * (1 + e) + e * ref.abs() + 2.0 ** -25, "output")
    assert_within(plain, ref, tol * (1 + e) + e * ref.abs() + 2.0 ** -25, "output without gradients")

    if keep == "8bit":
        far_g, far_u = near(g, dev_g), near(u, dev_u)
        g, u, X = O.held(g), O.held(u), O.held(X)
    else:
        def top(t):  # the largest of each group of 32
            t = torch.cat([t.abs(), t.new_zeros(t.shape[0], -t.shape[1] % 32)], 1).view(t.shape[0], -1, 32)
            return t.amax(-1).repeat_interleave(32, 1)[:, :F]
        # half a step of codes of 16 bits (fp32: as they are)
        step = 0 if dt == torch.float32 else 2.0 ** -15
        far_g, far_u = dev_g + step * top(g.abs() + dev_g), dev_u + step * top(u.abs() + dev_u)
    p, dp = O.share(g, act)
    a, da = g * p, p + g * dp
    h = a * u
    refs = O.ffn_grad(X, G, U, D, act, dY, g, u)
    dh = dY @ D
    dev_dh = summed(n_out) * (dY.abs() @ D.abs())
    dg, du = dh * u * da, dh * a
    far_a = slope * far_g + 2.0 ** -18 * (a.abs() + g.abs() * 2.0 ** -4)
    far_da = bend * far_g + 2.0 ** -18 * (1 + g.abs())
    D_, U_ = dh.abs() + dev_dh, u.abs() + far_u
    dev_dg = dev_dh * u.abs() * da.abs() + D_ * far_u * da.abs() + D_ * U_ * far_da
    dev_du = dev_dh * a.abs() + D_ * far_a
    dev_h = far_a * U_ + a.abs() * far_u
    dev_dg, dev_du, dev_h = (t + e * (v.abs() + t) + 2.0 ** -25 for t, v in ((dev_dg, dg), (dev_du, du), (dev_h, h)))
    adg, adu, ah = dg.abs() + dev_dg, du.abs() + dev_du, h.abs() + dev_h
    tols = [dev_dg @ G.abs() + dev_du @ U.abs() + summed(2 * F) * (adg @ G.abs() + adu @ U.abs()),
            dev_dg.T @ X.abs() + summed(T) * (adg.T @ X.abs()), dev_du.T @ X.abs() + summed(T) * (adu.T @ X.abs()),
            dY.abs().T @ dev_h + summed(T) * (dY.abs().T @ ah)]
    for got, ref, tol, name in zip(grads, refs, tols, ("x", "w_gate", "w_up", "w_down")):
        assert got.dtype == dt
        assert_within(got, ref, tol * (1 + e) + e * ref.abs() + 2.0 ** -25, "gradient of " + name)
        # and as a whole: the tolerances above add up worst cases
        miss = (got.double() - ref).norm() / ref.norm()
        assert miss <= 4 * e + 2.0 ** -16 + (2.0 ** -9 if keep == "8bit" else 0), (name, float(miss))


def ffn_inputs(T, d, F, d_out, dtype, seed=0):
    g = gen(seed + T + d + F)
    return (normal(g, T, d, dtype=dtype), normal(g, F, d, dtype=dtype, scale=d ** -0.5),
            normal(g, F, d, dtype=dtype, scale=d ** -0.5), normal(g, d_out, F, dtype=dtype, scale=F ** -0.5),
            normal(g, T, d_out, dtype=dtype, scale=0.1))


@pytest.mark.parametrize("dtype,keep", [("bf16", "16bit"), ("bf16", "8bit"), ("fp16", "16bit"), ("fp16", "8bit"),
                                        ("fp32", "16bit"), ("fp32", "8bit")])
@pytest.mark.parametrize("T,d,F,d_out,act", [
    (1, 64, 96, 64, "silu"), (1, 8, 8, 8, "gelu"), (3, 72, 40, 24, "silu"), (17, 256, 768, 256, "gelu"),
    (64, 512, 1408, 512, "silu"), (127, 128, 136, 200, "silu"), (300, 264, 520, 136, "gelu"), (513, 768, 2048, 768, "silu"),
    (1000, 200, 328, 200, "silu"), (2500, 512, 1408, 512, "silu"), (4100, 264, 2824, 520, "gelu"),
    (8, 520, 264, 1032, "silu"), (9, 1024, 2816, 72, "gelu"), (16, 200, 5504, 520, "silu"), (255, 72, 4104, 264, "silu"),
    (256, 1032, 520, 520, "gelu"), (40, 2056, 1000, 2048, "silu"), (6000, 72, 200, 72, "silu"), (1100, 256, 4104, 256, "silu")])
def test_ffn_matches_the_oracle(Y, dtype, keep, T, d, F, d_out, act):
    x, wg, wu, wd, dy = ffn_inputs(T, d, F, d_out, TYPES[dtype])
    check_ffn(Y, x, wg, wu, wd, act, keep, dy)


# where the forms without gradients meet, and where they are cut differently
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("T,d,F,d_out", [
    (48, 136, 1032, 72), (49, 136, 1032, 72), (64, 136, 1032, 2048), (65, 136, 1032, 2048), (128, 72, 19000, 64),
    (129, 72, 19000, 64), (193, 1024, 1048, 264), (640, 200, 1048, 264), (208, 72, 11008, 136), (209, 72, 11008, 136),
    (2048, 200, 1048, 264), (2049, 200, 1048, 264), (300, 64, 264, 9000), (1500, 2048, 8, 8)])
def test_ffn_at_the_borders_of_its_forms(Y, dtype, T, d, F, d_out):
    x, wg, wu, wd, dy = ffn_inputs(T, d, F, d_out, TYPES[dtype])
    check_ffn(Y, x, wg, wu, wd, "silu", "16bit", dy)


@pytest.mark.parametrize("dtype,keep", [("bf16", "16bit"), ("fp16", "8bit"), ("fp32", "8bit")])
@pytest.mark.parametrize("T,d,F,d_out", [(5, 7, 9, 3), (130, 33, 65, 129), (2, 64, 100, 64), (9, 65, 64, 64)])
def test_ffn_of_odd_sizes(Y, dtype, keep, T, d, F, d_out):
    x, wg, wu, wd, dy = ffn_inputs(T, d, F, d_out, TYPES[dtype])
    check_ffn(Y, x, wg, wu, wd, "silu", keep, dy)
