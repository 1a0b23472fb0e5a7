"""What ``gated_ffn(keep="16bit")`` keeps of gate and up is held value by value: features of other sizes, infinities and
values near the ends of the range do not touch their neighbours."""
import pytest
import torch

from oracle import layers_oracle as O

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def inputs(T, d, F, d_out, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    new = lambda scale, *s: torch.empty(*s, device="cuda").normal_(0, scale, generator=g).to(dtype)  # noqa: E731
    return new(1, T, d), new(d ** -0.5, F, d), new(d ** -0.5, F, d), new(F ** -0.5, d_out, F), new(1, T, d_out)


def gradients(x, wg, wu, wd, dy, act="silu"):
    from dsalt_b200 import layers, ops
    leaves = [t.detach().requires_grad_(True) for t in (x, wg, wu, wd)]
    grads = torch.autograd.grad(layers.gated_ffn(*leaves, activation=act), leaves, dy)
    assert ops.device_status() == 0
    return grads


@pytest.mark.parametrize("dtype,less", [("bf16", -10), ("bf16", -14), ("fp16", -10)])
@pytest.mark.parametrize("T,d,F,d_out", [(256, 64, 128, 64), (100, 33, 70, 65)])
def test_small_features_beside_large_ones_keep_their_gradients(dtype, less, T, d, F, d_out):
    """Of 32 neighbouring features one is as it is; the others' gate or up values are 2^less times as large."""
    dt = TYPES[dtype]
    e = torch.finfo(dt).eps / 2
    x, wg, wu, wd, dy = inputs(T, d, F, d_out, dt, 1)
    dy = dy * 8                                   # so that fp16 holds the small gradients in its normal range
    for which in (wg, wu):
        x_, w = x, [wg.clone(), wu.clone()]
        rows = torch.arange(F, device="cuda") % 32 != 5
        w[0 if which is wg else 1][rows] *= 2.0 ** less
        _, dwg, dwu, _ = gradients(x_, *w, wd, dy)
        X, G, U, D, Dy = (t.double() for t in (x, *w, wd, dy))
        _, rg, ru, _ = O.ffn_grad(X, G, U, D, "silu", Dy)
        # Row by row in the 2-norm: half a step each for the held gate, the held up, the gradient of their
        # sum as an operand and the result; sums of some hundred products in 32 bits are far below
        for got, ref in ((dwg, rg), (dwu, ru)):
            miss = (got.double() - ref).norm(dim=1) / ref.norm(dim=1)
            assert miss.max() <= 4 * e, (float(miss.max()), int(miss.argmax()))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("T,d,F", [(40, 64, 96), (300, 64, 128), (40, 33, 70)])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_a_feature_that_is_not_finite_leaves_the_others_gradients(dtype, T, d, F, bad):
    dt = TYPES[dtype]
    x, wg, wu, wd, dy = inputs(T, d, F, 40, dt, 2)
    ref = gradients(x, wg, wu, wd, dy)
    for i in (0, 1):
        w = [wg.clone(), wu.clone()]
        w[i][37, 3] = bad
        got = gradients(x, *w, wd, dy)
        others = torch.arange(F, device="cuda") != 37
        for j in (1, 2):
            assert torch.equal(got[j][others], ref[j][others])
        assert torch.equal(got[3][:, others], ref[3][:, others])
        assert not torch.isfinite(got[2 - i][37]).all()


@pytest.mark.parametrize("T,d,F", [(64, 64, 128), (64, 33, 70)])
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_gates_near_the_end_of_the_range(T, d, F, act):
    """Gate's sums of some 2^120, whose gradients are ordinary numbers."""
    e = torch.finfo(torch.bfloat16).eps / 2
    x, wg, wu, wd, dy = inputs(T, d, F, 64, torch.bfloat16, 3)
    x, wg, wu, dy = x * 2.0 ** 60, wg * 2.0 ** 60, wu * 2.0 ** -60, dy * 2.0 ** -100
    got = gradients(x, wg, wu, wd, dy, act)
    X, G, U, D, Dy = (t.double() for t in (x, wg, wu, wd, dy))
    ref = O.ffn_grad(X, G, U, D, act, Dy)
    for a, b in zip(got, ref):
        assert torch.isfinite(a).all()
        assert (a.double() - b).norm() <= 4 * e * b.norm()


@pytest.mark.parametrize("T,d,F", [(200, 64, 128), (64, 33, 70)])
def test_held_values_are_within_their_stated_bound(T, d, F):
    """dw_down = dy^T h with one token chosen: h = act(gate) up from the held values, each off by 2^-15 of itself."""
    x, wg, wu, wd, _ = inputs(T, d, F, F, torch.float16, 4)
    dy = torch.zeros(T, F, device="cuda", dtype=torch.float16)
    dy[7] = 1
    got = gradients(x, wg, wu, wd, dy)[3]
    X, G, U = x[7].double(), wg.double(), wu.double()
    g, u = G @ X, U @ X
    p, dp = O.share(g, "silu")
    h = g * p * u
    sums = (d + 8) * 2.0 ** -23                                     # of d products in 32 bits
    off = [2.0 ** -15 * v.abs() + sums * (w.abs() @ X.abs()) for v, w in ((g, G), (u, U))]
    tol = ((p + g * dp).abs() + 0.8 * off[0]) * off[0] * u.abs() + (g * p).abs() * off[1] + 2 * off[0] * off[1]
    tol = tol + 2.0 ** -11 * h.abs() + 2.0 ** -18 * h.abs() + 2.0 ** -24   # as an operand; the activation
    assert ((got[0].double() - h).abs() <= tol * (1 + 2.0 ** -10)).all()
    assert all(torch.equal(got[0], row) for row in got)


@pytest.mark.parametrize("size", [8, 3])
def test_sums_of_few_bits_are_held_exactly(size):
    """Gates that fp16 holds, where silu's derivative changes its sign: the gradient of x shows the slightest change of them."""
    from dsalt_b200 import layers
    v = torch.linspace(-1.32, -1.24, 100, device="cuda").half()
    x, w = torch.zeros(100, size, device="cuda").half(), torch.zeros(3, size, size, device="cuda").half()
    x[:, 0], x[:, 1] = v, 1
    w[0, 0, 0], w[1, 0, 1], w[2, 0, 0] = 1, 1024, 1
    leaf = x.clone().requires_grad_(True)
    dy = torch.zeros(100, size, device="cuda").half()
    dy[:, 0] = 1
    dx, = torch.autograd.grad(layers.gated_ffn(leaf, *w), leaf, dy)
    g = v.double()
    p, dp = O.share(g, "silu")
    ref = 1024 * (p + g * dp)
    # half a step of fp16, and some ten operations in 32 bits on terms of the size of p
    assert ((dx[:, 0].double() - ref).abs() <= 2.0 ** -11 * ref.abs() + 1024 * 2.0 ** -20 * p).all()
