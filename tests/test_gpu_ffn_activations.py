"""The feed-forward block's activations by themselves: inputs and weights that make gate and up known numbers, against their
formulas in 64 bits, from far negative gates on."""
import pytest
import torch

from oracle import layers_oracle as O

pytestmark = pytest.mark.gpu


def probe(v, size, up, dtype, keep, grad=True):
    """``(act(v) up, act'(v) up)`` of each value of ``v`` by the operator: one input is the value, another is 1."""
    from dsalt_b200 import layers
    T = v.shape[0]
    x = torch.zeros(T, size, device="cuda", dtype=dtype)
    x[:, 0], x[:, 1] = v, 1
    wg, wu, wd = (torch.zeros(size, size, device="cuda", dtype=dtype) for _ in range(3))
    wg[0, 0], wu[0, 1], wd[0, 0] = 1, up, 1
    out = {}
    for act in ("silu", "gelu"):
        leaf = x.clone().requires_grad_(grad)
        y = layers.gated_ffn(leaf, wg, wu, wd, activation=act, keep=keep)
        dy = torch.zeros_like(y)
        dy[:, 0] = 1
        out[act] = y[:, 0].detach(), torch.autograd.grad(y, leaf, dy)[0][:, 0] if grad else None
    return out


def test_activations_of_fp32_inputs():
    v = torch.cat([torch.linspace(-87, 87, 4001), torch.linspace(-13, 13, 4001), torch.linspace(-1e-3, 1e-3, 101)]).cuda()
    got = probe(v, 2, 1.0, torch.float32, "16bit")
    g = v.double()
    for act, (y, dx) in got.items():
        p, dp = O.share(g, act)
        far = (g * p).abs() >= 2.0 ** -126   # below it fewer bits are left
        # silu: an exponential of two steps of 2^-23, three operations of half a step; gelu: CUDA's distribution function
        # of five steps, or an exponential and a product, and three operations
        tol = {"silu": 2.0 ** -21, "gelu": 2.0 ** -20}[act]
        over = ((y.double() - g * p).abs() - tol * (g * p).abs())[far]
        assert (over <= 0).all(), (act, float(g[far][over.argmax()]))
        size = p + (g * dp).abs()
        far = size >= 2.0 ** -120
        over = ((dx.double() - (p + g * dp)).abs() - tol * size)[far]
        assert (over <= 0).all(), (act, float(g[far][over.argmax()]))


@pytest.mark.parametrize("T", [8, 16, 100, 6000])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("grad", [True, False])
def test_activations_of_16_bit_inputs(T, dtype, grad):
    e = torch.finfo(dtype).eps / 2
    for lo, hi in ((-5.5, -0.01), (-0.5, 3.0)):
        v = torch.linspace(lo, hi, T, device="cuda").to(dtype)
        got = probe(v, 8, 1024.0, dtype, "16bit", grad)
        g = v.double()
        for act, (y, dx) in got.items():
            p, dp = O.share(g, act)
            # half a step of the type for the product of gate and up (the last product and the result are exact then),
            # 2^-15 for the activation
            ref = 1024 * g * p
            over = (y.double() - ref).abs() - (e + 2.0 ** -15) * ref.abs()
            assert (over <= 0).all(), (act, float(g[over.argmax()]), float(over.max()))
            if grad:
                ref, size = 1024 * (p + g * dp), 1024 * (p + (g * dp).abs())
                over = (dx.double() - ref).abs() - e * ref.abs() - 2.0 ** -15 * size - 2.0 ** -25
                assert (over <= 0).all(), (act, float(g[over.argmax()]), float(over.max()))
