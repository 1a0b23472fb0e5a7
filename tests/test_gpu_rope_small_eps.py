"""Gradients of the head norms' weights with eps = 0: places of a warp that hold no head give nothing."""
import pytest
import torch

from oracle import layers_oracle as O

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("eps", [0.0, 1e-50])  # the second is 0 in 32 bits
@pytest.mark.parametrize("T,H,Hk,D", [(1, 1, 1, 64), (7, 3, 1, 64), (33, 5, 3, 32), (300, 12, 3, 128), (1001, 1, 1, 16)])
def test_weight_gradients_without_eps(dtype, eps, T, H, Hk, D):
    from dsalt_b200 import layers, ops
    g = torch.Generator(device="cuda").manual_seed(T + D)
    new = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    q, k, dq, dk = (new(T, n, D).to(dtype) for n in (H, Hk, H, Hk))
    w = [(torch.rand(D, device="cuda", generator=g) + 0.5) for _ in range(2)]
    cos, sin = new(T, D // 2), new(T, D // 2)
    leaves = [t.requires_grad_(True) for t in (q, k, *w)]
    out = layers.qk_norm_rope(q, k, cos, sin, q_weight=w[0], k_weight=w[1], eps=eps)
    grads = torch.autograd.grad(out, leaves, (dq, dk))
    assert ops.device_status() == 0
    for i, (x, d) in enumerate(((q, dq), (k, dk))):
        X, W, Dy = x.detach().double(), w[i].detach().double(), d.double()
        dx, dw = O.rope_grad(X, W, cos.double(), sin.double(), 0.0, Dy)
        # some twenty fp32 operations a term, n terms added up; dx is rounded to its type
        r = 1 / torch.sqrt((X * X).mean(-1, keepdim=True))
        size = Dy.abs().amax(-1, keepdim=True) * 8
        assert ((grads[2 + i].double() - dw).abs() <=
                (2.0 ** -19 + min(X.shape[0] * X.shape[1], 4096) * 2.0 ** -24) * (size * (X * r).abs().amax(-1, keepdim=True)).sum()).all()
        xr = (X * r).abs().amax(-1, keepdim=True)
        assert ((grads[i].double() - dx).abs() <=
                torch.finfo(dtype).eps / 2 * dx.abs() + 2.0 ** -19 * r * size * W.max() * (1 + xr * xr)).all()
