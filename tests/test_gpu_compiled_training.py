"""The fused feed-forward block and the registered forms have gradients, under torch.compile as without."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def normal(seed, *shape, dtype=torch.bfloat16, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.empty(*shape, device="cuda").normal_(0, scale, generator=g).to(dtype)


def compiled(f, **kw):
    torch._dynamo.reset()
    return torch.compile(f, backend="aot_eager", **kw)


@pytest.mark.parametrize("kind", ["fused", "fused_8bit"])
def test_a_compiled_feed_forward_block_trains(kind):
    from dsalt_b200.model import SwiGLUFFN
    torch.manual_seed(1)
    m = SwiGLUFFN(64, 104, kind=kind).cuda().bfloat16()
    # a compiled block keeps nothing but its inputs: its gradients are those without 8 bits
    plain = SwiGLUFFN(64, 104, kind="fused").cuda().bfloat16()
    plain.load_state_dict(m.state_dict())
    x, dy = normal(2, 90, 64), normal(3, 90, 64)
    got_x, ref_x = (x.clone().requires_grad_(True) for _ in range(2))
    y = compiled(m, fullgraph=True)(got_x)
    y.backward(dy)
    ref = plain(ref_x)
    ref.backward(dy)
    assert torch.equal(y, ref) and torch.equal(got_x.grad, ref_x.grad)
    for a, b in zip(m.parameters(), plain.parameters()):
        assert torch.equal(a.grad, b.grad)


@pytest.mark.parametrize("weights", [True, False])
def test_compiled_head_norms_train(weights):
    import dsalt_b200  # noqa: F401
    from dsalt_b200 import layers
    q, k, dq, dk = (normal(i, 33, n, 64) for i, n in ((4, 3), (5, 1), (6, 3), (7, 1)))
    cos, sin = normal(8, 40, 64, dtype=torch.float32), normal(9, 40, 64, dtype=torch.float32)
    pos = torch.arange(33, device="cuda", dtype=torch.int32)
    w = [torch.rand(64, device="cuda") + 0.5 for _ in range(2)] if weights else [None, None]

    def leaves():
        return [t.detach().clone().requires_grad_(True) for t in (q, k, *w) if t is not None]

    def op(q, k, wq=None, wk=None):
        return tuple(torch.ops.dsalt_b200.qk_norm_rope(q, k, cos, sin, pos, wq, wk, 1e-6))

    a, b, c = leaves(), leaves(), leaves()
    got = torch.autograd.grad(compiled(op, fullgraph=True)(*a), a, (dq, dk))
    eager = torch.autograd.grad(op(*c), c, (dq, dk))
    kw = dict(q_weight=b[2], k_weight=b[3]) if weights else {}
    ref = torch.autograd.grad(layers.qk_norm_rope(b[0], b[1], cos, sin, positions=pos, **kw), b, (dq, dk))
    assert all(torch.equal(x, y) and torch.equal(z, y) for x, y, z in zip(got, ref, eager))


def test_gradients_of_the_registered_form_that_are_not_wanted():
    import dsalt_b200  # noqa: F401
    from dsalt_b200 import layers
    ts = normal(1, 20, 64), normal(2, 96, 64, scale=0.1), normal(3, 96, 64, scale=0.1), normal(4, 40, 96, scale=0.1)
    dy = normal(5, 20, 40)
    for wanted in ((0,), (1,), (3,), (2, 3), (0, 1, 2, 3)):
        both = [[t.detach().requires_grad_(i in wanted) for i, t in enumerate(ts)] for _ in range(2)]
        got = torch.autograd.grad(torch.ops.dsalt_b200.gated_ffn(*both[0], "gelu"), [both[0][i] for i in wanted], dy)
        ref = torch.autograd.grad(layers.gated_ffn(*both[1], activation="gelu"), [both[1][i] for i in wanted], dy)
        assert all(torch.equal(a, b) for a, b in zip(got, ref))
    x = ts[0].detach().requires_grad_(True)
    with pytest.raises(RuntimeError):  # no second derivative
        g, = torch.autograd.grad(torch.ops.dsalt_b200.gated_ffn(x, *ts[1:], "silu").float().square().sum(), x, create_graph=True)
        g.sum().backward()
