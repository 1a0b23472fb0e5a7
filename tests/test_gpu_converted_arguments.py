"""Arguments that an operator converts (their type or layout) give the results of arguments that are
converted beforehand, whatever memory the copies get: a copy has to outlive the call that reads it."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def fresh_pool():
    """No free blocks of odd sizes: a copy that is given up is where the next one goes."""
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    yield


def same(a, b, tol=0.0):
    for x, y in zip(a, b):
        x, y = (torch.nan_to_num(t.double(), neginf=0.0) for t in (x, y))
        assert float((x - y).norm()) <= tol * float(y.norm())


def inputs(dtype):
    g = torch.Generator(device="cuda").manual_seed(5)
    cu = [0, 300, 760]
    T, H, Hk, D, k = cu[-1], 4, 2, 64, 16
    new = lambda *s: torch.randn(*s, device="cuda", generator=g).to(dtype)  # noqa: E731
    q, kk, v, do = new(T, H, D), new(T, Hk, D), new(T, Hk, D), new(T, H, D)
    w = (torch.rand(T, device="cuda", generator=g) * 56 + 8).bfloat16()
    pos = torch.stack([torch.stack([torch.randperm(n, device="cuda", generator=g)[:k] for n in (300, 460)]) for _ in range(H)])
    logw = (-torch.rand(H, 2, k, device="cuda", generator=g)).bfloat16()
    return cu, q, kk, v, do, w, pos, logw, torch.tensor(cu, device="cuda")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_training_attention(dtype):
    from dsalt_b200 import ops
    cu, q, k, v, do, w, pos, logw, cu_t = inputs(dtype)  # bf16 widths and log-weights, int64 positions and borders
    ready = w.float(), pos.to(torch.int32), logw.float(), cu_t.to(torch.int32)
    ref = ops.train_attention_forward(q, k, v, ready[1], ready[2], ready[0], ready[3], 1.0, 4.0, cu_list=cu)
    ref_g = ops.train_attention_backward(do, q, k, v, *ref, ready[1], ready[2], ready[0], ready[3], 1.0, 4.0, cu_list=cu)
    got = ops.train_attention_forward(q, k, v, pos, logw, w, cu_t, 1.0, 4.0, cu_list=cu)
    got_g = ops.train_attention_backward(do, q, k, v, *got, pos, logw, w, cu_t, 1.0, 4.0, cu_list=cu)
    same(got, ref)
    same(got_g, ref_g, 1e-6)  # fp32 atomics in any order


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_and_selection(dtype):
    from dsalt_b200 import ops
    cu, q, k, v, do, w, pos, _, cu_t = inputs(dtype)
    bias = torch.randn(pos.shape, device="cuda").bfloat16()
    i32 = w.to(torch.int32), cu_t.to(torch.int32)
    ref = ops.dsalt_attention(q, k, v, pos, bias, i32[0], i32[1], cu_list=cu, return_lse=True)
    got = ops.dsalt_attention(q, k, v, pos, bias, w, cu_t, cu_list=cu, return_lse=True)
    same(got, ref)
    ref_g = ops.dsalt_attention_backward(do, q, k, v, ref[0].to(dtype), ref[1], pos, bias, *i32, cu_list=cu)
    got_g = ops.dsalt_attention_backward(do, q, k, v, ref[0].to(dtype), ref[1], pos, bias, w, cu_t, cu_list=cu)
    same(got_g, ref_g, 1e-6)
    T = cu[-1]
    xn, vn = torch.rand(T, 2, device="cuda")[:, 0], torch.rand(2, T, device="cuda").t()  # neither is contiguous
    alpha = torch.full((4,), 0.625, device="cuda").bfloat16()
    ref = ops.select_landmarks(xn.contiguous(), vn.contiguous(), i32[0], alpha.float(), i32[1], 16, 4, "block_causal", 128, cu)
    assert torch.equal(ops.select_landmarks(xn, vn, w, alpha, cu_t, 16, 4, "block_causal", 128, cu), ref)
