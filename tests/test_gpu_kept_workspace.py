"""Memory that a training forward pass of the feed-forward block asks for beside what it keeps."""
import pytest
import torch

from dsalt_b200 import _lib as L


@pytest.fixture(scope="module")
def lib():
    import os
    if not os.path.exists(L.LIB_PATH):
        from dsalt_b200 import build
        build.build()
    return L.load()


def test_workspaces_by_what_is_kept(lib):
    def need(dtype, keep, F=96):
        return lib.dsalt_gated_ffn_keep_workspace_bytes(dtype, 1000, 64, F, 64, keep)

    for dtype in (L.F32, L.BF16, L.F16):
        for F in (96, 100):
            whole = lib.dsalt_gated_ffn_workspace_bytes(dtype, 1000, 64, F, 64)
            assert need(dtype, L.KEEP_NONE, F) == whole
            assert need(dtype, L.KEEP_8BIT, F) == whole
            # kept as it is, fp32's sums and their product are formed where they are kept
            assert need(dtype, L.KEEP_INPUT, F) == (256 if dtype == L.F32 else whole)
    assert need(7, L.KEEP_NONE) == 0 and need(L.F32, 5) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,more", [(torch.float32, 0), (torch.bfloat16, 2)])
def test_a_training_forward_pass_needs_what_it_keeps(lib, dtype, more):
    from dsalt_b200 import layers
    T, d, F = 4096, 64, 2048
    x = torch.randn(T, d, device="cuda", dtype=dtype)
    w = [torch.randn(s, device="cuda", dtype=dtype).mul_(0.1).requires_grad_(True) for s in ((F, d), (F, d), (d, F))]
    layers.gated_ffn(x, *w)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    y = layers.gated_ffn(x, *w)
    kept = 3 * T * F * x.element_size()
    # gate, up and the product's rows or third bytes, the result, and of 16-bit types the product as an operand
    assert torch.cuda.max_memory_allocated() - before <= kept + more * T * F + y.numel() * x.element_size() + (4 << 20)
