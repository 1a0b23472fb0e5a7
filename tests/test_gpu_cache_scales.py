"""Attention over caches whose scales are not the powers of two that ``append_cache`` writes."""
import numpy as np
import pytest
import torch
from test_gpu_serving import attend_case, oracle_of, to_gpu

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("H,Hkv,D,page,lens,q_lens,w_max,k", [
    (4, 2, 64, 16, [200, 40], [1, 1], 0, 0), (2, 1, 128, 32, [400], [3], 60, 12), (4, 4, 64, 64, [2500], [1], 0, 0),
    (8, 1, 128, 16, [90, 500], [1, 2], 100, 33)])
def test_scales_of_any_size(dtype, H, Hkv, D, page, lens, q_lens, w_max, k):
    """Against the float64 oracle. A row's error, relative to sum p|v| / sum p, counted as for powers of two:
    logits (D + 8) 2^-22 of their largest sum of magnitudes, |lse| 2^-21, sums (n + 8) 2^-22, P half a step of
    its fp16 terms, each twice at most; and of the logarithm of a page's scale 2^-22, times ln 2, once, with
    one rounding of it (its size is below 16: 2^-20 times ln 2)."""
    from dsalt_b200 import ops, serving
    c = attend_case(21, lens, q_lens, H, Hkv, D, page, dtype, w_max, k)
    g = np.random.default_rng(3)
    for name in ("ks", "vs"):  # significands over [1, 2), held in fp32
        c[name] = (c[name] * g.uniform(1, 2, c[name].shape)).astype(np.float32).astype(np.float64)
    out, lse = serving.cache_attention(**to_gpu(c), return_lse=True)
    assert ops.device_status() == 0
    ref, rl, spread, size, n = oracle_of(c)
    E = (D + 8) * 2.0 ** -22 * size + (np.abs(rl) + 1) * 2.0 ** -21 + (n + 8) * 2.0 ** -22
    half = torch.finfo(dtype).eps / 2
    flat = torch.finfo(dtype).smallest_normal * half
    p = 2.0 ** -21 if dtype == torch.float32 else 2.0 ** -11
    log = (2.0 ** -22 + 2.0 ** -20) * np.log(2)
    tol = half * np.abs(ref) * (1 + 2 ** -8) + (2 * np.expm1(E) + p + log)[..., None] * spread + flat
    assert (np.abs(out.double().cpu().numpy() - ref) <= tol).all()
    assert (np.abs(lse.double().cpu().numpy() - rl) <= E + 2.0 ** -22 * (np.abs(rl) + 1)).all()


def test_one_scale_of_all_values_multiplies_the_result():
    """out is linear in a scale that all pages share: the same P whatever the significand (the logarithm is the
    same for all, its error too: 2^-22 and a rounding of x + e below 2^-20, times ln 2, either side)."""
    from dsalt_b200 import serving
    c = to_gpu(attend_case(22, [300], [1], 2, 1, 64, 16, torch.float32))
    c["v_scale"].fill_(1.0)
    one = serving.cache_attention(**c)
    for s in (1.9999999, 1.3, 0.7, 3e-5, 0.0123):
        c["v_scale"].fill_(s)
        got = serving.cache_attention(**c).double() / float(c["v_scale"][0, 0])
        assert ((got - one.double()).abs() <= 2 * 2.0 ** -20 * one.double().abs().max()).all()
