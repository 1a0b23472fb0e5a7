"""Sampling on the GPU at the limits of its settings and sizes, against the float64 oracle
(``oracle.serving_oracle``)."""
import numpy as np
import pytest
import torch

from oracle import serving_oracle as O

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def V():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from dsalt_b200 import serving
    return serving


# ------------------------------------------------------------------ the largest vocabulary, few values
@pytest.mark.parametrize("low,dtype", [(-8.317767, torch.float32), (-8.375, torch.bfloat16), (0.0, torch.float16)])
def test_largest_vocabulary_of_two_values(V, low, dtype):
    """All logits but one equal (or all): whole shares fall into one bin, and each border is a place among
    equal logits. Every setting's borders lie further away than the order of 64-bit sums can move them."""
    vocab = 1 << 20
    lg = torch.full((1, vocab), low, device="cuda").to(dtype)
    lg[0, 777777] = 0.0
    row = lg[0].double().cpu().numpy()
    for p, k, u in ((0.99999, 0, 0.71), (0.6180339, 0, 0.123), (0.8, 0, 0.5001), (1.0, 700001, 0.4142)):
        tok, lp = V.sample_tokens(lg, torch.tensor([u], device="cuda"), top_k=k, top_p=p, return_logprob=True)
        t, l, margin = O.sample(row, float(np.float32(u)), 1.0, k, float(np.float32(p)), 0.0)
        assert margin >= 2.0 ** -43 * vocab
        assert int(tok) == t
        assert abs(float(lp) - l) <= 2.0 ** -23 * (abs(l) + 1)
