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


# ------------------------------------------------------------------ min_p above 1
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab,top_k,top_p", [(40, 0, 1.0), (5000, 0, 1.0), (5000, 0, 0.999), (5000, 3000, 1.0),
                                               (5000, 20, 0.9), (151936, 0, 0.9999)])
def test_min_p_above_one_leaves_the_first_of_the_order(V, dtype, vocab, top_k, top_p):
    """The largest weight is 1: nothing reaches a larger min_p, and the first of the order stays, as it does under
    every filter. Rows with such a min_p stand among ordinary ones."""
    g = torch.Generator(device="cuda").manual_seed(vocab)
    lg = (torch.randn(6, vocab, device="cuda", generator=g) * 2).to(dtype)
    lg[2, 31] = lg[2, 7] = 40.0  # two largest: the lower index
    min_p = torch.tensor([1.5, 0.0, 1.5, 0.01, float("inf"), 1.0], device="cuda")
    u = torch.tensor([0.9, 0.3, 0.999, 0.6, 0.0, 0.7], device="cuda")
    tok, lp = V.sample_tokens(lg, u, temperature=1.7, top_k=top_k, top_p=top_p, min_p=min_p, return_logprob=True)
    f32 = lambda x: float(np.float32(x))  # noqa: E731
    for i in range(6):
        t, l, margin = O.sample(lg[i].double().cpu().numpy(), float(u[i]), f32(1.7), top_k, f32(top_p), float(min_p[i]))
        if i in (0, 2, 4):
            assert (t, l) == (int(lg[i].float().argmax()) if i != 2 else 7, 0.0)
        if margin >= 2.0 ** -43 * vocab:  # as far as the order of sums may move a border
            assert int(tok[i]) == t
            assert abs(float(lp[i]) - l) <= 2.0 ** -23 * (abs(l) + 1)
    assert (lp[[0, 2, 4]] == 0).all()


# ------------------------------------------------------------------ rare tokens
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("vocab", [5, 3000, 60000])
def test_log_probability_of_rare_tokens(V, dtype, vocab):
    """The log-probability is that of the drawn logit, whatever its weight: log w - log of the sum. Bound: the
    result's own rounding, half a step of |lp|, and the sum's: at most V + 1 roundings of 2^-44 against a sum of
    at least 1, 2^-28 here, both well within 2^-23 (|lp| + 1)."""
    ones = -(2.0 ** -6) * (torch.arange(vocab, device="cuda") % 3)
    rows = torch.stack([ones] * 5).to(dtype)
    rare = [-25.0, -28.0, -29.25, -27.0, -20.0]
    for i, x in enumerate(rare):
        rows[i, 0] = x  # the first in index order: a small u draws it
    mass = torch.exp(rows.double()).sum(1)
    u = (torch.exp(rows[:, 0].double()) / mass * 0.4).float()
    for min_p in (0.0, 1e-15):
        tok, lp = V.sample_tokens(rows, u, min_p=min_p, return_logprob=True)
        for i in range(5):
            t, l, _ = O.sample(rows[i].double().cpu().numpy(), float(u[i]), 1.0, 0, 1.0, min_p)
            assert t == 0 and int(tok[i]) == 0
            assert abs(float(lp[i]) - l) <= 2.0 ** -23 * (abs(l) + 1), (i, float(lp[i]), l)


def test_log_probability_of_rare_tokens_in_a_list(V):
    # five candidates of 100, as top-k leaves them: settled in the list of one block
    lg = torch.full((1, 100), -60.0, device="cuda")
    lg[0, 2], lg[0, 50:54] = -26.0, torch.tensor([0.0, -0.5, -1.0, 0.25], device="cuda")
    row = lg[0].double().cpu().numpy()
    keep = np.sort(np.argsort(-row, kind="stable")[:5])
    p = np.exp(row[keep] - row.max())
    u = torch.tensor([0.4 * p[0] / p.sum()], device="cuda").float()
    tok, lp = V.sample_tokens(lg, u, top_k=5, return_logprob=True)
    t, l, _ = O.sample(row, float(u[0]), 1.0, 5, 1.0, 0.0)
    assert t == 2 and int(tok) == 2
    assert abs(float(lp) - l) <= 2.0 ** -23 * (abs(l) + 1)
