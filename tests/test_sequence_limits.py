"""Sequences longer than a module's tables of angles are refused on the host, before anything runs."""
import pytest
import torch

SMALL = dict(n_heads=2, n_min=4, n_max=16, k_lmk=4, max_seq_len=64)


@pytest.mark.parametrize("qk_norm", [True, False])
@pytest.mark.parametrize("training", [True, False])
def test_attention_refuses_sequences_beyond_its_tables(qk_norm, training):
    from dsalt_b200 import DSALTAttention
    m = DSALTAttention(64, **SMALL, qk_norm=qk_norm).train(training)
    cu = [0, 10, 75]
    with pytest.raises(ValueError, match="65 tokens.*max_seq_len 64"):
        m(torch.zeros(75, 64), torch.tensor(cu, dtype=torch.int32), cu_list=cu)


@pytest.mark.parametrize("qk_norm", [True, False])
def test_model_refuses_sequences_beyond_its_tables(qk_norm):
    from dsalt_b200 import DSALTLMHeadModel
    m = DSALTLMHeadModel(100, 64, 1, **SMALL, qk_norm=qk_norm).eval()
    cu = [0, 65, 70]
    with pytest.raises(ValueError, match="65 tokens.*max_seq_len 64"):
        m(torch.zeros(70, dtype=torch.long), torch.tensor(cu, dtype=torch.int32), cu_list=cu)
