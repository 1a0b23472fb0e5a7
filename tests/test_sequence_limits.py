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


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_training_keeps_no_more_of_the_tables_than_its_sequences_need(dtype):
    from dsalt_b200 import DSALTAttention
    torch.manual_seed(1)
    rows = 16384
    m = DSALTAttention(128, 2, 4, 16, 4, rows, qk_norm=True).cuda().to(dtype).train()
    cu = [0, 100, 130]
    x = torch.randn(130, 128, device="cuda", dtype=dtype)
    kept = []

    def pack(t):
        kept.append(t.untyped_storage().nbytes() if t.untyped_storage().data_ptr() not in own else 0)
        return t

    own = {t.untyped_storage().data_ptr() for t in (*m.parameters(), *m.buffers(), x)}
    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
        q, _, _ = m._qkv(x, cu, 130, x.device, None)
    q.float().sum().backward()
    assert 0 < max(kept) <= 130 * 128 * 4  # a projection of the pack at most, of the tables 100 rows
    pos = torch.cat([torch.arange(b - a) for a, b in zip(cu, cu[1:])]).cuda()
    with torch.no_grad():
        ref, _, _ = m._qkv(x, cu, 130, x.device, (m.rope_cos.float()[pos], m.rope_sin.float()[pos]))
    assert torch.equal(q.detach(), ref)
