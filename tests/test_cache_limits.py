"""What a paged cache refuses when it is made, without a GPU: sizes that its operators do not take."""
import pytest
import torch

from dsalt_b200 import DSALTConfig, DSALTLMHeadModel, PagedCache


def _model(**kw):
    return DSALTLMHeadModel.from_config(DSALTConfig(**{**dict(
        vocab_size=50, d_model=128, n_layers=1, n_heads=2, n_min=4, n_max=8, k_lmk=4, max_seq_len=64, d_ff=64,
        selection="block_causal", block=16), **kw}))


@pytest.mark.parametrize("n_heads", [4, 1, 8])  # heads of 32, 128, 16
def test_head_sizes_are_refused_before_a_cache_is_made(n_heads):
    m = _model(n_heads=n_heads)
    if n_heads == 1:
        assert m.new_cache(2, 40, page_size=16).k.shape[-1] == 128
        return
    with pytest.raises(ValueError, match=f"head size {128 // n_heads}"):
        m.new_cache(2, 40)


def test_a_vocabulary_beyond_sampling_is_refused():
    m = _model(n_heads=2)
    m.embed_tokens = torch.nn.Embedding((1 << 20) + 1, 1)
    with pytest.raises(ValueError, match="vocabulary of 1048577"):
        m.eval().generate([[1, 2]], 2)


def test_cache_sizes_are_refused():
    make = lambda **kw: PagedCache(**{**dict(n_layers=1, n_heads=4, n_kv_heads=2, head_dim=64, k_lmk=4, max_seqs=2,  # noqa: E731
                                             max_len=40, page_size=16, device="cpu"), **kw})
    assert make().k.shape == (1, 6, 2, 16, 64)
    for kw, match in ((dict(page_size=24), "page_size"), (dict(max_seqs=0), "max_seqs"), (dict(max_seqs=8193), "max_seqs"),
                      (dict(head_dim=96), "head size 96"), (dict(n_kv_heads=3), "multiple"),
                      (dict(n_pages=1 << 27), "pool"), (dict(max_len=1 << 31), "max_len")):
        with pytest.raises(ValueError, match=match):
            make(**kw)
