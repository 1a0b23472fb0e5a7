"""Rows of a cache that end and begin on their own: prompts and decode steps of some rows while
the others hold sequences, or nothing."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _model(**kw):
    from dsalt_b200 import DSALTConfig, DSALTLMHeadModel
    torch.manual_seed(3)
    cfg = DSALTConfig(**{**dict(vocab_size=777, d_model=256, n_layers=2, n_heads=4, n_min=8, n_max=64, k_lmk=16,
                                max_seq_len=400, d_ff=512, n_kv_heads=2, qkv_bias=True, selection="block_causal", block=128), **kw})
    return DSALTLMHeadModel.from_config(cfg).cuda().bfloat16().eval()


def _prompts(*lens):
    g = torch.Generator().manual_seed(5)
    return [torch.randint(0, 777, (n,), generator=g).cuda() for n in lens]


def _cu(*lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return cu


def test_rows_without_a_sequence_are_passed_over():
    """Prompts for two of three rows and their decode steps equal those of a cache of two rows, bit for
    bit: the same tokens are packed and nothing else is computed."""
    from dsalt_b200 import ops
    m = _model()
    a, b = _prompts(125, 60)
    three, two = m.new_cache(3, 200, page_size=16), m.new_cache(2, 200, page_size=16)
    ids = torch.cat([a, b])
    x, y = m.prefill(ids, _cu(125, 0, 60), three), m.prefill(ids, _cu(125, 60), two)
    assert three.lens == [125, 0, 60] and three.seq_lens.tolist() == [125, 0, 60]
    for _ in range(8):  # the first row crosses a block border
        assert x.shape == (3, 777) and torch.equal(x[[0, 2]], y) and (x[1] == 0).all()
        tokens = x.argmax(1)
        tokens[1] = 10**6  # of a row without a sequence: not looked at
        x, y = m.decode(tokens, three), m.decode(y.argmax(1), two)
    assert three.lens == [133, 0, 68] and three.seq_lens.tolist() == [133, 0, 68]
    assert int(three.n_free) == three.n_pages - three.pages_held()
    assert ops.device_status() == 0


def test_a_row_ends_and_another_takes_its_place():
    """One row ends, the others go on, a new prompt takes its place, all go on. A cache without the first
    life of the row makes the same calls on the same tokens: everything is equal bit for bit, although the
    pages, the landmark sets and the statistics of the first life were written over."""
    from dsalt_b200 import ops
    m = _model()
    a, first, b, second = _prompts(125, 140, 60, 90)
    used, fresh = (m.new_cache(3, 200, n_pages=21, page_size=16) for _ in range(2))
    x = m.prefill(first, _cu(0, 140, 0), used)
    for _ in range(3):
        x = m.decode(x.argmax(1), used)
    assert used.lens == [0, 143, 0]
    used.release([1])
    assert int(used.n_free) == used.n_pages and used.lens == [0, 0, 0]
    caches = used, fresh
    xs = [m.prefill(torch.cat([a, b]), _cu(125, 0, 60), c) for c in caches]
    for _ in range(2):
        assert torch.equal(*xs)
        xs = [m.decode(x.argmax(1), c) for x, c in zip(xs, caches)]
    ys = [m.prefill(second, _cu(0, 90, 0), c) for c in caches]  # rows 0 and 2 hold sequences meanwhile
    assert torch.equal(*ys) and (ys[0][[0, 2]] == 0).all() and not (ys[0][1] == 0).all()
    for x, y in zip(xs, ys):
        x[1] = y[1]
    for step in range(6):  # row 0 crosses a block border
        assert torch.equal(*xs)
        assert all(torch.isfinite(x).all() for x in xs)
        xs = [m.decode(x.argmax(1), c) for x, c in zip(xs, caches)]
    assert used.lens == fresh.lens == [133, 96, 68]
    assert used.seq_lens.tolist() == used.lens
    # a row that ends while the others go on gives its pages back
    used.release([0])
    assert int(used.n_free) == used.n_pages - used.pages_held() and used.lens == [0, 96, 68]
    x = m.decode(xs[0].argmax(1), used)
    assert used.lens == [0, 97, 69] and (x[0] == 0).all()
    assert ops.device_status() == 0


def test_a_full_row_can_end_alone():
    m = _model()
    a, b = _prompts(30, 5)
    cache = m.new_cache(2, 32, page_size=16)
    x = m.prefill(torch.cat([a, b]), _cu(30, 5), cache)
    for _ in range(2):
        x = m.decode(x.argmax(1), cache)
    with pytest.raises(ValueError, match="cache for 32"):
        m.decode(x.argmax(1), cache)
    assert cache.lens == [32, 7]
    cache.release([0])
    x = m.decode(x.argmax(1), cache)
    assert cache.lens == [0, 8] and x.shape == (2, 777)


def test_refusals_name_rows_that_hold_sequences():
    m = _model()
    a, b = _prompts(9, 4)
    cache = m.new_cache(2, 40, page_size=16)
    m.prefill(a, _cu(9, 0), cache)
    with pytest.raises(ValueError, match="empty rows"):
        m.prefill(torch.cat([a, b]), _cu(9, 4), cache)
    with pytest.raises(ValueError, match="at least one"):
        m.prefill(a[:0], _cu(0, 0), cache)
    with pytest.raises(ValueError, match="one prompt"):
        m.prefill(a, [0, 9, 8], cache)  # borders that fall
    assert cache.lens == [9, 0]
    m.prefill(b, _cu(0, 4), cache)
    assert cache.lens == [9, 4]
    cache.release([0, 1])
    with pytest.raises(ValueError, match="prompt"):
        m.decode(a[:2], cache)


def test_prompts_and_steps_make_their_device_the_current_one(monkeypatch):
    """The signals, the selection and the packed attention launch on the current device: a model that is
    elsewhere has to make its own the current one first (seen here by the guards that are entered)."""
    from dsalt_b200 import ops
    m = _model()
    cache = m.new_cache(2, 200, page_size=16)
    a, b = _prompts(140, 9)
    guard, inside, calls = torch.cuda.device, [], []

    class Recorded(guard):
        def __enter__(self):
            inside.append(self.idx)
            return super().__enter__()

        def __exit__(self, *args):
            inside.pop()
            return super().__exit__(*args)

    monkeypatch.setattr(torch.cuda, "device", Recorded)
    run = ops.L.call
    monkeypatch.setattr(ops.L, "call", lambda name, *args: calls.append((name, list(inside))) or run(name, *args))
    x = m.prefill(torch.cat([a, b]), _cu(140, 9), cache)
    m.decode(x.argmax(1), cache)
    older = [c for c in calls if c[0] in ("dsalt_token_signals", "dsalt_select_landmarks", "dsalt_attention_fwd",
                                          "dsalt_select_block_range")]
    assert len(older) >= 2 * 5 and all(at and at[-1] == cache.lmk.device.index for _, at in older)
