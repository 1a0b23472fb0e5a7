"""Prompts and decode steps of the module and the model over the paged 8-bit cache, against the
packed attention of the same package on the values that the cache holds."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _module(n_kv, bias, dtype, **kw):
    from dsalt_b200 import DSALTAttention
    torch.manual_seed(0)
    m = DSALTAttention(256, 4, 8, 60, kw.get("k_lmk", 16), 1024, n_kv_heads=n_kv, qkv_bias=bias, selection="block_causal",
                       block=128)
    torch.nn.init.normal_(m.win_gate.weight, std=0.1)  # widths over their whole range
    m._collect_last_P = False
    return m.cuda().to(dtype).eval()


def _rope(m, positions):
    return m.rope_cos.cuda()[positions.long()], m.rope_sin.cuda()[positions.long()]


def _held(cache, layer, which, row, n):
    """The first n keys or values of a row, as the cache holds them: [n, H_kv, D] fp32."""
    x, s = (cache.k, cache.k_scale) if which == "k" else (cache.v, cache.v_scale)
    pages = cache.block_tables[row].long()[: -(-n // cache.page_size)]
    vals = x[layer][pages].float() * s[layer][pages][..., None, None]
    return vals.permute(0, 2, 1, 3).reshape(-1, x.shape[2], x.shape[4])[:n]


@pytest.mark.parametrize("n_kv,bias,dtype,k_lmk", [(4, False, torch.bfloat16, 16), (2, True, torch.float16, 16),
                                                   (4, False, torch.float32, 0)])
def test_decode_attends_as_the_packed_attention_does(n_kv, bias, dtype, k_lmk):
    """Each decode step equals the packed block-causal attention of the whole sequence so far at its
    last position: same widths, same landmark sets (across block borders), on the cached values."""
    from dsalt_b200 import ops
    from dsalt_b200.serving import PagedCache
    m = _module(n_kv, bias, dtype, k_lmk=k_lmk)
    D, H = m.head_dim, m.n_heads
    prompts, steps = [125, 3, 250], 9
    cache = PagedCache(1, H, n_kv, D, k_lmk, max_seqs=3, max_len=300, page_size=16)
    g = torch.Generator(device="cuda").manual_seed(1)
    xs = [torch.randn(n + steps, 256, device="cuda", generator=g).to(dtype) for n in prompts]
    cu = [0, 125, 128, 378]
    plan = cache.reserve(prompts)
    x0 = torch.cat([x[:n] for x, n in zip(xs, prompts)])
    whole, _ = m(x0, plan.cu_new, cu_list=cu)
    got = m.prefill(x0, plan.cu_new, cu, _rope(m, plan.positions), cache, plan)
    assert torch.equal(got, whole)  # prompts run as forward does
    seen = []
    keep = cache.attention
    cache.attention = lambda layer, q, w: seen.append((q, w, keep(layer, q, w))) or seen[-1][2]
    for t in range(steps):
        plan = cache.reserve([1] * 3)
        x = torch.stack([xs[r][prompts[r] + t] for r in range(3)])
        m.decode(x, _rope(m, plan.positions), cache, plan)
        q, w, out = seen[-1]
        for r in range(3):
            n = prompts[r] + t + 1
            full = xs[r][:n]
            cu_r = torch.tensor([0, n], dtype=torch.int32, device="cuda")
            v_all = m.v_proj(full).view(n, n_kv, D)
            w_all, xn, vn = m._signals(full, v_all)
            # a row alone or in a batch: the library products may differ in the last bit, and so may a width
            assert abs(int(w[r]) - int(w_all[-1])) <= 1
            held = cache.width[0, r, :n].contiguous()
            lmk = ops.select_landmarks(cache.xnorm[0, r, :n].contiguous(), cache.vnorm[0, r, :n].contiguous(), held,
                                       m._alpha().detach().float(), cu_r, k_lmk, H, "block_causal", 128, [0, n])
            b = (n - 1) // 128
            if k_lmk:
                assert torch.equal(lmk[:, b], cache.lmk[0][:, r])
            kk, vv = _held(cache, 0, "k", r, n), _held(cache, 0, "v", r, n)
            qq = torch.zeros(n, H, D, device="cuda")
            qq[-1] = q[r].float()
            ref = ops.dsalt_attention(qq, kk.contiguous(), vv.contiguous(), lmk, None, held, cu_r, lmk_block=128,
                                      cu_list=[0, n], out_dtype=torch.float32)[-1]
            # the reference runs in fp32; the cached attention rounds P to fp16 (2^-11 relative, twice in
            # out = sum p v / sum p) and its result to the type, all relative to the largest value
            half = torch.finfo(dtype).eps / 2
            tol = (2.0 ** -10 + half if dtype != torch.float32 else 1e-5) * vv.abs().max()
            assert (out[r].float() - ref).abs().max() <= tol
    assert ops.device_status() == 0


def _model(**kw):
    from dsalt_b200 import DSALTConfig, DSALTLMHeadModel
    torch.manual_seed(3)
    cfg = DSALTConfig(**{**dict(vocab_size=777, d_model=256, n_layers=2, n_heads=4, n_min=8, n_max=64, k_lmk=16,
                                max_seq_len=400, d_ff=512, n_kv_heads=2, qkv_bias=True, selection="block_causal", block=128), **kw})
    return DSALTLMHeadModel.from_config(cfg).cuda().bfloat16().eval()


def test_generate_is_repeatable_and_follows_its_own_steps():
    m = _model()
    g = torch.Generator().manual_seed(5)
    prompts = [torch.randint(0, 777, (n,), generator=g).tolist() for n in (125, 1, 130)]
    runs = [m.generate(prompts, 12, temperature=0.9, top_k=40, top_p=0.95,
                       generator=torch.Generator(device="cuda").manual_seed(8)) for _ in range(2)]
    assert runs[0] == runs[1] and [len(a) for a in runs[0]] == [12] * 3
    assert all(0 <= t < 777 for a in runs[0] for t in a)
    # greedy: the first token is the largest logit of the packed forward
    greedy = m.generate(prompts, 3, temperature=0.0)
    ids = torch.tensor([t for p in prompts for t in p], device="cuda")
    cu = [0, 125, 126, 256]
    logits = m(ids, torch.tensor(cu, dtype=torch.int32, device="cuda"), cu_list=cu)["logits"]
    last = logits[torch.tensor(cu[1:], device="cuda") - 1].float()
    cache = m.new_cache(3, 140)
    own = m.prefill(ids, cu, cache).float()
    # the head runs on 3 rows instead of 256: its sums of 256 products may differ in order
    assert (own - last).abs().max() <= 2.0 ** -7 * last.abs().max()
    assert [a[0] for a in greedy] == own.argmax(1).tolist()
    step = m.decode(own.argmax(1), cache)
    assert step.shape == (3, 777) and torch.isfinite(step.float()).all()
    assert cache.lens == [126, 2, 131] and cache.seq_lens.tolist() == [126, 2, 131]
    assert int(cache.n_free) == cache.n_pages - cache.pages_held()


def test_generate_ends_at_the_eos_token_and_rows_are_reused():
    m = _model()
    prompts = [[1, 2, 3], [4] * 65]
    free = m.generate(prompts, 8, temperature=0.0)
    eos = free[0][2]
    cut = m.generate(prompts, 8, temperature=0.0, eos_token=eos)
    assert cut[0] == free[0][: free[0].index(eos) + 1]
    assert cut[1] == (free[1][: free[1].index(eos) + 1] if eos in free[1] else free[1][: len(cut[1])])
    cache = m.new_cache(2, 100, page_size=16)
    ids = torch.tensor(prompts[0] + prompts[1], device="cuda")
    a = m.prefill(ids, [0, 3, 68], cache)
    m.decode(a.argmax(1), cache)
    cache.release([0, 1])
    assert int(cache.n_free) == cache.n_pages and cache.lens == [0, 0]
    b = m.prefill(ids, [0, 3, 68], cache)
    assert torch.equal(a, b)


def test_generation_refuses_what_it_cannot_hold():
    m = _model(selection="global")
    with pytest.raises(NotImplementedError, match="block_causal"):
        m.generate([[1, 2]], 2)
    m = _model()
    with pytest.raises(ValueError, match="max_seq_len"):
        m.generate([[1] * 390], 20)
    with pytest.raises(ValueError, match="at least one token"):
        m.generate([[1], []], 2)
    cache = m.new_cache(2, 40, n_pages=2, page_size=16)
    with pytest.raises(ValueError, match="pool of 2"):
        m.prefill(torch.ones(50, dtype=torch.long, device="cuda"), [0, 25, 50], cache)
    with pytest.raises(ValueError, match="cache for 40"):
        cache.reserve([41, 0])
    with pytest.raises(ValueError, match="prompt in every row"):
        m.decode(torch.ones(2, dtype=torch.long, device="cuda"), cache)
    m.prefill(torch.ones(10, dtype=torch.long, device="cuda"), [0, 4, 10], cache)
    with pytest.raises(ValueError, match="empty rows"):
        m.prefill(torch.ones(10, dtype=torch.long, device="cuda"), [0, 4, 10], cache)


def test_refused_calls_leave_the_cache_as_it_was():
    m = _model()
    vocab = m.embed_tokens.num_embeddings
    for bad in (-1, vocab):
        with pytest.raises(ValueError, match="token ids"):
            m.generate([[1, bad]], 2)
    cache = m.new_cache(2, 40, page_size=16)
    ids = torch.ones(10, dtype=torch.long, device="cuda")
    for cu in ([2, 4, 10], [0, 4, 9], [0, 10]):
        with pytest.raises(ValueError, match="one prompt"):
            m.prefill(ids, cu, cache)
    assert cache.lens == [0, 0]
    m.prefill(ids, [0, 4, 10], cache)
    with pytest.raises(ValueError, match="one per row"):
        m.decode(ids[:1], cache)
    for rows in ([0, 2], [-1]):
        with pytest.raises(ValueError, match="rows must lie"):
            cache.release(rows)
    assert cache.lens == [4, 6] and cache.seq_lens.tolist() == [4, 6]
    cache.release([1, 1])  # the same row twice
    assert cache.lens == [4, 0] and int(cache.n_free) == cache.n_pages - 1


def test_registered_operators():
    """The torch.library forms: opcheck (schema, mutation, shape functions) and equality."""
    from dsalt_b200 import library, serving  # noqa: F401
    g = torch.Generator(device="cuda").manual_seed(2)
    f8 = lambda: torch.randn(6, 2, 16, 64, device="cuda", generator=g).to(torch.float8_e4m3fn)  # noqa: E731
    kc, vc = f8(), f8()
    ks, vs = torch.full((6, 2), 0.25, device="cuda"), torch.full((6, 2), 0.5, device="cuda")
    tables = torch.tensor([[0, 1, 2], [3, 4, 5]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([40, 20], dtype=torch.int32, device="cuda")
    q = torch.randn(2, 4, 64, device="cuda", generator=g).bfloat16()
    w = torch.tensor([9, 20], dtype=torch.int32, device="cuda")
    lmk = torch.tensor([[[3, -1], [0, -1]]] * 4, dtype=torch.int32, device="cuda")
    args = (q, kc, vc, ks, vs, tables, lens, None, w, lmk, None, torch.float32)
    out = torch.ops.dsalt_b200.cache_attention(*args)
    assert torch.equal(out, serving.cache_attention(q, kc, vc, ks, vs, tables, lens, w_sizes=w, lmk_indices=lmk,
                                                    out_dtype=torch.float32))
    tests = ("test_schema", "test_faketensor")
    # (the schema test compares inputs by arithmetic that torch lacks for float8)
    torch.library.opcheck(torch.ops.dsalt_b200.cache_attention.default, args, test_utils=("test_faketensor",))
    lg, u = torch.randn(3, 100, device="cuda", generator=g), torch.rand(3, device="cuda", generator=g)
    torch.library.opcheck(torch.ops.dsalt_b200.sample_tokens.default, (lg, u, 0.8, 10, 0.9, 0.0), test_utils=tests)
    k = torch.randn(3, 2, 64, device="cuda", generator=g).bfloat16()
    slots = torch.tensor([16, 17, 18], device="cuda")
    a, b = (kc.clone(), vc.clone(), ks.clone(), vs.clone()), (kc.clone(), vc.clone(), ks.clone(), vs.clone())
    torch.ops.dsalt_b200.append_cache(k, k, *a, slots)
    serving.append_cache(k, k, *b, slots)
    assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(a, b))
