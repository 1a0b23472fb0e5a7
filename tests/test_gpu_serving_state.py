"""The state that the serving operators leave behind, looked at in full: every cache tensor and every grant
of a sequence of steps, lengths beyond a full table, answers that do not end."""
import numpy as np
import pytest
import torch
from test_gpu_serving import F8, attend_case, check_attend, to_gpu

from oracle import serving_oracle as O

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("q_lens,w_max", [([1, 1], 0), ([1, 1], 20), ([5, 2], 33), ([9, 1], 40)])
def test_a_length_beyond_a_full_table_counts_to_the_tables_end(dtype, q_lens, w_max):
    from dsalt_b200 import ops, serving
    page = 16
    c = attend_case(31, [4 * page, 40], q_lens, 4, 2, 64, page, dtype, w_max, 6 if w_max else 0)
    c["tables"] = np.ascontiguousarray(c["tables"][:, :4])  # the first row fills its table
    args = to_gpu(c)
    for n in (4 * page, 4 * page + 1, 10**9, 2**31 - 1):
        args["seq_lens"][0] = n
        out, lse = serving.cache_attention(**args, return_lse=True)
        check_attend(c, out, lse, f"length {n}")
    assert ops.device_status() == 0


def test_serving_steps_leave_the_state_that_the_oracle_says():
    from dsalt_b200 import ops, serving as V
    g = np.random.default_rng(41)
    S, H, Hkv, D, page, n_pages, max_pages = 6, 4, 2, 64, 16, 30, 9
    tg = torch.Generator().manual_seed(41)
    free0 = g.permutation(n_pages).astype(np.int32)
    tables = torch.full((S, max_pages), -1, dtype=torch.int32, device="cuda")
    lens = torch.zeros(S, dtype=torch.int32, device="cuda")
    free, n_free = torch.from_numpy(free0).cuda(), torch.tensor([n_pages], dtype=torch.int32, device="cuda")
    kc, vc = (torch.zeros(n_pages, Hkv, page, D, device="cuda").to(F8) for _ in range(2))
    ks, vs = (torch.zeros(n_pages, Hkv, device="cuda") for _ in range(2))
    rt, rl, rf, rn = tables.cpu().numpy(), lens.cpu().numpy(), free0, n_pages
    rk, rv = ((np.zeros((n_pages, Hkv, page, D)), np.zeros((n_pages, Hkv))) for _ in range(2))
    refused = 0
    for step in range(16):
        most = 70 if step in (0, 6, 11) else 4
        new = g.integers(0, most, S).astype(np.int32)
        room = int(new.sum()) + (3 if step % 3 else -2)  # at times too little
        plan = V.reserve_slots(tables, lens, torch.from_numpy(new).cuda(), free, n_free, page, max(room, 0), inplace=True)
        rt, slots, positions, cu, granted, rl, rn = O.reserve(rt, rl, new, rf, rn, page, max(room, 0))
        for a, b, name in ((tables, rt, "tables"), (plan.slots, slots, "slots"), (plan.positions, positions, "positions"),
                           (plan.cu_new, cu, "cu_new"), (plan.granted, granted, "granted"), (lens, rl, "lens"),
                           (n_free, np.array([rn]), "n_free")):
            np.testing.assert_array_equal(a.cpu().numpy(), b, err_msg=f"{name} of step {step}")
        refused += int((~granted).sum())
        T = len(slots)
        k, v, q = (torch.randn(T, h, D, generator=tg).bfloat16() for h in (Hkv, Hkv, H))
        V.append_cache(k.cuda(), v.cuda(), kc, vc, ks, vs, plan.slots)
        rk, rv = O.append(k.double().numpy(), *rk, slots, page), O.append(v.double().numpy(), *rv, slots, page)
        for (a, s), (b, t) in (((kc, ks), rk), ((vc, vs), rv)):
            np.testing.assert_array_equal(a.double().cpu().numpy(), b, err_msg=f"step {step}")
            np.testing.assert_array_equal(s.cpu().numpy(), t, err_msg=f"step {step}")
        # of rows that were refused the last tokens are asked again
        out, lse = V.cache_attention(q.cuda(), kc, vc, ks, vs, tables, lens, cu_q=plan.cu_new, return_lse=True)
        c = dict(q=q[:cu[-1]], kc=rk[0], vc=rv[0], ks=rk[1], vs=rv[1], tables=rt, lens=rl, cu=cu, w=None, lmk=None, bias=None)
        check_attend(c, out[:cu[-1]], lse[:cu[-1]], f"step {step}")
        assert (out[cu[-1]:] == 0).all()
        if step in (5, 9, 13):
            flags = g.random(S) < 0.5
            V.release_slots(tables, lens, torch.from_numpy(flags).cuda(), free, n_free, page)
            rt, rl, rf, rn = O.release(rt, rl, flags, rf, rn, page)
            np.testing.assert_array_equal(tables.cpu().numpy(), rt)
            np.testing.assert_array_equal(free.cpu().numpy()[:rn], rf[:rn])
    assert refused > 0 and ops.device_status() == 0


def test_an_answer_without_the_eos_token_runs_to_its_end():
    from dsalt_b200 import DSALTConfig, DSALTLMHeadModel
    torch.manual_seed(3)
    m = DSALTLMHeadModel.from_config(DSALTConfig(vocab_size=777, d_model=256, n_layers=2, n_heads=4, n_min=8, n_max=64, k_lmk=16,
                                                 max_seq_len=400, d_ff=512, selection="block_causal", block=128))
    m = m.cuda().bfloat16().eval()
    prompts = [[1, 2, 3], [4] * 65, [9, 8]]
    draw = lambda **kw: m.generate(prompts, 9, temperature=1.0,  # noqa: E731
                                   generator=torch.Generator(device="cuda").manual_seed(2), **kw)
    free = draw()
    never = next(t for t in range(777) if all(t not in a for a in free))
    assert draw(eos_token=never) == free
    # a token of one answer: that one ends with it, the others go on to theirs or to the end
    eos = free[0][4]
    want = [a[:a.index(eos) + 1] if eos in a else a for a in free]
    assert draw(eos_token=eos) == want and len(want[0]) < 9


def test_registered_attention_and_sampling_of_several_tokens():
    """The registered forms with packed query tokens, biased landmarks and types of their own equal the
    functions."""
    from dsalt_b200 import library, serving  # noqa: F401
    for dtype, out_dtype in ((torch.float16, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float32, torch.float16)):
        c = to_gpu(attend_case(51, [90, 33, 7], [3, 1, 7], 4, 2, 64, 16, dtype, 30, 9, True))
        names = ("q", "k_cache", "v_cache", "k_scale", "v_scale", "block_tables", "seq_lens", "cu_q", "w_sizes",
                 "lmk_indices", "lmk_bias")
        got = torch.ops.dsalt_b200.cache_attention(*(c[n] for n in names), out_dtype)
        assert torch.equal(got, serving.cache_attention(**c, out_dtype=out_dtype)) and got.dtype == out_dtype
    g = torch.Generator(device="cuda").manual_seed(5)
    lg, u = torch.randn(9, 4000, device="cuda", generator=g).half(), torch.rand(9, device="cuda", generator=g)
    tok, lp = torch.ops.dsalt_b200.sample_tokens(lg, u, 0.7, 0, 0.9, 0.01)
    want = serving.sample_tokens(lg, u, temperature=0.7, top_p=0.9, min_p=0.01, return_logprob=True)
    assert torch.equal(tok, want[0]) and torch.equal(lp, want[1])
