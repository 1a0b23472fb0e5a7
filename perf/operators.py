"""The serving operators as cases with work in them: slot maps, the 8-bit paged cache, the
attention that reads it, and sampling.

``run`` computes a case either in plain torch operations (``own`` false) or by the calls a
user's program makes of ``dsalt_b200`` (``own`` true). Definitions:

* slots: row ``s`` holds ``seq_lens[s]`` tokens in the pages ``block_tables[s]`` and wants
  ``new_lens[s]`` more. A row is granted when its table and the token budget hold it and it
  needs no page or the running sum of needed pages up to it is at most ``n_free``; the j-th
  page of that running order is ``free_pages[n_free - 1 - j]``.
* append: a page holds its tokens of one kv head in e4m3 with one power-of-two scale,
  ``2^e`` with the smallest ``e`` for which the largest magnitude is at most ``448 * 2^e``; ``e``
  never falls while the page fills, and a page whose first token is among the new ones
  starts afresh.
* attend: query at position ``i`` of width ``w`` attends to ``[i - w + 1, i]`` and to its head's
  landmarks ``p < i - w + 1`` (their logits plus ``bias``); without widths to ``[0, i]``.
* sample: of the weights ``exp((l - max l) / T)`` keep the ``top_k`` largest (order: logit
  descending, then index), of those the shortest prefix whose mass reaches ``top_p`` of
  theirs, of those the weights of at least ``min_p``; the token is the first index whose
  running sum over the kept weights exceeds ``u`` times their total.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
E_MIN = -110  # lowest scale exponent: 2^-110 times the smallest e4m3 value is a normal fp32
BIG = 448.0   # largest e4m3 value


def listed():
    return [
        # the start of one decode step of a half-busy server: one token for each running request
        dict(name="slots_step_64", op="slots", seqs=64, page=64, max_pages=512, cached=32768, new=1, budget=64,
             pool=100, cycle=False),
        # admission of 509 prompts at once, small pages, the pool too short for the last of them,
        # and their release
        dict(name="slots_admit_131072", op="slots", seqs=509, page=16, max_pages=64, cached=0, new=513,
             budget=131072, pool=85, cycle=True),
        # one decode step of one layer: a token for each of 64 requests, 16 kv heads of 64
        dict(name="append_step_64", op="append", seqs=64, kv_heads=16, head_dim=64, page=64, dtype="bf16", cached=4000,
             new=1),
        # four ragged prompts of about 8192 tokens, 12 kv heads of 64
        dict(name="append_prompts_4x8192", op="append", seqs=4, kv_heads=12, head_dim=64, page=64, dtype="bf16",
             cached=0, new=8192),
        # the next piece of three long prompts in fp32, 2 kv heads of 128, small pages half filled before
        dict(name="append_gqa_fp32", op="append", seqs=3, kv_heads=2, head_dim=128, page=16, dtype="fp32",
             cached=5001, new=1111),
        # one request's decode step in fp32, a short sequence: latency
        dict(name="attend_one_fp32", op="attend", seqs=1, heads=4, kv_heads=4, head_dim=64, page=16, dtype="fp32",
             cached=1021, q_len=1, w_max=128, k_lmk=32, bias=False),
        # a decode step of 64 requests with windows and landmarks, 16 heads of 64
        dict(name="attend_dsalt_64", op="attend", seqs=64, heads=16, kv_heads=16, head_dim=64, page=64, dtype="bf16",
             cached=16384, q_len=1, w_max=512, k_lmk=128, bias=False),
        # one very long sequence, every key: the key axis has to be split
        dict(name="attend_full_131072", op="attend", seqs=1, heads=16, kv_heads=16, head_dim=64, page=64,
             dtype="bf16", cached=131072, q_len=1, w_max=0, k_lmk=0, bias=False),
        # sixteen ragged sequences up to 32768, every key, 16 query heads on 2 kv heads of 128
        dict(name="attend_full_gqa_16", op="attend", seqs=16, heads=16, kv_heads=2, head_dim=128, page=64,
             dtype="bf16", cached=32768, q_len=1, w_max=0, k_lmk=0, bias=False),
        # up to seven drafted tokens for each of 23 requests, windows and biased landmarks, grouped heads
        dict(name="attend_drafts_fp16", op="attend", seqs=23, heads=16, kv_heads=2, head_dim=128, page=32,
             dtype="fp16", cached=8191, q_len=7, w_max=512, k_lmk=128, bias=True),
        # one request's token: latency
        dict(name="sample_one", op="sample", rows=1, vocab=50257, dtype="fp32", filters="all"),
        # 64 requests that each bring their own settings, the larger vocabulary
        dict(name="sample_mixed_64", op="sample", rows=64, vocab=151936, dtype="bf16", filters="mixed"),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["slots", "append", "attend", "attend", "sample"])
    page = rng.choice([16, 32, 64, 128])
    if op == "slots":
        if rng.random() < 0.5:
            seqs, cached = _log_uniform(rng, 1, 509), _log_uniform(rng, 1, 32768)
            return dict(op=op, seqs=seqs, page=page, max_pages=-(-cached // page) + 2, cached=cached,
                        new=rng.choice([1, 1, 5]), budget=5 * seqs, pool=rng.choice([60, 100]), cycle=False)
        seqs = _log_uniform(rng, 1, 509)
        new = _log_uniform(rng, 1, 131072 // seqs)
        return dict(op=op, seqs=seqs, page=page, max_pages=-(-new // page) + 1, cached=0, new=new,
                    budget=seqs * new, pool=rng.choice([60, 85, 100]), cycle=True)
    if op == "append":
        kv_heads, head_dim = rng.choice([(16, 64), (12, 64), (4, 64), (2, 128), (8, 128), (1, 128)])
        seqs = _log_uniform(rng, 1, 128)
        new = rng.choice([1, _log_uniform(rng, 1, max(1, 24576 // seqs // max(1, kv_heads * head_dim // 1024)))])
        return dict(op=op, seqs=seqs, kv_heads=kv_heads, head_dim=head_dim, page=page,
                    dtype=rng.choice(["bf16", "fp16", "fp32"]), cached=_log_uniform(rng, 1, 4096 // max(1, seqs // 16)),
                    new=new)
    if op == "attend":
        heads, kv_heads, head_dim = rng.choice([(16, 16, 64), (12, 12, 64), (4, 4, 64), (16, 2, 128), (16, 4, 128),
                                                (6, 2, 64), (5, 1, 128)])
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        if rng.random() < 0.5:  # every key
            seqs = _log_uniform(rng, 1, 32)
            cached = _log_uniform(rng, 1, 131072 // seqs // max(1, kv_heads // 4))
            return dict(op=op, seqs=seqs, heads=heads, kv_heads=kv_heads, head_dim=head_dim, page=page, dtype=dtype,
                        cached=cached, q_len=rng.choice([1, 1, 3]) if cached < 4096 else 1, w_max=0, k_lmk=0,
                        bias=False)
        seqs, q_len = _log_uniform(rng, 1, 64), rng.choice([1, 1, 2, 5])
        return dict(op=op, seqs=max(1, seqs // q_len), heads=heads, kv_heads=kv_heads, head_dim=head_dim, page=page,
                    dtype=dtype, cached=_log_uniform(rng, 1, 16384), q_len=q_len, w_max=rng.choice([64, 256, 512]),
                    k_lmk=rng.choice([0, 1, 33, 64, 128]), bias=rng.random() < 0.5)
    vocab = rng.choice([50257, 151936, _log_uniform(rng, 100, 151936)])
    return dict(op=op, rows=_log_uniform(rng, 1, 9_700_000 // max(vocab, 37890)), vocab=vocab,
                dtype=rng.choice(["bf16", "fp16", "fp32"]), filters=rng.choice(["all", "mixed", "top_p", "none"]))


# ---------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return {"slots": _prepare_slots, "append": _prepare_append, "attend": _prepare_attend,
            "sample": _prepare_sample}[case["op"]](case, g)


def _randint(g, lo, hi, shape):
    """Whole numbers in [lo, hi]."""
    return torch.randint(lo, hi + 1, shape, device="cuda", generator=g, dtype=torch.int32)


def _lengths(case, lo, hi, shape):
    """The lengths are the case's, whatever the seed: they are the sizes of its tensors."""
    g = torch.Generator(device="cuda").manual_seed(case["seqs"] * 131071 + case["cached"] * 31 + case["page"])
    return _randint(g, lo, hi, shape)


def _tables(g, lens, page, max_pages, n_pages):
    """Block tables of `lens` over a shuffled pool, and the pages that are left, as a stack."""
    pages = (lens + page - 1) // page
    upto = torch.cumsum(pages, 0)
    order = torch.randperm(n_pages, device="cuda", generator=g).to(torch.int32)
    cols = torch.arange(max_pages, device="cuda")
    held = cols < pages[:, None]
    at = ((upto - pages)[:, None] + cols).clamp(max=n_pages - 1)
    tables = torch.where(held, order[at], -1).to(torch.int32).contiguous()
    free = torch.cat([order[int(upto[-1]):], order.new_full((int(upto[-1]),), -1)])
    return tables, free.contiguous()


def _prepare_slots(case, g):
    S, page = case["seqs"], case["page"]
    if case["cycle"]:
        lens = torch.zeros(S, dtype=torch.int32, device="cuda")
        new = _randint(g, 0, case["new"], (S,))
    else:
        lens = _randint(g, 0, case["cached"], (S,))
        new = torch.where(_randint(g, 0, 7, (S,)) > 0, _randint(g, 1, case["new"], (S,)), 0).to(torch.int32)
        if S > 1:  # a row whose next token opens a page
            lens[S // 2] = lens[S // 2] // page * page
    wanted = int(((lens + new + page - 1) // page - (lens + page - 1) // page).sum())
    spare = max(1, wanted * case["pool"] // 100)
    held = int(((lens + page - 1) // page).sum())
    pool = S * (-(-case["cached"] // page) + -(-case["new"] // page) + 1)
    tables, free = _tables(g, lens, page, case["max_pages"], held + spare)
    free = torch.cat([free, free.new_full((pool - len(free),), -1)])
    return dict(case=case, block_tables=tables, seq_lens=lens, new_lens=new, free_pages=free,
                n_free=torch.full((1,), spare, dtype=torch.int32, device="cuda"),
                every=torch.ones(S, dtype=torch.bool, device="cuda"))


def _cache(g, n_pages, H, page, D):
    """A pool in use: bytes of normal values under scales that differ from page to page."""
    x = torch.randn(n_pages, H, page, D, device="cuda", generator=g) * 100.0
    return x.clamp(-BIG, BIG).to(torch.float8_e4m3fn), torch.exp2(_randint(g, -8, -5, (n_pages, H)).float())


def _prepare_append(case, g):
    S, page, H, D = case["seqs"], case["page"], case["kv_heads"], case["head_dim"]
    old = _lengths(case, 0, case["cached"], (S,))
    new = _lengths(case, max(1, case["new"] * 3 // 4), case["new"], (S,))
    n_pages = int(((old + new + page - 1) // page).sum()) + 3
    tables, _ = _tables(g, old + new, page, int((old + new).max()) // page + 1, n_pages)
    cu = torch.cumsum(new, 0)
    tok = torch.arange(int(cu[-1]), device="cuda")
    s = torch.searchsorted(cu, tok, right=True)
    pos = old[s] + tok - (cu - new)[s]
    slots = tables[s, pos // page].long() * page + pos % page
    dt = DTYPES[case["dtype"]]
    kc, ks = _cache(g, n_pages, H, page, D)
    vc, vs = _cache(g, n_pages, H, page, D)
    # keys carry channels of larger size, as rotary keys do
    k = torch.randn(len(tok), H, D, device="cuda", generator=g) * (1 + 4 * (torch.arange(D, device="cuda") % 16 == 3))
    v = torch.randn(len(tok), H, D, device="cuda", generator=g)
    return dict(case=case, k=k.to(dt), v=v.to(dt), k_cache=kc, v_cache=vc, k_scale=ks, v_scale=vs, slots=slots)


def _prepare_attend(case, g):
    S, page, H, Hkv, D = case["seqs"], case["page"], case["heads"], case["kv_heads"], case["head_dim"]
    n = case["cached"]
    lens = _lengths(case, max(1, n // 4), n, (S,))
    lens[0] = n
    q_lens = torch.minimum(_lengths(case, 1, case["q_len"], (S,)), lens)
    cu = torch.cat([q_lens.new_zeros(1), torch.cumsum(q_lens, 0).to(torch.int32)]).contiguous()
    T = int(cu[-1])
    n_pages = int(((lens + page - 1) // page).sum()) + 1
    tables, _ = _tables(g, lens, page, -(-n // page), n_pages)
    kc, ks = _cache(g, n_pages, Hkv, page, D)
    vc, vs = _cache(g, n_pages, Hkv, page, D)
    q = torch.randn(T, H, D, device="cuda", generator=g).to(DTYPES[case["dtype"]])
    w = lmk = bias = None
    if case["w_max"]:
        w = _randint(g, 16, case["w_max"], (T,))
        if case["k_lmk"]:
            # ascending distinct positions of the part a whole number of blocks back, -1 behind them
            k = case["k_lmk"]
            step = torch.rand(H, S, k, device="cuda", generator=g)
            at = torch.cumsum(step + 1e-3, 2)
            at = (at / (at[..., -1:] + 1) * lens[:, None]).floor().to(torch.int32)
            keep = torch.cat([torch.ones_like(at[..., :1], dtype=torch.bool), at[..., 1:] > at[..., :-1]], 2)
            at = torch.where(keep & (at < (lens // 512 * 512)[:, None]), at, 2**31 - 1)
            at = torch.sort(at, dim=2).values
            lmk = torch.where(at < 2**31 - 1, at, -1).to(torch.int32).contiguous()
            if case["bias"]:
                bias = -torch.rand(H, S, k, device="cuda", generator=g) * 3
    return dict(case=case, q=q, k_cache=kc, v_cache=vc, k_scale=ks, v_scale=vs, block_tables=tables, seq_lens=lens,
                cu_q=None if case["q_len"] == 1 else cu, w=w, lmk=lmk, bias=bias)


def _prepare_sample(case, g):
    B, V = case["rows"], case["vocab"]
    logits = torch.randn(B, V, device="cuda", generator=g) * 2.2
    # a few tokens stand out, by an amount that differs from row to row
    top = torch.randint(0, V, (B, 24), device="cuda", generator=g)
    logits.scatter_add_(1, top, torch.rand(B, 24, device="cuda", generator=g) * 9 * torch.rand(
        B, 1, device="cuda", generator=g))
    if V > 1000:
        logits[:, V - 11:] = float("-inf")  # padding of the vocabulary
    u = torch.rand(B, device="cuda", generator=g)
    f = case["filters"]
    t = dict(temperature=0.8, top_k=0, top_p=1.0, min_p=0.0)
    if f == "all":
        t = dict(temperature=0.8, top_k=50, top_p=0.9, min_p=0.02)
    elif f == "top_p":
        t = dict(temperature=1.0, top_k=0, top_p=0.95, min_p=0.0)
    elif f == "mixed":
        pick = lambda v, dt: torch.tensor(v, dtype=dt, device="cuda")[  # noqa: E731
            torch.randint(0, len(v), (B,), device="cuda", generator=g)].contiguous()
        t = dict(temperature=pick([0.0, 0.6, 0.8, 1.0, 1.3], torch.float32), top_k=pick([0, 0, 20, 50, 1000], torch.int32),
                 top_p=pick([0.7, 0.9, 0.95, 1.0], torch.float32), min_p=pick([0.0, 0.0, 0.05], torch.float32))
    return dict(case=case, logits=logits.to(DTYPES[case["dtype"]]), u=u, **t)


# ---------------------------------------------------------------------- one pass
def run(state):
    op = state["case"]["op"]
    if own:
        return {"slots": _own_slots, "append": _own_append, "attend": _own_attend, "sample": _own_sample}[op](state)
    return {"slots": _plain_slots, "append": _plain_append, "attend": _plain_attend,
            "sample": _plain_sample}[op](state)


def _own_slots(s):
    import dsalt_b200 as D
    case = s["case"]
    if not case["cycle"]:
        p = D.reserve_slots(s["block_tables"], s["seq_lens"], s["new_lens"], s["free_pages"], s["n_free"],
                            case["page"], case["budget"])
        return p.slots, p.positions, p.cu_new, p.granted, p.seq_lens, p.n_free, s["block_tables"]
    p = D.reserve_slots(s["block_tables"], s["seq_lens"], s["new_lens"], s["free_pages"], s["n_free"], case["page"],
                        case["budget"], inplace=True)
    D.release_slots(s["block_tables"], s["seq_lens"], s["every"], s["free_pages"], s["n_free"], case["page"])
    return (p.slots, p.positions, p.cu_new, p.granted, s["seq_lens"], s["n_free"], s["block_tables"],
            s["free_pages"])


def _own_append(s):
    import dsalt_b200 as D
    D.append_cache(s["k"], s["v"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["slots"])
    return s["k_cache"], s["k_scale"], s["v_cache"], s["v_scale"]


def _own_attend(s):
    import dsalt_b200 as D
    return D.cache_attention(s["q"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["block_tables"],
                             s["seq_lens"], cu_q=s["cu_q"], w_sizes=s["w"], lmk_indices=s["lmk"], lmk_bias=s["bias"],
                             return_lse=True)


def _own_sample(s):
    import dsalt_b200 as D
    return D.sample_tokens(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                           min_p=s["min_p"], return_logprob=True)


def _plain_slots(s):
    case, page, n_tokens = s["case"], s["case"]["page"], s["case"]["budget"]
    tables, free, n_free = s["block_tables"], s["free_pages"], s["n_free"]
    old, new = s["seq_lens"].clamp(min=0).long(), s["new_lens"].clamp(min=0).long()
    S, max_pages = tables.shape
    end = torch.cumsum(new, 0)
    have, want = (old + page - 1) // page, (old + new + page - 1) // page
    fits = (want <= max_pages) & (end <= n_tokens)
    need = torch.where(fits, want - have, 0)
    upto = torch.cumsum(need, 0)
    granted = fits & ((need == 0) | (upto <= n_free))
    take = torch.where(granted, need, 0)
    cols = torch.arange(max_pages, device=tables.device)
    j = (upto - need)[:, None] + cols - have[:, None]
    fresh = (cols >= have[:, None]) & (cols < (have + take)[:, None])
    tables.copy_(torch.where(fresh, free[(n_free.long() - 1 - j).clamp(0, free.numel() - 1)], tables))
    cu = torch.cat([end.new_zeros(1), end]).clamp(max=n_tokens)
    tok = torch.arange(n_tokens, device=tables.device)
    row = torch.searchsorted(end, tok, right=True)
    real = row < S
    row = row.clamp(max=S - 1)
    pos = old[row] + tok - cu[row]
    at = tables[row, (pos // page).clamp(max=max_pages - 1)].long()
    real = real & granted[row]
    slots = torch.where(real & (at >= 0), at * page + pos % page, -1)
    positions = torch.where(real, pos, 0).to(torch.int32)
    lens = torch.where(granted, old + new, old).to(torch.int32)
    left = (n_free - take.sum()).to(torch.int32)
    if not case["cycle"]:
        return slots, positions, cu.to(torch.int32), granted, lens, left, tables
    held = (lens.long() + page - 1) // page
    upto = torch.cumsum(held, 0)
    total = upto[-1]
    j = (upto - held)[:, None] + cols
    mine = cols < held[:, None]
    # page j of the rows in order goes to free[left + total - 1 - j]
    to = torch.where(mine, left.long() + total - 1 - j, free.numel())
    more = torch.cat([free, free.new_zeros(1)])
    more[to.reshape(-1)] = tables.reshape(-1)
    free.copy_(more[:-1])
    tables.fill_(-1)
    n_free.copy_(left + total.to(torch.int32))
    s["seq_lens"].zero_()
    return slots, positions, cu.to(torch.int32), granted, s["seq_lens"], n_free, tables, free


def _need_exponent(amax):
    """The smallest e with amax <= 448 * 2^e, at least E_MIN: 448 = 0.875 * 2^9."""
    m, x = torch.frexp(amax)
    e = torch.where(m <= 0.875, x - 9, x - 8)
    return torch.where(amax > 0, e, E_MIN).clamp(min=E_MIN)


def _plain_put(x, cache, scale, slots):
    n_pages, H, page, D = cache.shape
    at, off = slots // page, slots % page
    x = x.float()
    size = torch.where(torch.isfinite(x), x.abs(), 0.0).amax(2)
    amax = torch.zeros(n_pages, H, device=x.device).scatter_reduce(0, at[:, None].expand(-1, H), size, "amax")
    fresh = torch.zeros(n_pages, dtype=torch.int32, device=x.device).index_add(0, at, (off == 0).to(torch.int32)) > 0
    touched = torch.zeros(n_pages, dtype=torch.bool, device=x.device).index_fill(0, at, True)
    was = (torch.frexp(scale)[1] - 1).clamp(min=E_MIN)
    was = torch.where((scale > 0) & ~fresh[:, None], was, E_MIN)
    e = torch.where(touched[:, None], torch.maximum(was, _need_exponent(amax)), was)
    pages = at if len(at) <= n_pages else torch.arange(n_pages, device=x.device)
    older = cache[pages].float()
    shrink = torch.where(touched & ~fresh, 1.0, 0.0)[:, None] * (was - e)
    cache[pages] = (older * torch.exp2(shrink[pages])[:, :, None, None]).to(torch.float8_e4m3fn)
    bits = (x * torch.exp2(-e[at].float())[:, :, None]).clamp(-BIG, BIG).to(torch.float8_e4m3fn)
    cache[at, :, off] = bits
    scale.copy_(torch.where(touched[:, None], torch.exp2(e.float()), scale))


def _plain_append(s):
    _plain_put(s["k"], s["k_cache"], s["k_scale"], s["slots"])
    _plain_put(s["v"], s["v_cache"], s["v_scale"], s["slots"])
    return s["k_cache"], s["k_scale"], s["v_cache"], s["v_scale"]


def _plain_attend(s):
    q, tables, lens, page = s["q"], s["block_tables"], s["seq_lens"].long(), s["case"]["page"]
    T, H, D = q.shape
    Hkv = s["k_cache"].shape[1]
    G = H // Hkv
    tok = torch.arange(T, device=q.device)
    if s["cu_q"] is None:
        row, pos = tok, lens - 1
    else:
        cu = s["cu_q"].long()
        row = torch.searchsorted(cu[1:], tok, right=True)
        pos = lens[row] - cu[row + 1] + tok
    W = s["case"]["w_max"] or s["case"]["cached"]
    w = s["w"].long() if s["w"] is not None else torch.full_like(pos, W)
    first = (pos - w + 1).clamp(min=0)
    j = pos[:, None] - torch.arange(W, device=q.device)                                    # [T, W]
    in_window = j >= first[:, None]
    j = j.clamp(min=0)
    at = tables[row[:, None], j // page].long()
    k = s["k_cache"][at, :, j % page].float() * s["k_scale"][at][..., None]                # [T, W, Hkv, D]
    v = s["v_cache"][at, :, j % page].float() * s["v_scale"][at][..., None]
    qg = q.float().view(T, Hkv, G, D) / math.sqrt(D)
    logits = torch.matmul(qg, k.permute(0, 2, 3, 1)).view(T, H, W)
    logits = torch.where(in_window[:, None], logits, float("-inf"))
    if s["lmk"] is not None:
        p = s["lmk"].long().transpose(0, 1)[row]                                           # [T, H, k]
        valid = (p >= 0) & (p < first[:, None, None])
        p = torch.where(valid, p, 0)
        at = tables[row[:, None, None], p // page].long()
        h = (torch.arange(H, device=q.device) // G)[:, None]
        lk = s["k_cache"][at, h, p % page].float() * s["k_scale"][at, h][..., None]        # [T, H, k, D]
        lv = s["v_cache"][at, h, p % page].float() * s["v_scale"][at, h][..., None]
        more = torch.matmul(lk, qg.reshape(T, H, D, 1))[..., 0]
        if s["bias"] is not None:
            more = more + s["bias"].transpose(0, 1)[row]
        logits = torch.cat([logits, torch.where(valid, more, float("-inf"))], 2)
    top = logits.amax(2, keepdim=True)
    e = torch.exp(logits - top)
    total = e.sum(2, keepdim=True)
    out = torch.matmul(e[..., :W].reshape(T, Hkv, G, W), v.permute(0, 2, 1, 3)).reshape(T, H, D)
    if s["lmk"] is not None:
        out = out + torch.matmul(e[:, :, None, W:], lv)[:, :, 0]
    return (out / total).to(q.dtype), (top + torch.log(total))[..., 0]


def _column(v, like, dtype):
    return v.to(dtype)[:, None] if isinstance(v, torch.Tensor) else torch.full((like.shape[0], 1), v, dtype=dtype,
                                                                               device=like.device)


def _plain_sample(s):
    # in 64 bits: whether a running sum reaches a border decides a token
    lg = s["logits"].float()
    V = lg.shape[1]
    t = _column(s["temperature"], lg, torch.float32).double()
    k = _column(s["top_k"], lg, torch.int64)
    top_p = _column(s["top_p"], lg, torch.float32).double()
    min_p = _column(s["min_p"], lg, torch.float32).double()
    ranked, order = torch.sort(lg, dim=1, descending=True, stable=True)
    top = ranked[:, :1]
    z = (ranked.double() - top.double()) / torch.where(t > 0, t, 1.0)
    w = torch.where(ranked == top, 1.0, torch.exp(z))
    rank = torch.arange(V, device=lg.device)
    keep = (rank < torch.where(k > 0, k, V)) & ((t > 0) | (rank == 0))
    run_sum = torch.cumsum(torch.where(keep, w, 0.0), 1)
    total = run_sum[:, -1:]
    before = torch.cat([torch.zeros_like(total), run_sum[:, :-1]], 1)
    keep = keep & ((before < top_p * total) | (top_p >= 1) | (rank == 0)) & (w >= min_p)
    kept = torch.zeros_like(w).scatter_(1, order, torch.where(keep, w, 0.0))
    cdf = torch.cumsum(kept, 1)
    total = cdf[:, -1:]
    over = cdf > s["u"].double()[:, None] * total
    token = torch.argmax(over.to(torch.uint8), 1)
    mass = torch.gather(kept, 1, token[:, None])
    return token, torch.log(mass / total)[:, 0].float()


# ---------------------------------------------------------------------- work
def work(case):
    op = case["op"]
    if op == "slots":
        S, page = case["seqs"], case["page"]
        tokens = S * (case["new"] + 1) / 2 if case["cycle"] else S
        pages = tokens / page
        # lengths and grants in and out, 12 bytes a token of the budget, a page's entry in and out
        return {"bytes": S * 21 + case["budget"] * 12 + pages * (24 if case["cycle"] else 8), "flops": tokens}
    if op == "append":
        n = case["seqs"] * (case["new"] + max(1, case["new"] * 3 // 4)) / 2 * case["kv_heads"] * case["head_dim"]
        return {"bytes": 2 * n * (BYTES[case["dtype"]] + 1) + case["seqs"] * case["new"] * 8, "flops": 4 * n}
    if op == "attend":
        S, H, Hkv, D, n = case["seqs"], case["heads"], case["kv_heads"], case["head_dim"], case["cached"]
        queries = S * (1 + case["q_len"]) / 2
        mean = (n + (S - 1) * 0.625 * n) / S
        window = min(mean, (16 + case["w_max"]) / 2) if case["w_max"] else mean
        lmk = min(case["k_lmk"], max(0, mean - window)) * 0.9 if case["w_max"] else 0
        seen = min(mean, window + (case["q_len"] - 1) / 2)  # the drafted tokens of a row share their window
        return {"bytes": 2 * S * D * (Hkv * seen + H * lmk) + S * H * lmk * (8 if case["bias"] else 4) +
                queries * H * (2 * D * BYTES[case["dtype"]] + 4),
                "flops": 4 * queries * H * D * (window + lmk)}
    B, V = case["rows"], case["vocab"]
    return {"bytes": B * V * BYTES[case["dtype"]] + B * 32, "flops": 8 * B * V}


# ---------------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"slots": lambda s: None, "append": _exact_append, "attend": _exact_attend,
            "sample": _exact_sample}[case["op"]](s)


def _e4m3(x):
    """Nearest e4m3 value, ties to even, of 64-bit numbers; beyond the largest: the largest."""
    a = x.abs().clamp(max=BIG)
    step = torch.exp2((torch.frexp(a.clamp(min=2.0 ** -6))[1] - 4).double())
    return torch.sign(x) * (torch.round(a / step) * step).clamp(max=BIG)


def _exact_append(s):
    slots = s["slots"].tolist()
    page = s["k_cache"].shape[2]
    runs, at = [], 0
    while at < len(slots):  # the tokens of one page stand together
        n = 1
        while at + n < len(slots) and slots[at + n] // page == slots[at] // page:
            n += 1
        runs.append((at, n, slots[at] // page, slots[at] % page))
        at += n
    outs = []
    for x, cache, scale in ((s["k"], s["k_cache"], s["k_scale"]), (s["v"], s["v_cache"], s["v_scale"])):
        x, c, sc = x.double(), cache.double(), scale.double()
        for at, n, p, off in runs:
            amax = x[at:at + n].abs().amax((0, 2))
            e = torch.ceil(torch.log2(amax / BIG))
            e = torch.where(amax <= BIG * torch.exp2(e - 1), e - 1, e)  # log2 may be off by its last bit
            e = torch.where(amax > BIG * torch.exp2(e), e + 1, e)
            if off > 0:
                old = sc[p].clone()
                e = torch.maximum(e, torch.round(torch.log2(old)))
                c[p] = _e4m3(c[p] * (old * torch.exp2(-e))[:, None, None])
            sc[p] = torch.exp2(e)
            c[p, :, off:off + n] = _e4m3(x[at:at + n].transpose(0, 1) * torch.exp2(-e)[:, None, None])
        outs += [c, sc]
    return outs


def _exact_attend(s):
    q, lens = s["q"].double(), s["seq_lens"].tolist()
    T, H, D = q.shape
    Hkv = s["k_cache"].shape[1]
    cu = s["cu_q"].tolist() if s["cu_q"] is not None else list(range(len(lens) + 1))
    out, lse = torch.zeros_like(q), torch.zeros(T, H, dtype=torch.float64, device=q.device)
    for b, n in enumerate(lens):
        at = s["block_tables"][b, :-(-n // s["case"]["page"])].long()
        k = (s["k_cache"][at].double() * s["k_scale"][at].double()[..., None, None]).transpose(0, 1)
        v = (s["v_cache"][at].double() * s["v_scale"][at].double()[..., None, None]).transpose(0, 1)
        k, v = k.reshape(Hkv, -1, D)[:, :n], v.reshape(Hkv, -1, D)[:, :n]
        for t in range(cu[b], cu[b + 1]):
            i = n - cu[b + 1] + t
            lo = max(0, i - int(s["w"][t]) + 1) if s["w"] is not None else 0
            qt = q[t].view(Hkv, H // Hkv, D)
            x = torch.einsum("hgd,hnd->hgn", qt, k).reshape(H, n) / math.sqrt(D)
            add = torch.full((H, n), -math.inf, dtype=torch.float64, device=q.device)
            add[:, lo:i + 1] = 0
            if s["lmk"] is not None:
                p = s["lmk"][:, b].long()
                b_p = s["bias"][:, b].double() if s["bias"] is not None else torch.zeros_like(p, dtype=torch.float64)
                ok = (p >= 0) & (p < lo)
                h = torch.arange(H, device=q.device)[:, None].expand_as(p)
                add[h[ok], p[ok]] = b_p[ok]
            x = x + add
            lse[t] = torch.logsumexp(x, 1)
            prob = torch.exp(x - lse[t][:, None]).view(Hkv, H // Hkv, n)
            out[t] = torch.einsum("hgn,hnd->hgd", prob, v).reshape(H, D)
    return out, lse


def _exact_sample(s):
    lg, u = s["logits"].double(), s["u"].double()
    B, V = lg.shape
    row = lambda name, i: float(s[name][i]) if isinstance(s[name], torch.Tensor) else s[name]  # noqa: E731
    f32 = lambda x: float(torch.tensor(x, dtype=torch.float32))  # noqa: E731
    logprob = torch.zeros(B, dtype=torch.float64, device=lg.device)
    for i in range(B):
        t, k, top_p, min_p = f32(row("temperature", i)), int(row("top_k", i)), f32(row("top_p", i)), f32(row("min_p", i))
        if t <= 0:
            continue
        p = torch.exp(lg[i] / t - torch.logsumexp(lg[i] / t, 0))
        idx = torch.argsort(-lg[i], stable=True)
        if k > 0:
            idx = idx[:k]
        mass = torch.cumsum(p[idx], 0)
        if top_p < 1:
            idx = idx[:max(1, int((mass - p[idx] < top_p * mass[-1]).sum()))]
        idx = idx[p[idx] >= min_p * p.max() * (1 - 1e-15)]
        idx = torch.sort(idx).values
        mass = torch.cumsum(p[idx], 0)
        at = int((mass <= u[i] * mass[-1]).sum())
        logprob[i] = torch.log(p[idx[min(at, len(idx) - 1)]] / mass[-1])
    return None, logprob
